// Root-mean-square norm, with the residual's addition in front of it and an output in 8 bits behind.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"

namespace b200 {
namespace {

constexpr unsigned kMany = 4 * 148;   // rows from which on a thread has kEach pieces of each (four blocks for each SM)
constexpr int kEach = 2;
constexpr int kMaxThreads = 1024, kShort = 32, kShortThreads = 256, kRows = 2;   // threads of a row; of a row that shares its block with others

template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<2> { typedef uint16_t type; };
template <> struct Raw<1> { typedef uint8_t type; };
// VEC elements that lie side by side, moved at once.
template <typename T, int VEC> union Piece {
  typename Raw<sizeof(T) * VEC>::type raw;
  T e[VEC];
  __device__ __forceinline__ Piece() {}
};
template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
// A piece's values, and back, rounded; two-byte types by pairs.
template <typename T, int VEC> __device__ __forceinline__ void unpack(const Piece<T, VEC>& p, float (&v)[VEC]) {
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) {
      const uint32_t u = ((const uint32_t*)&p.raw)[k / 2];
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*(const __half2*)&u);
        v[k] = f.x;
        v[k + 1] = f.y;
      } else {
        v[k] = __uint_as_float(u << 16);
        v[k + 1] = __uint_as_float(u & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = widen<T>(p.e[k]);
  }
}
template <typename T, int VEC> __device__ __forceinline__ void pack(const float (&v)[VEC], Piece<T, VEC>& p) {
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[k], v[k + 1]);
        ((uint32_t*)&p.raw)[k / 2] = *(const uint32_t*)&h;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[k], v[k + 1]);
        ((uint32_t*)&p.raw)[k / 2] = *(const uint32_t*)&h;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) p.e[k] = narrow<T>(v[k]);
  }
}
// The largest magnitude; a NaN stays one.
template <int VEC> __device__ __forceinline__ float magnitude(const float (&v)[VEC]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int k = 1; k < VEC; ++k) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[k])));
  return m;
}
// Values in 8 bits, to the nearest.  int8: 1.5 * 2^23 more, a number's lowest bits are the whole number (a conversion is issued at a quarter of the rate of
// a sum); `bounded` values are numbers of no more than 127.
template <int VEC> __device__ __forceinline__ void to_int8(float (&v)[VEC], bool bounded, Piece<uint8_t, VEC>& q) {
  if (!bounded) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = fminf(fmaxf(v[k] == v[k] ? v[k] : 0.f, -128.f), 127.f);
  }
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(v[k + e] + 12582912.f);
      ((uint32_t*)&q.raw)[k / 4] = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    }
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) q.e[k] = (uint8_t)(__float_as_uint(v[k] + 12582912.f) & 0xffu);
  }
}
template <int VEC> __device__ __forceinline__ void to_e4m3(const float (&v)[VEC], Piece<uint8_t, VEC>& q) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int k = 0; k < VEC; k += 4)
      ((uint32_t*)&q.raw)[k / 4] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[k], v[k + 1]), __NV_SATFINITE, __NV_E4M3) |
                                   (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[k + 2], v[k + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) q.e[k] = (uint8_t)__nv_cvt_float_to_fp8(v[k], __NV_SATFINITE, __NV_E4M3);
  }
}
template <int VEC> __device__ __forceinline__ void load_weight(const RmsNorm& n, int c, float (&w)[VEC]) {   // of piece c, with the offset
#pragma unroll
  for (int k = 0; k < VEC; ++k) w[k] = 1.f;
  if (n.weight && n.weight_dt == DT_F32) {
    constexpr int W = VEC >= 4 ? 4 : 1;
#pragma unroll
    for (int k = 0; k < VEC; k += W) {
      Piece<float, W> v;
      v.raw = *(const decltype(v.raw)*)((const float*)n.weight + (int64_t)c * VEC + k);
#pragma unroll
      for (int e = 0; e < W; ++e) w[k + e] = v.e[e];
    }
  } else if (n.weight) {
    Piece<uint16_t, VEC> v;
    v.raw = *(const decltype(v.raw)*)((const uint16_t*)n.weight + (int64_t)c * VEC);
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[k] = n.weight_dt == DT_F16 ? __half2float(__ushort_as_half(v.e[k])) : __uint_as_float((uint32_t)v.e[k] << 16);
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) w[k] += n.weight_offset;
}
// What values of a group are multiplied by, for its largest magnitude as a whole number.
__device__ __forceinline__ float inverse_of(uint32_t top, float most) {
  const float inverse = most / __uint_as_float(top);
  if (top == 0 || top >= 0x7f800000u || inverse == INFINITY) return top > 0x7f800000u ? __uint_as_float(top) : 0.f;
  return inverse;
}

// A mean of squares below 2^-90 or beyond fp32 (fp16 has none): the row is multiplied by a power of two that brings the sum of up to 32768 squares into range, epsilon
// likewise, and summed again.  Of a row around 2^56 or more, values below 2^-54 lose bits then, of which less than 2^-126 is left in the result.
template <typename T> __device__ __forceinline__ bool out_of_range(float mean) {
  return !std::is_same<T, __half>::value && __float_as_uint(mean) - 0x12800000u > 0x7f7fffffu - 0x12800000u;
}
__device__ __forceinline__ float into_range(float mean) { return mean < 0x1p-90f ? 0x1p90f : 0x1p-72f; }

struct Params {
  RmsNorm n;
  float per_channel;      // 1 / channels
  int pieces, lanes;      // VEC channels each; threads of a row
  int rows_of_block, step_row, step_head;   // short rows of a block at a time, and what that is in rows and heads
  int group_shift;        // a group is 1 << group_shift pieces of neighbouring threads; -1: the row; -2: any, counted in shared memory; -3: no scales to find
};

// h = round(x + residual), y = h / sqrt(mean(h h) + epsilon) * (w + offset), and y in 8 bits with scales.
// Bound by memory: x and residual are read once and stay in registers (NP pieces of 16 bytes a thread), each result is written once.  Sums of squares
// are 32-bit, by thread, then by warp, then by block.
// Largest magnitudes are compared as whole numbers across threads, which order them and keep a NaN.
// 8191 rows of 5120 fp16 values with residual, sum and int8: 69 us, 5.5 TB/s and three quarters of the issue slots; without the 8 bits 52 us.
// 64 rows of 4096: 2.5 us, a chain of loads, two sums over the block and stores.
// Rows that are no whole pieces of 16 bytes, or lie off them, go element by element: 2048 x 4001 bf16 52 us where 2048 x 4096 take 10 (in L2), 512 x 20001 117 us
// (up to 32 elements a thread, which do not all stay in registers).
template <typename T, int VEC, int NP>
__global__ void __launch_bounds__(NP == 2 ? 512 : kMaxThreads, NP == 2 ? 3 : 1) norm_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint32_t tops[];      // of each group (group_shift -2)
  __shared__ float sums[32];
  __shared__ uint32_t largest[32];
  const RmsNorm& n = p.n;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const unsigned at = blockIdx.x;
  const unsigned row = n.heads == 1 ? at : at / n.heads, head = at - row * n.heads;
  auto place = [&](const void* base, int part) { return (T*)base + (int64_t)row * n.row[part] + (int64_t)head * n.head[part]; };
  float h[NP][VEC];
  float square = 0.f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  {
    Piece<T, VEC> x[NP], r[NP];
    const T *xp = place(n.x, 0), *rp = place(n.residual, 1);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = t + i * p.lanes;
      const bool there = c < p.pieces;
      if (there) x[i].raw = *(const decltype(x[i].raw)*)(xp + (int64_t)c * VEC);
      if (there && n.residual) r[i].raw = *(const decltype(x[i].raw)*)(rp + (int64_t)c * VEC);
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = t + i * p.lanes;
      const bool there = c < p.pieces;
      if (there) {
        unpack<T, VEC>(x[i], h[i]);
        if (n.residual) {
          float v[VEC];
          unpack<T, VEC>(r[i], v);
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[k] += h[i][k];
          pack<T, VEC>(v, x[i]);
          unpack<T, VEC>(x[i], h[i]);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) square += h[i][k] * h[i][k];
      }
      if (there && n.sum) *(decltype(x[i].raw)*)(place(n.sum, 2) + (int64_t)c * VEC) = x[i].raw;
    }
  }
  if (!n.y && !n.quant) return;
#pragma unroll
  for (int o = 16; o; o >>= 1) square += __shfl_xor_sync(~0u, square, o);
  if (lane == 0) sums[warp] = square;
  if (p.group_shift == -2)
    for (int g = threadIdx.x; g < n.channels / n.group; g += blockDim.x) tops[g] = 0;
  __syncthreads();
  square = lane < (int)(blockDim.x >> 5) ? sums[lane] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) square += __shfl_xor_sync(~0u, square, o);
  float mean = square * p.per_channel + n.epsilon;
  if (out_of_range<T>(mean)) {   // (all threads have the same)
    const float by = into_range(mean);
    square = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (t + i * p.lanes < p.pieces) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          h[i][k] *= by;
          square += h[i][k] * h[i][k];
        }
      }
#pragma unroll
    for (int o = 16; o; o >>= 1) square += __shfl_xor_sync(~0u, square, o);
    __syncthreads();   // (the first sums have been read)
    if (lane == 0) sums[warp] = square;
    __syncthreads();
    square = lane < (int)(blockDim.x >> 5) ? sums[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) square += __shfl_xor_sync(~0u, square, o);
    mean = square * p.per_channel + n.epsilon * by * by;
  }
  const float factor = rsqrtf(mean);
  uint32_t top[NP];
  uint32_t row_top = 0;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int c = t + i * p.lanes;
    const bool there = c < p.pieces;
    top[i] = 0;
    if (!there) continue;
    float w[VEC];
    load_weight<VEC>(n, c, w);
    Piece<T, VEC> y;
#pragma unroll
    for (int k = 0; k < VEC; ++k) h[i][k] = h[i][k] * factor * w[k];
    pack<T, VEC>(h[i], y);
    if (n.quant) {
      top[i] = __float_as_uint(magnitude<VEC>(h[i]));
      row_top = max(row_top, top[i]);
    }
    if (n.y) *(decltype(y.raw)*)(place(n.y, 3) + (int64_t)c * VEC) = y.raw;
  }
  if (!n.quant) return;
  const float most = n.quant == 1 ? 127.f : 448.f;
  const int64_t groups = n.group ? n.channels / n.group : 1;
  if (p.group_shift == -1) {
    row_top = __reduce_max_sync(~0u, row_top);
    if (lane == 0) largest[warp] = row_top;
    __syncthreads();
    row_top = __reduce_max_sync(~0u, lane < (int)(blockDim.x >> 5) ? largest[lane] : 0u);
    if (t == 0) n.scales[at] = __uint_as_float(row_top) / most;
  } else if (p.group_shift >= 0) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      for (int o = 1; o < 1 << p.group_shift; o <<= 1) top[i] = max(top[i], __shfl_xor_sync(~0u, top[i], o));
      const int c = t + i * p.lanes;
      if (c < p.pieces && (c & ((1 << p.group_shift) - 1)) == 0) n.scales[at * groups + (c >> p.group_shift)] = __uint_as_float(top[i]) / most;
    }
  } else if (p.group_shift == -2) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = t + i * p.lanes;
      if (c < p.pieces) atomicMax(&tops[c * VEC / n.group], top[i]);
    }
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += blockDim.x) n.scales[at * groups + g] = __uint_as_float(tops[g]) / most;
  }
  const float given = p.group_shift == -3 ? n.scales[0] : 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int c = t + i * p.lanes;
    if (c >= p.pieces) continue;
    float inverse = 0.f;
    uint32_t u = 0xffffffffu;
    if (p.group_shift != -3) {
      u = p.group_shift == -1 ? row_top : p.group_shift == -2 ? tops[c * VEC / n.group] : top[i];
      inverse = inverse_of(u, most);
    }
    Piece<uint8_t, VEC> q;
    float v[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = p.group_shift == -3 ? h[i][k] / given : h[i][k] * inverse;
    if (n.quant == 1) to_int8<VEC>(v, u < 0x7f800000u, q); else to_e4m3<VEC>(v, q);
    *(decltype(q.raw)*)((uint8_t*)n.quantised + (int64_t)row * n.row[4] + (int64_t)head * n.head[4] + (int64_t)c * VEC) = q.raw;
  }
}

// The same for rows of up to 32 pieces (heads): `lanes` threads of a warp have a piece each, of ROWS rows, whose loads are under way together and which
// share the weight (4097 tokens of 32 heads of 128 bf16: 14.8 us out of a graph, three quarters of the issue slots; fp32 29 us).
template <typename T, int VEC, int ROWS>
__global__ void __launch_bounds__(kShortThreads) short_kernel(const __grid_constant__ Params p) {
  const RmsNorm& n = p.n;
  const int c = threadIdx.x & (p.lanes - 1);
  unsigned at = blockIdx.x * (unsigned)(p.rows_of_block * ROWS) + threadIdx.x / p.lanes;
  unsigned row = n.heads == 1 ? at : at / n.heads, head = at - row * n.heads;
  unsigned rows[ROWS], heads[ROWS];
  bool there[ROWS];
  Piece<T, VEC> x[ROWS], r[ROWS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    rows[i] = row;
    heads[i] = head;
    there[i] = at + i * p.rows_of_block < n.total && c < p.pieces;
    if (there[i]) x[i].raw = *(const decltype(x[i].raw)*)((const T*)n.x + (int64_t)row * n.row[0] + (int64_t)head * n.head[0] + c * VEC);
    if (there[i] && n.residual) r[i].raw = *(const decltype(x[i].raw)*)((const T*)n.residual + (int64_t)row * n.row[1] + (int64_t)head * n.head[1] + c * VEC);
    row += p.step_row;
    head += p.step_head;
    if (head >= (unsigned)n.heads) { head -= n.heads; ++row; }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  float w[VEC];
  if (c < p.pieces) load_weight<VEC>(n, c, w);
  const float most = n.quant == 1 ? 127.f : 448.f, given = p.group_shift == -3 ? n.scales[0] : 0.f;
  const int groups = n.group ? n.channels / n.group : 1;
  float h[ROWS][VEC], mean[ROWS];
  bool odd = false;
  auto mean_of = [&](int i, float by) {
    float square = 0.f;
    if (there[i]) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) square += h[i][k] * h[i][k];
    }
    for (int o = p.lanes / 2; o; o >>= 1) square += __shfl_xor_sync(~0u, square, o);
    return square * p.per_channel + n.epsilon * by * by;
  };
  auto place = [&](int i, void* base, int part) { return (T*)base + (int64_t)rows[i] * n.row[part] + (int64_t)heads[i] * n.head[part] + c * VEC; };
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (there[i]) {
      unpack<T, VEC>(x[i], h[i]);
      if (n.residual) {
        float v[VEC];
        unpack<T, VEC>(r[i], v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] += h[i][k];
        pack<T, VEC>(v, x[i]);
        unpack<T, VEC>(x[i], h[i]);
      }
    }
    if (there[i] && n.sum) *(decltype(x[i].raw)*)place(i, n.sum, 2) = x[i].raw;
    mean[i] = mean_of(i, 1.f);
    odd = odd || out_of_range<T>(mean[i]);
  }
  if (__any_sync(~0u, odd)) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const float by = out_of_range<T>(mean[i]) ? into_range(mean[i]) : 1.f;
#pragma unroll
      for (int k = 0; k < VEC; ++k) h[i][k] *= by;
      mean[i] = mean_of(i, by);
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const float factor = rsqrtf(mean[i]);
    Piece<T, VEC> y;
#pragma unroll
    for (int k = 0; k < VEC; ++k) h[i][k] = h[i][k] * factor * w[k];
    pack<T, VEC>(h[i], y);
    if (there[i] && n.y) *(decltype(y.raw)*)place(i, n.y, 3) = y.raw;
    if (!n.quant) continue;
    uint32_t top = there[i] ? __float_as_uint(magnitude<VEC>(h[i])) : 0u;
    float inverse = 0.f;
    if (p.group_shift != -3) {
      const int across = p.group_shift == -1 ? p.lanes : 1 << p.group_shift;
      for (int o = 1; o < across; o <<= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
      inverse = inverse_of(top, most);
      if (there[i] && (c & (across - 1)) == 0) n.scales[(int64_t)(at + i * p.rows_of_block) * groups + c / across] = __uint_as_float(top) / most;
    }
    Piece<uint8_t, VEC> q;
#pragma unroll
    for (int k = 0; k < VEC; ++k) h[i][k] = p.group_shift == -3 ? h[i][k] / given : h[i][k] * inverse;
    if (n.quant == 1) to_int8<VEC>(h[i], p.group_shift != -3 && top < 0x7f800000u, q); else to_e4m3<VEC>(h[i], q);
    if (there[i]) *(decltype(q.raw)*)((uint8_t*)n.quantised + (int64_t)rows[i] * n.row[4] + (int64_t)heads[i] * n.head[4] + c * VEC) = q.raw;
  }
}

template <typename T> int launch(const RmsNorm& n, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  bool wide = n.channels % VEC == 0;
  auto row = [&](const void* p, int part, int bytes) {
    if (p) wide = wide && (uintptr_t)p % bytes == 0 && n.row[part] % VEC == 0 && n.head[part] % VEC == 0;
  };
  row(n.x, 0, 16); row(n.residual, 1, 16); row(n.sum, 2, 16); row(n.y, 3, 16);
  if (n.quant) row(n.quantised, 4, VEC);
  if (n.weight) wide = wide && (uintptr_t)n.weight % (n.weight_dt == DT_F32 ? 16 : 2 * VEC) == 0;
  Params p{};
  p.n = n;
  p.per_channel = 1.f / (float)n.channels;
  const int vec = wide ? VEC : 1;
  p.pieces = n.channels / vec;
  if (n.quant && n.group == 0) p.group_shift = -3;
  else if (!n.quant || n.group == n.channels) p.group_shift = -1;
  else {
    const int of = n.group / vec;
    int shift = 0;
    while (1 << shift < of) ++shift;
    p.group_shift = n.group % vec == 0 && 1 << shift == of && of <= 32 ? shift : -2;
  }
  int threads, each;   // rows of a thread
  void (*fn)(Params);
  if (wide && p.pieces <= kShort && p.group_shift != -2) {
    p.lanes = 1;
    while (p.lanes < p.pieces) p.lanes *= 2;
    threads = kShortThreads;
    p.rows_of_block = threads / p.lanes;
    p.step_row = p.rows_of_block / n.heads;
    p.step_head = p.rows_of_block % n.heads;
    each = n.total / p.rows_of_block >= kMany * kRows ? kRows : 1;
    fn = each == 1 ? short_kernel<T, VEC, 1> : short_kernel<T, VEC, kRows>;
  } else {
    // one piece for each thread, up to 1024; two where rows are many, so that more of them are under way (rows of 4096 bf16 with
    // a residual and e4m3, one and two: 64 rows 2.5 and 2.8 us, 512 5.0 and 5.7, 1024 7.8 both, 2048 17.0 and 14.2)
    p.rows_of_block = 1;
    const int wanted = wide && n.total >= kMany ? (p.pieces + kEach - 1) / kEach : p.pieces;
    threads = std::max(64, std::min(kMaxThreads, (wanted + 31) / 32 * 32));
    p.lanes = threads;
    const int pieces = (p.pieces + threads - 1) / threads;
    if (!wide) fn = pieces <= 8 ? norm_kernel<T, 1, 8> : norm_kernel<T, 1, 32>;
    else if (pieces == 1) fn = norm_kernel<T, VEC, 1>;
    else if (pieces == 2 && threads <= 512) fn = norm_kernel<T, VEC, 2>;
    else if (pieces <= 4) fn = norm_kernel<T, VEC, 4>;
    else fn = norm_kernel<T, VEC, VEC == 4 ? 8 : 4>;   // (32768 channels of two bytes are four pieces for each of 1024 threads)
    each = 1;
  }
  const size_t smem = p.group_shift == -2 ? sizeof(uint32_t) * (size_t)(n.channels / n.group) : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((n.total + p.rows_of_block * each - 1) / (p.rows_of_block * each));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, fn, p) == cudaSuccess) return 0;
  cudaGetLastError();
  return -2;
}

}  // namespace

int rms_norm(const RmsNorm& n, cudaStream_t stream) {
  switch (n.dt) {
    case DT_F32: return launch<float>(n, stream);
    case DT_F16: return launch<__half>(n, stream);
    case DT_BF16: return launch<__nv_bfloat16>(n, stream);
  }
  return -1;
}

}  // namespace b200
