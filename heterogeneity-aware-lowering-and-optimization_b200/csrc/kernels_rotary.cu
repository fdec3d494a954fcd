// Positions that turn pairs of channels, and the same on the way into a paged cache.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"

namespace b200 {
namespace {

constexpr int kThreads = 256;

struct alignas(16) Sixteen { uint32_t w[4]; };
template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements at once: 16 bytes, or one element where pointers, strides or sizes are no multiples of 16 bytes.
template <typename T, int VEC> struct Piece { T e[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ Piece<T, VEC> load(const T* p) {
  Piece<T, VEC> v;
  if constexpr (VEC > 1) *(Sixteen*)v.e = *(const Sixteen*)p; else v.e[0] = *p;
  return v;
}
template <typename T, int VEC> __device__ __forceinline__ void store(T* p, const Piece<T, VEC>& v) {
  if constexpr (VEC > 1) *(Sixteen*)p = *(const Sixteen*)v.e; else *p = v.e[0];
}

// (a, b) -> (a cos - b sin, a sin + b cos), t = position * frequency.  Bound by memory: every row is read and written once.
//
// Angles.  A frequency arrives as turns per position in units of 2^-64 (host: turn_units), so that position * frequency modulo 2^64
// is the angle modulo one turn, exactly, however far the position: no reduction in floating point, whose error grows with
// it.  The nearest quarter turn is taken off as whole numbers of 64 bits; what is left, at most an eighth, becomes fp32 with a relative error
// of 2^-24, beside that of the frequency's own rounding, |position| * 2^-65 turns.  (Its upper 32 bits alone, 2^-32 of a turn, would leave the sine of
// 1e-4 sixteen bits.)
//
// A block takes a few tokens and works out their cosines and sines once, for all heads, into shared memory (in planes of four values, so that
// the pieces of a row read them without bank conflicts); the first rows are already on their way then.  A thread has one
// piece of a row, 2 * VEC channels (VEC pairs, or, past the pairs, channels that are copied), and walks over rows.  Many threads with one row each in
// flight do better than fewer with more: 40 registers and six blocks per SM move 2 x 12288 x 16 rows of 128 channels (201 MB) in
// 41 us, 4.9 TB/s; two rows ahead in 64 registers take 43 us, four 66 us; angles kept in registers, a thread for one token, 59 us.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(VEC == 1 ? 2 * kThreads : kThreads, VEC == 1 ? 2 : 6) turn_kernel(const __grid_constant__ TurnGeom g, const int block_tokens, const int per_row) {
  extern __shared__ float4 planes[];   // [cosine, sine][(VEC + 3) / 4][block_tokens][pairs / VEC], four pairs each (one where VEC is 1)
  constexpr int kPlanes = (VEC + 3) / 4, kEach = VEC < 4 ? 1 : 4;
  const int total = g.batch * g.tokens, first = blockIdx.x * block_tokens, n_tok = min(block_tokens, total - first);
  const int pieces = g.pairs / VEC, plane = block_tokens * pieces;
  const int lanes = (int)blockDim.x / per_row, mine = threadIdx.x / per_row, c = threadIdx.x - mine * per_row;   // rows at once, which of them, which piece
  const int heads = g.heads + 2 * g.kv_heads, inner = g.heads_outside ? n_tok : heads, rows = n_tok * heads;
  const int d_inner = lanes % inner, d_outer = lanes / inner;
  const bool turns = c < pieces;
  int r = mine, in = r % inner, out = r / inner;   // row r is (out, in) = (head, token) or (token, head)
  int left = mine < lanes && mine < rows ? (rows - mine + lanes - 1) / lanes : 0;   // this thread's rows
  if (left == 0) r = rows;

  struct Row {
    const T* src;
    T* dst;
    int at, step, token;
    bool any, turn, second;
    Piece<T, VEC> x[2];
  };
  auto fetch = [&](Row& w) {
    w.any = r < rows;
    if (w.any) {
      const int h = g.heads_outside ? out : in, tl = g.heads_outside ? in : out, t = first + tl;
      w.token = tl;
      w.turn = turns && h < g.heads + g.kv_heads;
      w.at = w.turn && !INTERLEAVED ? c * VEC : c * 2 * VEC;
      w.step = w.turn && !INTERLEAVED ? g.pairs : VEC;
      w.second = VEC > 1 || w.at + w.step < g.channels;
      if (h < g.heads) {
        const int b = g.batch > 1 ? t / g.tokens : 0, tb = t - b * g.tokens;
        w.src = (const T*)g.src[0] + (int64_t)b * g.s_batch + (int64_t)tb * g.s_token[0] + (int64_t)h * g.s_head[0];
        w.dst = (T*)g.dst[0] + (int64_t)b * g.d_batch + (int64_t)tb * g.d_token + (int64_t)h * g.d_head;
      } else {
        const int64_t slot = g.slots[t];
        w.any = slot >= 0 && slot < (int64_t)g.pages * g.page_size;
        if (w.any) {
          const int part = h < g.heads + g.kv_heads ? 1 : 2, hk = h - g.heads - (part - 1) * g.kv_heads;
          const int64_t page = slot / g.page_size;
          w.src = (const T*)g.src[part] + (int64_t)t * g.s_token[part] + (int64_t)hk * g.s_head[part];
          w.dst = (T*)g.dst[part] + page * g.c_page + (slot - page * g.page_size) * g.c_token + (int64_t)hk * g.c_head;
        }
      }
      if (w.any) {
        w.x[0] = load<T, VEC>(w.src + w.at);
        if (w.second) w.x[1] = load<T, VEC>(w.src + w.at + w.step);
      }
    }
    r += lanes;
    in += d_inner;
    out += d_outer;
    if (in >= inner) { in -= inner; ++out; }
  };
  auto finish = [&](Row& w) {
    if (!w.any) return;
    if (w.turn) {
      float cs[VEC], sn[VEC];
      if constexpr (VEC == 1) {
        const float* angle = (const float*)planes;
        cs[0] = angle[w.token * pieces + c];
        sn[0] = angle[plane + w.token * pieces + c];
      } else {
#pragma unroll
        for (int k = 0; k < kPlanes; ++k) {
          const float4 x = planes[k * plane + w.token * pieces + c], y = planes[(kPlanes + k) * plane + w.token * pieces + c];
          cs[4 * k] = x.x; cs[4 * k + 1] = x.y; cs[4 * k + 2] = x.z; cs[4 * k + 3] = x.w;
          sn[4 * k] = y.x; sn[4 * k + 1] = y.y; sn[4 * k + 2] = y.z; sn[4 * k + 3] = y.w;
        }
      }
      Piece<T, VEC> y[2];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        // pair k: elements 2k, 2k + 1 of the two pieces, or element k of each
        const int p0 = INTERLEAVED ? 2 * k / VEC : 0, e0 = INTERLEAVED ? 2 * k % VEC : k, p1 = INTERLEAVED ? (2 * k + 1) / VEC : 1, e1 = INTERLEAVED ? (2 * k + 1) % VEC : k;
        const float a = widen<T>(w.x[p0].e[e0]), d = widen<T>(w.x[p1].e[e1]);
        y[p0].e[e0] = narrow<T>(a * cs[k] - d * sn[k]);
        y[p1].e[e1] = narrow<T>(a * sn[k] + d * cs[k]);
      }
      w.x[0] = y[0];
      w.x[1] = y[1];
    }
    store<T, VEC>(w.dst + w.at, w.x[0]);
    if (w.second) store<T, VEC>(w.dst + w.at + w.step, w.x[1]);
  };

  asm volatile("griddepcontrol.wait;" ::: "memory");   // (launched while the kernel in front may still be writing what this one reads)
  Row now;
  fetch(now);
  if (g.pairs > 0) {
    const int groups = (int)blockDim.x / g.pairs, p = threadIdx.x % g.pairs;
    if ((int)threadIdx.x < groups * g.pairs) {
      const uint64_t f = g.frequency[p];
      const int* pos = g.positions + (int64_t)g.axis[p] * total + first;
      float* to = (float*)planes + (p % VEC / kEach * plane + p / VEC) * kEach + p % kEach;
      for (int t = threadIdx.x / g.pairs; t < n_tok; t += groups) {
        const uint64_t phase = (uint64_t)(int64_t)pos[t] * f;
        const uint32_t quarter = ((uint32_t)(phase >> 32) + 0x20000000u) >> 30;
        float sine, cosine;
        sincospif((float)(int64_t)(phase - ((uint64_t)quarter << 62)) * 0x1p-63f, &sine, &cosine);
        const float x = (quarter & 1) ? sine : cosine, y = (quarter & 1) ? cosine : sine;
        to[t * pieces * kEach] = quarter == 1 || quarter == 2 ? -x : x;
        to[(kPlanes * plane + t * pieces) * kEach] = quarter >= 2 ? -y : y;
      }
    }
    __syncthreads();
  }
  for (; left > 0; --left) {
    finish(now);
    fetch(now);
  }
}

template <typename T> int launch(const TurnGeom& g, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  bool wide = g.pairs % VEC == 0 && g.channels % (2 * VEC) == 0;
  auto row = [&](const void* p, std::initializer_list<int64_t> strides) {
    wide = wide && (uintptr_t)p % 16 == 0;
    for (int64_t s : strides) wide = wide && s % VEC == 0;
  };
  if (g.heads) { row(g.src[0], {g.s_batch, g.s_token[0], g.s_head[0]}); row(g.dst[0], {g.d_batch, g.d_token, g.d_head}); }
  for (int i = 1; i < 3 && g.kv_heads; ++i) { row(g.src[i], {g.s_token[i], g.s_head[i]}); row(g.dst[i], {g.c_page, g.c_token, g.c_head}); }
  const int vec = wide ? VEC : 1, per_row = (g.channels + 2 * vec - 1) / (2 * vec);
  const int threads = per_row > kThreads ? 2 * kThreads : kThreads;   // (1024 channels, two at a time, are 512 pieces)
  const int64_t total = (int64_t)g.batch * g.tokens;
  // Four rows for each thread pay for a block's angles (two: 47 us instead of 41 for 16 heads, eight: 45 instead of 39 for 48); fewer where SMs
  // would have less than four blocks.
  const int per_token = (g.heads + 2 * g.kv_heads) * per_row;
  int block_tokens = 16;
  while (block_tokens > 1 && block_tokens * per_token > 4 * threads) block_tokens /= 2;
  while (block_tokens > 1 && (total + block_tokens - 1) / block_tokens < 4 * 148) block_tokens /= 2;
  const int64_t blocks = (total + block_tokens - 1) / block_tokens;
  const size_t smem = 2 * sizeof(float) * (size_t)block_tokens * (size_t)g.pairs;
  auto* fn = wide ? (g.interleaved ? turn_kernel<T, VEC, true> : turn_kernel<T, VEC, false>) : (g.interleaved ? turn_kernel<T, 1, true> : turn_kernel<T, 1, false>);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, fn, g, block_tokens, per_row) == cudaSuccess) return 0;
  cudaGetLastError();
  return -2;
}

}  // namespace

int turn_rows(const TurnGeom& g, int dt, cudaStream_t stream) {
  if ((int64_t)g.batch * g.tokens <= 0 || g.heads + g.kv_heads == 0) return 0;
  switch (dt) {
    case DT_F32: return launch<float>(g, stream);
    case DT_F16: return launch<__half>(g, stream);
    case DT_BF16: return launch<__nv_bfloat16>(g, stream);
  }
  return -1;
}

}  // namespace b200
