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

// Where one (token, head) row comes from and goes to, or no destination.
template <typename T> __device__ __forceinline__ bool row_of(const TurnGeom& g, int token, int head, const T*& src, T*& dst) {
  const int part = head < g.heads ? 0 : head < g.heads + g.kv_heads ? 1 : 2;
  if (part == 0) {
    const int b = g.batch > 1 ? token / g.tokens : 0, t = token - b * g.tokens;
    src = (const T*)g.src[0] + (int64_t)b * g.s_batch + (int64_t)t * g.s_token[0] + (int64_t)head * g.s_head[0];
    dst = (T*)g.dst[0] + (int64_t)b * g.d_batch + (int64_t)t * g.d_token + (int64_t)head * g.d_head;
    return true;
  }
  const int64_t slot = g.slots[token];
  if (slot < 0 || slot >= (int64_t)g.pages * g.page_size) return false;
  const int64_t page = slot / g.page_size, at = slot - page * g.page_size;
  const int h = head - g.heads - (part - 1) * g.kv_heads;
  src = (const T*)g.src[part] + (int64_t)token * g.s_token[part] + (int64_t)h * g.s_head[part];
  dst = (T*)g.dst[part] + page * g.c_page + at * g.c_token + (int64_t)h * g.c_head;
  return true;
}

// (a, b) -> (a cos - b sin, a sin + b cos), t = position * frequency.  Bound by memory: every row is read and written once.
//
// Angles.  A frequency arrives as turns per position in units of 2^-64 (host: turn_units), so that position * frequency modulo 2^64
// is the angle modulo one turn, exactly, however far the position: no reduction in floating point, whose error grows with
// it.  The nearest quarter turn is taken off as whole numbers; what is left, at most an eighth, becomes fp32 with a relative error
// of 2^-24.  A block computes cosine and sine once for its tokens and uses them for every head.
//
// A thread takes 2 * VEC channels of a row at a time: VEC pairs, or, past the pairs, channels that are copied.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) turn_kernel(const __grid_constant__ TurnGeom g, const int block_tokens) {
  extern __shared__ float2 cs[];   // [block_tokens][pairs]
  const int total = g.batch * g.tokens, first = blockIdx.x * block_tokens, n_tok = min(block_tokens, total - first);
  if (g.pairs > 0) {
    const int groups = kThreads / g.pairs, p = threadIdx.x % g.pairs;
    if ((int)threadIdx.x < groups * g.pairs) {
      const uint64_t f = g.frequency[p];
      const int* pos = g.positions + (int64_t)g.axis[p] * total + first;
      for (int t = threadIdx.x / g.pairs; t < n_tok; t += groups) {
        const uint32_t phase = (uint32_t)(((uint64_t)(int64_t)pos[t] * f) >> 32);
        const uint32_t quarter = (phase + 0x20000000u) >> 30;
        float s, c;
        sincospif((float)(int)(phase - (quarter << 30)) * (1.0f / 2147483648.0f), &s, &c);
        cs[t * g.pairs + p] = quarter == 0 ? make_float2(c, s) : quarter == 1 ? make_float2(-s, c) : quarter == 2 ? make_float2(-c, -s) : make_float2(s, -c);
      }
    }
    __syncthreads();
  }
  const int per_row = (g.channels + 2 * VEC - 1) / (2 * VEC), turning = g.pairs / VEC, heads = g.heads + 2 * g.kv_heads;
  const int tasks = n_tok * heads * per_row;
  for (int i = threadIdx.x; i < tasks; i += kThreads) {
    const int r = i / per_row, c = i - r * per_row;
    int t, h;
    if (g.heads_outside) { h = r / n_tok; t = r - h * n_tok; } else { t = r / heads; h = r - t * heads; }
    const T* src;
    T* dst;
    if (!row_of<T>(g, first + t, h, src, dst)) continue;
    if (c < turning && h < g.heads + g.kv_heads) {
      const float2* angle = cs + t * g.pairs + c * VEC;
      const int at = INTERLEAVED ? c * 2 * VEC : c * VEC, step = INTERLEAVED ? VEC : g.pairs;
      Piece<T, VEC> x[2] = {load<T, VEC>(src + at), load<T, VEC>(src + at + step)}, y[2];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float2 w = angle[k];
        // pair k: elements 2k, 2k + 1 of the two pieces, or element k of each
        const int p0 = INTERLEAVED ? 2 * k / VEC : 0, e0 = INTERLEAVED ? 2 * k % VEC : k, p1 = INTERLEAVED ? (2 * k + 1) / VEC : 1, e1 = INTERLEAVED ? (2 * k + 1) % VEC : k;
        const float a = widen<T>(x[p0].e[e0]), b = widen<T>(x[p1].e[e1]);
        y[p0].e[e0] = narrow<T>(a * w.x - b * w.y);
        y[p1].e[e1] = narrow<T>(a * w.y + b * w.x);
      }
      store<T, VEC>(dst + at, y[0]);
      store<T, VEC>(dst + at + step, y[1]);
    } else {
      const int at = c * 2 * VEC;
      if (src == dst) continue;
      store<T, VEC>(dst + at, load<T, VEC>(src + at));
      if (VEC > 1 || at + 1 < g.channels) store<T, VEC>(dst + at + VEC, load<T, VEC>(src + at + VEC));
    }
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
  const int64_t total = (int64_t)g.batch * g.tokens;
  int block_tokens = 16;
  while (block_tokens > 1 && (total + block_tokens - 1) / block_tokens < 4 * 148) block_tokens /= 2;
  const int64_t blocks = (total + block_tokens - 1) / block_tokens;
  const size_t smem = sizeof(float2) * (size_t)block_tokens * (size_t)g.pairs;
  auto* fn = wide ? (g.interleaved ? turn_kernel<T, VEC, true> : turn_kernel<T, VEC, false>) : (g.interleaved ? turn_kernel<T, 1, true> : turn_kernel<T, 1, false>);
  fn<<<(unsigned)blocks, kThreads, smem, stream>>>(g, block_tokens);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
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
