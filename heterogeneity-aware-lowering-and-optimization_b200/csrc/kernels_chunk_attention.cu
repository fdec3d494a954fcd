// Attention of the new tokens of each sequence of a batch over a paged cache.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>

#include "kernels.h"

namespace b200 {
namespace {

constexpr int kWarps = 8;

template <typename T> __device__ __forceinline__ float2 widen2(uint32_t u);
template <> __device__ __forceinline__ float2 widen2<__half>(uint32_t u) { return __half22float2(*(const __half2*)&u); }
template <> __device__ __forceinline__ float2 widen2<__nv_bfloat16>(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
template <typename T> __device__ __forceinline__ uint32_t narrow2(float x, float y);
template <> __device__ __forceinline__ uint32_t narrow2<__half>(float x, float y) { const __half2 h = __floats2half2_rn(x, y); return *(const uint32_t*)&h; }
template <> __device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(float x, float y) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *(const uint32_t*)&h; }

// A warp for each row (token, query head): a position after the other, each lane with D / 32 channels.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) row_kernel(const __grid_constant__ ChunkAttention a) {
  constexpr int N = D / 64;   // pairs of channels
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (id >= (int64_t)a.tokens * a.heads) return;
  const int row = (int)(id / a.heads), head = (int)(id - (int64_t)row * a.heads), kv = head / (a.heads / a.kv_heads);
  if (row < a.starts[0] || row >= a.starts[a.batch]) return;
  int lo = 0, hi = a.batch;   // starts[lo] <= row < starts[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) / 2;
    if (a.starts[m] <= row) lo = m; else hi = m;
  }
  const int count = a.starts[hi] - a.starts[lo];
  const int length = (int)min((long long)max(a.lengths[lo], 0), (long long)a.table_width * a.page_size);
  const int sees = a.prefix_length + max(0, length - count + (row - a.starts[lo]) + 1);
  float2 q[N], acc[N];
  const uint32_t* qp = (const uint32_t*)((const T*)a.q + row * a.q_token + head * a.q_head) + lane * N;
#pragma unroll
  for (int k = 0; k < N; ++k) { q[k] = widen2<T>(qp[k]); acc[k] = make_float2(0.f, 0.f); }
  float top = -INFINITY, sum = 0.f;
  for (int at = 0; at < sees; ++at) {
    const int own = at - a.prefix_length, i = own < 0 ? at : own;
    const int page = own < 0 ? a.prefix_pages[i / a.page_size] : a.page_table[(int64_t)lo * a.table_width + i / a.page_size];
    if (page < 0 || page >= a.pages) continue;
    const int64_t off = page * a.c_page + (int64_t)(i % a.page_size) * a.c_token + kv * a.c_head;
    const uint32_t *kp = (const uint32_t*)((const T*)a.k + off) + lane * N, *vp = (const uint32_t*)((const T*)a.v + off) + lane * N;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) { const float2 x = widen2<T>(kp[k]); s += q[k].x * x.x + q[k].y * x.y; }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    s *= a.scale;
    if (s == -INFINITY) continue;
    const float next = fmaxf(top, s), corr = expf(top - next), w = expf(s - next);
    top = next;
    sum = sum * corr + w;
#pragma unroll
    for (int k = 0; k < N; ++k) { const float2 v = widen2<T>(vp[k]); acc[k].x = acc[k].x * corr + w * v.x; acc[k].y = acc[k].y * corr + w * v.y; }
  }
  uint32_t* y = (uint32_t*)((T*)a.y + row * a.y_token + head * a.y_head) + lane * N;
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int k = 0; k < N; ++k) y[k] = narrow2<T>(acc[k].x * inverse, acc[k].y * inverse);
}

template <typename T, int D> int launch(const ChunkAttention& a, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((int64_t)a.tokens * a.heads + kWarps - 1) / kWarps));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, row_kernel<T, D>, a) == cudaSuccess) return 0;
  cudaGetLastError();
  return -2;
}

}  // namespace

int chunk_attention(const ChunkAttention& a, cudaStream_t stream) {
  if (a.dt == DT_F16) return a.channels == 64 ? launch<__half, 64>(a, stream) : launch<__half, 128>(a, stream);
  return a.channels == 64 ? launch<__nv_bfloat16, 64>(a, stream) : launch<__nv_bfloat16, 128>(a, stream);
}

}  // namespace b200
