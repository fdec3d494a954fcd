// Log probabilities of given tokens, entropy and the likeliest alternatives, from logits.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "kernels.h"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kBatch = 4;       // 16-byte pieces that a thread has in flight, whose largest logit it remembers
constexpr int kCandidates = 2048;               // logits that may be sorted for the alternatives
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
  LogProbs l;
  int share;        // CTAs (a cluster) that share a row
  int batches;      // of a thread, at most
};

// What a row's CTA says to the others: sums relative to its own maximum, its best logits.
struct Shared {
  float top, sum, mean;                         // largest logit; sum of w; sum of w log2 w
  int found;                                    // its alternatives
  float best[kMaxTop];
  int best_at[kMaxTop];
  float red[3][kThreads / 32];
  int count, above, kept;
  uint32_t bins[256], key;
  float candidate[kCandidates];
  int candidate_at[kCandidates];
};

template <typename T> struct alignas(16) Sixteen { T e[16 / sizeof(T)]; };
template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float exp2_fast(float x) {
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
  return x;
}
// Whole numbers in the order of the floats; minus infinity, and NaN, which counts as that, are 0.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float below_infinity(float v) { return fminf(v, FLT_MAX); }

// A row's slice: pieces lo ... hi - 1 of 16 aligned bytes, the first and last of the row perhaps partly outside it.
template <typename T> struct Slice {
  static constexpr int VEC = 16 / sizeof(T);
  const T* row;       // (logit 0)
  int off, vocab, lo, hi;
  __device__ __forceinline__ int first(int piece) const { return piece * VEC - off; }   // index of its first logit
  __device__ __forceinline__ void load(int piece, float (&v)[VEC]) const {
    const int i = first(piece);
    if (piece < hi && i >= 0 && i + VEC <= vocab) {
      const Sixteen<T> x = *(const Sixteen<T>*)(row + i);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = widen<T>(x.e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = piece < hi && i + k >= 0 && i + k < vocab ? widen<T>(row[i + k]) : -INFINITY;
    }
  }
};

__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
  for (int o = kThreads / 64; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
  for (int o = kThreads / 64; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The n largest logits of a slice where more than kCandidates are no smaller than the bound (long runs of equal logits): the n-th largest key bit
// by bit (eight at a time, over the slice again), then all above it, then as many of its equals, in the order of their index.
template <typename T> __device__ __noinline__ void gather_exactly(const Slice<T>& s, int n, Shared& w) {
  constexpr int VEC = Slice<T>::VEC;
  uint32_t prefix = 0;
  int left = n;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) w.bins[i] = 0;
    __syncthreads();
    for (int p = s.lo + threadIdx.x; p < s.hi; p += kThreads) {
      float v[VEC];
      s.load(p, v);
      for (int k = 0; k < VEC; ++k) {
        const uint32_t key = key_of(v[k]);
        if (key && (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8))) atomicAdd(&w.bins[key >> shift & 255], 1);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int bin = 255, more = left;
      while (bin > 0 && (int)w.bins[bin] < more) more -= w.bins[bin--];
      w.key = prefix | (uint32_t)bin << shift;
      w.above = more;
    }
    __syncthreads();
    prefix = w.key;
    left = w.above;
  }
  // `left` equals of the key `prefix` are wanted
  if (threadIdx.x == 0) { w.count = 0; w.kept = 0; }
  __syncthreads();
  for (int base = s.lo; base < s.hi; base += kThreads) {
    const int p = base + threadIdx.x;
    float v[VEC];
    s.load(p, v);
    int equal = 0;
    for (int k = 0; k < VEC; ++k) {
      const uint32_t key = key_of(v[k]);
      if (key > prefix) {
        const int at = atomicAdd(&w.count, 1);
        if (at < kCandidates) { w.candidate[at] = v[k]; w.candidate_at[at] = s.first(p) + k; }
      }
      equal += key == prefix && key;
    }
    // equals in front of this thread's, in this turn and in those before
    int before = equal;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) w.bins[warp] = before;
    __syncthreads();
    before -= equal;
    int all = 0;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) before += w.bins[i];
      all += w.bins[i];
    }
    const int kept = w.kept;
    before += kept;
    for (int k = 0; k < VEC; ++k)
      if (key_of(v[k]) == prefix && prefix && before++ < left) {
        const int at = atomicAdd(&w.count, 1);
        if (at < kCandidates) { w.candidate[at] = v[k]; w.candidate_at[at] = s.first(p) + k; }
      }
    __syncthreads();
    if (threadIdx.x == 0) w.kept = kept + all;
    __syncthreads();
  }
}

// One pass over a row's logits: each thread keeps its largest one and, relative to it, the sums of w = 2^t and of w t, t = (l - max) / T in
// base 2; then threads, and the CTAs that share the row, are put together.
// Alternatives: the n-th largest of the threads' maxima is no larger than the n-th largest logit, so that only logits from there on can be among the n; they
// are few, and are found again through the remembered maximum of each batch of pieces.
template <typename T>
__global__ void __launch_bounds__(kThreads) log_probs_kernel(const __grid_constant__ Params p) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ float group_top[];      // [batches][threads]
  __shared__ Shared w;
  const LogProbs& l = p.l;
  const int t = threadIdx.x, rank = blockIdx.x % p.share;
  const int64_t r = blockIdx.x / p.share;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Slice<T> s;
  s.row = (const T*)l.logits + r * l.row;
  s.off = (int)((uintptr_t)s.row % 16 / sizeof(T));
  s.vocab = l.vocab;
  const int pieces = (s.off + l.vocab + VEC - 1) / VEC, each = (pieces + p.share - 1) / p.share;
  s.lo = min(pieces, rank * each);
  s.hi = min(pieces, s.lo + each);
  const float temperature = l.temperature ? l.temperature[r] : 1.f, T1 = temperature > 0.f ? temperature : 1.f;
  const float k2 = fminf(kLog2e / T1, FLT_MAX);

  float top = -INFINITY, sum = 0.f, mean = 0.f;
  for (int b = 0; b < p.batches; ++b) {
    const int piece = s.lo + b * (kThreads * kBatch) + t;
    if (s.lo + b * (kThreads * kBatch) >= s.hi) break;
    float v[kBatch][VEC];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) s.load(piece + j * kThreads, v[j]);
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) mx = fmaxf(mx, v[j][k]);
    if (l.top) group_top[b * kThreads + t] = mx;
    if (mx > below_infinity(top)) {     // (infinities share all probability: each counts as the largest number)
      if (mx == INFINITY) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[j][k] = v[j][k] == INFINITY ? FLT_MAX : v[j][k];
      }
      if (top > -INFINITY) {
        const float shift = fmaxf((below_infinity(top) - below_infinity(mx)) * k2, -200.f), f = exp2_fast(shift);
        mean = f * (mean + shift * sum);
        sum *= f;
      }
      top = mx;
    }
    const float base = below_infinity(top);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float x = fmaxf((v[j][k] - base) * k2, -150.f), e = exp2_fast(x);   // (2^-150 is 0; NaN becomes that, too)
        sum += e;
        mean += e * x;
      }
  }
  // ---- the block's, then the row's ----
  const float block_top = block_max(top, w.red[0]);
  {
    const float shift = top > -INFINITY ? fmaxf((below_infinity(top) - below_infinity(block_top)) * k2, -200.f) : 0.f, f = exp2_fast(shift);
    mean = f * (mean + shift * sum);
    sum *= f;
  }
  sum = block_sum(sum, w.red[1]);
  mean = block_sum(mean, w.red[2]);
  if (t == 0) { w.top = block_top; w.sum = sum; w.mean = mean; w.found = 0; w.count = 0; }
  __syncthreads();
  if (l.top) {
    // the n-th largest of the threads' maxima, bit by bit
    const uint32_t key = key_of(top);
    uint32_t bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t next = bound | 1u << bit;
      if (__syncthreads_count(key >= next) >= l.top) bound = next;
    }
    bound = max(bound, 1u);      // (0: logits of probability 0)
    if (key >= bound)
      for (int b = 0; b < p.batches; ++b) {
        const int piece = s.lo + b * (kThreads * kBatch) + t;
        if (piece >= s.hi) break;
        if (key_of(group_top[b * kThreads + t]) < bound) continue;
        for (int j = 0; j < kBatch; ++j) {
          float v[VEC];
          s.load(piece + j * kThreads, v);
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            if (key_of(v[k]) >= bound) {
              const int at = atomicAdd(&w.count, 1);
              if (at < kCandidates) { w.candidate[at] = v[k]; w.candidate_at[at] = s.first(piece + j * kThreads) + k; }
            }
        }
      }
    __syncthreads();
    if (w.count > kCandidates) gather_exactly(s, l.top, w);
    __syncthreads();
    const int n = min(w.count, kCandidates);
    for (int c = t; c < n; c += kThreads) {
      const uint32_t mine = key_of(w.candidate[c]);
      const int at = w.candidate_at[c];
      int place = 0;
      for (int i = 0; i < n; ++i) {
        const uint32_t other = key_of(w.candidate[i]);
        place += other > mine || (other == mine && w.candidate_at[i] < at);
      }
      if (place < l.top) { w.best[place] = w.candidate[c]; w.best_at[place] = at; }
    }
    if (t == 0) w.found = min(n, l.top);
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (p.share > 1) cluster.sync(); else __syncthreads();
  if (rank == 0) {
    float row_top = -INFINITY, row_sum = 0.f, row_mean = 0.f;
    for (int i = 0; i < p.share; ++i) row_top = fmaxf(row_top, p.share > 1 ? cluster.map_shared_rank(&w, i)->top : w.top);
    const float base = below_infinity(row_top);
    for (int i = 0; i < p.share; ++i) {
      const Shared* o = p.share > 1 ? cluster.map_shared_rank(&w, i) : &w;
      const float shift = o->top > -INFINITY ? fmaxf((below_infinity(o->top) - base) * k2, -200.f) : 0.f, f = exp2_fast(shift);
      row_mean += f * (o->mean + shift * o->sum);
      row_sum += f * o->sum;
    }
    const float log_sum = logf(row_sum);
    auto log_prob = [&](float v) {
      if (!(v > -INFINITY) || (row_top == INFINITY && v < INFINITY)) return -INFINITY;
      return (below_infinity(v) - base) / T1 - log_sum;
    };
    if (t == 0 && l.entropy) l.entropy[r] = row_sum > 0.f ? log_sum - kLn2 * row_mean / row_sum : 0.f;
    for (int i = t; i < l.given; i += kThreads) {
      const int token = l.tokens[r * l.given + i];
      l.token_log_probs[r * l.given + i] = token >= 0 && token < l.vocab ? log_prob(widen<T>(s.row[token])) : -INFINITY;
    }
    // the CTAs' alternatives, each in order: a place is the number of those in front
    int all = 0;
    for (int i = 0; i < p.share; ++i) all += p.share > 1 ? cluster.map_shared_rank(&w, i)->found : w.found;
    for (int c = t; c < p.share * l.top; c += kThreads) {
      const int i = c / l.top, k = c - i * l.top;
      const Shared* o = p.share > 1 ? cluster.map_shared_rank(&w, i) : &w;
      if (k >= o->found) continue;
      const float v = o->best[k];
      const uint32_t mine = key_of(v);
      int place = k;
      for (int j = 0; j < p.share; ++j) {
        if (j == i) continue;
        const Shared* q = cluster.map_shared_rank(&w, j);
        for (int m = 0; m < q->found; ++m) {
          const uint32_t other = key_of(q->best[m]);
          if (other > mine || (other == mine && j < i)) ++place; else break;
        }
      }
      if (place < l.top) { l.top_tokens[r * l.top + place] = o->best_at[k]; l.top_log_probs[r * l.top + place] = log_prob(v); }
    }
    for (int k = all + t; k < l.top; k += kThreads) { l.top_tokens[r * l.top + k] = -1; l.top_log_probs[r * l.top + k] = -INFINITY; }
  }
  if (p.share > 1) cluster.sync();   // (what the others read stays until they have)
}

template <typename T> int launch(const LogProbs& l, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  Params p{};
  p.l = l;
  const int pieces = (l.vocab + VEC - 1) / VEC + 1;
  p.share = 1;
  while (p.share < 8 && l.rows * p.share < 148 && pieces / p.share > 2 * kThreads) p.share *= 2;
  p.batches = ((pieces + p.share - 1) / p.share + kThreads * kBatch - 1) / (kThreads * kBatch);
  const size_t smem = l.top ? sizeof(float) * (size_t)p.batches * kThreads : 0;
  auto* fn = log_probs_kernel<T>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024) != cudaSuccess) { cudaGetLastError(); return -2; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(l.rows * p.share));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.share;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, fn, p) == cudaSuccess) return 0;
  cudaGetLastError();
  return -2;
}

}  // namespace

int log_probs(const LogProbs& l, cudaStream_t stream) {
  switch (l.dt) {
    case DT_F32: return launch<float>(l, stream);
    case DT_F16: return launch<__half>(l, stream);
    case DT_BF16: return launch<__nv_bfloat16>(l, stream);
  }
  return -1;
}

}  // namespace b200
