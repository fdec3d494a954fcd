// Log probabilities of given tokens, entropy and the likeliest alternatives, from logits.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "kernels.h"
#include "per_device.h"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kBatch = 4;       // 16-byte pieces that a thread has in flight, whose largest logit it remembers
constexpr size_t kMostSmem = 96 * 1024;         // for the batches' largest logits: 33 KB for 262144 of four bytes
constexpr int kHits = 512;                      // batches that may hold some of them
constexpr int kCandidates = 1024;               // logits that may be sorted for the alternatives
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
  LogProbs l;
  int share;        // CTAs (a cluster) that share a row
  int batches;      // of a thread, at most
};

constexpr int kMaxShare = 8, kWarps = kThreads / 32;
// A row's largest logit (of a warp, of a CTA), and relative to it the sums of w and of w log2 w.
struct Sums { float top, sum, mean; };
struct Shared {
  // what a row's first CTA is told by the others
  Sums all[kMaxShare];
  int found[kMaxShare];
  unsigned long long best[kMaxShare][kMaxTop];   // alternatives of each slice in descending order: key and complement of the index
  // a CTA's own
  Sums warp[kWarps];
  float log_sum, base, top;
  uint32_t key[kThreads];                        // of the threads' largest logits
  int above[2][16];
  int count, left, kept, hits, hit[kHits];
  uint32_t bins[256], prefix;
  unsigned long long candidate[kCandidates];
};

template <typename T> union alignas(16) Sixteen {
  uint4 raw;
  uint32_t u[4];
  T e[16 / sizeof(T)];
  __device__ __forceinline__ Sixteen() {}
};
template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T minus_infinity();
template <> __device__ __forceinline__ float minus_infinity<float>() { return -INFINITY; }
template <> __device__ __forceinline__ __half minus_infinity<__half>() { return __ushort_as_half(0xfc00); }
template <> __device__ __forceinline__ __nv_bfloat16 minus_infinity<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
// The largest of a few pieces' numbers (NaN where there is none but that); two-byte ones by pairs.
template <int N> __device__ __forceinline__ float largest(const Sixteen<float> (&x)[N]) {
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < N; ++j) m = fmaxf(m, fmaxf(fmaxf(x[j].e[0], x[j].e[1]), fmaxf(x[j].e[2], x[j].e[3])));
  return m;
}
template <int N> __device__ __forceinline__ float largest(const Sixteen<__half> (&x)[N]) {
  uint32_t m = x[0].u[0];
#pragma unroll
  for (int i = 1; i < 4 * N; ++i) asm("max.f16x2 %0, %0, %1;" : "+r"(m) : "r"(x[i >> 2].u[i & 3]));
  const float2 f = __half22float2(*(const __half2*)&m);
  return fmaxf(f.x, f.y);
}
template <int N> __device__ __forceinline__ float largest(const Sixteen<__nv_bfloat16> (&x)[N]) {
  uint32_t m = x[0].u[0];
#pragma unroll
  for (int i = 1; i < 4 * N; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(x[i >> 2].u[i & 3]));
  return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
// Two numbers, raised to the lowest (minus infinity and NaN become that): fp16's own, -2^122 for bf16.  (The largest bf16 numbers less that pass fp32: `far` is
// infinite then, and the other way is taken.)
template <typename T> __device__ __forceinline__ float lowest() { return 0.f; }
template <> __device__ __forceinline__ float lowest<__half>() { return -65504.f; }
template <> __device__ __forceinline__ float lowest<__nv_bfloat16>() { return -0x1p122f; }
template <typename T> __device__ __forceinline__ float2 pair_above(uint32_t u) { return make_float2(0.f, 0.f); }
template <> __device__ __forceinline__ float2 pair_above<__half>(uint32_t u) {
  asm("max.f16x2 %0, %0, %1;" : "+r"(u) : "r"(0xfbfffbffu));
  return __half22float2(*(const __half2*)&u);
}
template <> __device__ __forceinline__ float2 pair_above<__nv_bfloat16>(uint32_t u) {
  asm("max.bf16x2 %0, %0, %1;" : "+r"(u) : "r"(0xfc80fc80u));
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Whole numbers in the order of the floats; minus infinity, and NaN, which counts as that, are 0.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (!(v > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return u >> 31 ? ~u : u | 0x80000000u;
}
// Its number (0: the lowest; a key between two numbers: one of them or nothing that is below it).
__device__ __forceinline__ float value_of(uint32_t key) { return key < 0x00800000u ? -FLT_MAX : __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ unsigned long long entry(float v, int index) { return (unsigned long long)key_of(v) << 32 | (uint32_t)~index; }   // larger: in front
__device__ __forceinline__ float below_infinity(float v) { return fminf(v, FLT_MAX); }

// A row's slice: pieces lo ... hi - 1 of 16 aligned bytes, the first and last of the row perhaps partly outside it.
template <typename T> struct Slice {
  static constexpr int VEC = 16 / sizeof(T);
  const T* row;       // (logit 0)
  int off, vocab, lo, hi;
  __device__ __forceinline__ int first(int piece) const { return piece * VEC - off; }   // index of its first logit
  __device__ __forceinline__ Sixteen<T> load(int piece) const {   // (minus infinity outside)
    Sixteen<T> x;
    const int i = first(piece);
#pragma unroll
    for (int k = 0; k < VEC; ++k) x.e[k] = minus_infinity<T>();
    if (piece < hi) {
      if (i >= 0 && i + VEC <= vocab) x.raw = *(const uint4*)(row + i);
      else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (i + k >= 0 && i + k < vocab) x.e[k] = row[i + k];
      }
    }
    return x;
  }
  __device__ __forceinline__ void load(int piece, float (&v)[VEC]) const {
    const Sixteen<T> x = load(piece);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = widen<T>(x.e[k]);
  }
};

// Relative to a larger maximum.  (Below an infinite one nothing is left of finite logits.)
__device__ __forceinline__ void lower(float& sum, float& mean, float top, float to, float k2) {
  const float shift = top == to || !(top > -INFINITY) ? 0.f : to < INFINITY ? fmaxf((top - to) * k2, -200.f) : -200.f, f = exp2f(shift);
  mean = f * (mean + shift * sum);
  sum *= f;
}
template <int LANES> __device__ __forceinline__ Sums together(Sums x, float k2) {
  float top = x.top;
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  lower(x.sum, x.mean, x.top, top, k2);
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) {
    x.sum += __shfl_xor_sync(~0u, x.sum, o);
    x.mean += __shfl_xor_sync(~0u, x.mean, o);
  }
  x.top = top;
  return x;
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
      w.prefix = prefix | (uint32_t)bin << shift;
      w.left = more;
    }
    __syncthreads();
    prefix = w.prefix;
    left = w.left;
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
        if (at < kCandidates) w.candidate[at] = entry(v[k], s.first(p) + k);
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
        if (at < kCandidates) w.candidate[at] = entry(v[k], s.first(p) + k);
      }
    __syncthreads();
    if (threadIdx.x == 0) w.kept = kept + all;
    __syncthreads();
  }
}

// One pass over a row's logits: each thread keeps its largest one and, relative to it, the sums of w = 2^t and of w t, t = (l - max) / T in
// base 2; then lanes, warps, and the CTAs that share the row, are put together.
// Alternatives: the n-th largest of the threads' maxima is no larger than the n-th largest logit, so that only logits from there on can be among the n; they
// are few, and are found again through the remembered maximum of each batch of pieces.  The sixteen upper bits of the bound are enough; four at a
// time, each warp counts for one of their sixteen values (bit by bit, 32 barriers and lists that the first CTA fetched entry by entry
// made up 22 of 32 us for 64 rows of 128000 logits).  A candidate's place is the number of those in front of it.
// 1024 rows of 131072 fp32 logits: 100 us, 5.4 TB/s, 90 without alternatives.  Two-byte logits are bound by the issue slots, some nine instructions each: 2048 rows of 128000 bf16 97 us
// (5.4 TB/s), 113 with 20 alternatives.  64 such rows take 11.5 us, 7 without, a chain of barriers; four CTAs share each.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) log_probs_kernel(const __grid_constant__ Params p) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ uint16_t group_top[];   // [batches][threads]: the upper halves of their keys
  __shared__ Shared w;
  const LogProbs& l = p.l;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rank = p.share == 1 ? 0 : blockIdx.x % p.share;
  const int64_t r = p.share == 1 ? blockIdx.x : blockIdx.x / p.share;
  cg::cluster_group cluster = cg::this_cluster();
  if (p.share > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");   // (the first CTA is there before others write to it)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Slice<T> s;
  s.row = (const T*)l.logits + r * l.row;
  s.off = (int)((uintptr_t)s.row % 16 / sizeof(T));
  s.vocab = l.vocab;
  const int pieces = (s.off + l.vocab + VEC - 1) / VEC, each = p.share == 1 ? pieces : (pieces + p.share - 1) / p.share;
  s.lo = min(pieces, rank * each);
  s.hi = min(pieces, s.lo + each);
  const float temperature = l.temperature ? l.temperature[r] : 1.f, T1 = temperature > 0.f ? fminf(temperature, 0x1p100f) : 1.f;   // (up to there a difference beyond fp32 weighs nothing)
  const float k2 = fminf(kLog2e / T1, FLT_MAX);
  if (t == 0) { w.count = 0; w.hits = 0; }

  // the first given tokens' logits, on their way while the row is read
  float given = -INFINITY;
  if (rank == 0 && t < l.given) {
    const int token = l.tokens[r * l.given + t];
    if (token >= 0 && token < l.vocab) given = widen<T>(s.row[token]);
  }

  float top = -INFINITY, sum = 0.f, mean = 0.f;
  auto load = [&](int b, Sixteen<T> (&x)[kBatch]) {
    const int piece = s.lo + b * (kThreads * kBatch) + t;
    if (s.lo + (b + 1) * (kThreads * kBatch) < s.hi && s.first(s.lo + b * (kThreads * kBatch)) >= 0) {   // all inside the row
#pragma unroll
      for (int j = 0; j < kBatch; ++j) x[j].raw = *(const uint4*)(s.row + s.first(piece + j * kThreads));
    } else {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) x[j] = s.load(piece + j * kThreads);
    }
  };
  const int batches = (s.hi - s.lo + kThreads * kBatch - 1) / (kThreads * kBatch);
  Sixteen<T> x[kBatch];
  if (batches) load(0, x);
  // (two at a time save four-byte types a twentieth and cost two-byte ones, with their longer code, a tenth)
#pragma unroll (sizeof(T) == 4 ? 2 : 1)
  for (int b = 0; b < batches; ++b) {
    Sixteen<T> next[kBatch];
    if (b + 1 < batches) load(b + 1, next);
    const float mx = largest(x);
    if (l.top) group_top[b * kThreads + t] = (uint16_t)(key_of(mx) >> 16);
    if (mx > top) {     // (infinities share all probability)
      if (top > -INFINITY) lower(sum, mean, top, mx, k2);
      top = mx;
    }
    float2 sums[2] = {}, means[2] = {};
    const float far = (top - lowest<T>()) * k2;   // (infinite with the largest logit, whatever the temperature)
    if (sizeof(T) == 2 && far >= 64.f && far <= 1e30f) {   // (the lowest stands for what has no probability)
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 y = mul2(add2(pair_above<T>(x[j].u[k]), make_float2(-top, -top)), make_float2(k2, k2));
          const float2 e = make_float2(exp2_fast(y.x), exp2_fast(y.y));
          sums[k & 1] = add2(sums[k & 1], e);
          means[k & 1] = fma2(e, y, means[k & 1]);
        }
    } else if (top < INFINITY) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int k = 0; k < VEC; k += 2) {
          float2 y = mul2(add2(make_float2(widen<T>(x[j].e[k]), widen<T>(x[j].e[k + 1])), make_float2(-top, -top)), make_float2(k2, k2));
          y.x = fmaxf(y.x, -150.f);   // (2^-150 is 0; NaN becomes that, too)
          y.y = fmaxf(y.y, -150.f);
          const float2 e = make_float2(exp2_fast(y.x), exp2_fast(y.y));
          sums[k >> 1 & 1] = add2(sums[k >> 1 & 1], e);
          means[k >> 1 & 1] = fma2(e, y, means[k >> 1 & 1]);
        }
    } else {   // (infinities alone have a weight, of 1)
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sums[k & 1].x += widen<T>(x[j].e[k]) == INFINITY ? 1.f : 0.f;
    }
    sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
    mean += (means[0].x + means[0].y) + (means[1].x + means[1].y);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) x[j].raw = next[j].raw;
  }
  // ---- the warp's, the block's ----
  w.key[t] = key_of(top);
  {
    const Sums mine = together<32>(Sums{top, sum, mean}, k2);
    if (lane == 0) w.warp[warp] = mine;
  }
  __syncthreads();
  Sums block{};
  if (warp == 0) block = together<kWarps>(w.warp[lane & (kWarps - 1)], k2);
  int found = 0;
  if (l.top) {
    uint32_t keys[kThreads / 32];
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) keys[i] = w.key[i * 32 + lane];
    uint32_t bound = 0;
    if (l.top == 1) {          // (the largest logit itself)
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) bound = max(bound, keys[i]);
      bound = __reduce_max_sync(~0u, bound);
    } else {
#pragma unroll
      for (int shift = 28; shift >= 16; shift -= 4) {
        int* counts = w.above[shift >> 2 & 1];
#pragma unroll
        for (int e = 0; e < 16; e += kWarps) {
          const uint32_t at = bound | (uint32_t)(warp + e) << shift;
          int above = 0;
#pragma unroll
          for (int i = 0; i < kThreads / 32; ++i) above += keys[i] >= at;
          above = __reduce_add_sync(~0u, above);
          if (lane == 0) counts[warp + e] = above;
        }
        __syncthreads();
        const uint32_t enough = __ballot_sync(~0u, lane < 16 && counts[lane & 15] >= l.top) | 1u;   // (falling counts)
        bound |= (uint32_t)(31 - __clz(enough)) << shift;
      }
    }
    // batches that hold one, then their pieces, a thread for each
    const float least = value_of(bound);
    const uint16_t upper = (uint16_t)max(bound >> 16, 1u);
    if (top >= least) {
#pragma unroll 4
      for (int b = 0; b < batches; ++b)
        if (group_top[b * kThreads + t] >= upper) {
          const int at = atomicAdd(&w.hits, 1);
          if (at < kHits) w.hit[at] = s.lo + b * (kThreads * kBatch) + t;
        }
    }
    __syncthreads();
    const int hits = w.hits;
    if (hits > kHits) {
      if (t == 0) w.count = kCandidates + 1;
    } else {
      for (int i = t; i < hits * kBatch; i += kThreads) {
        const int piece = w.hit[i / kBatch] + i % kBatch * kThreads;
        float v[VEC];
        s.load(piece, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          if (v[k] >= least) {
            const int at = atomicAdd(&w.count, 1);
            if (at < kCandidates) w.candidate[at] = entry(v[k], s.first(piece) + k);
          }
      }
    }
    __syncthreads();
    if (w.count > kCandidates) gather_exactly(s, l.top, w);
    __syncthreads();
    const int n = min(w.count, kCandidates);
    found = min(n, l.top);
    for (int c = t; c < n; c += kThreads) {
      const unsigned long long mine = w.candidate[c];
      int place = 0;
#pragma unroll 8
      for (int i = 0; i < n; ++i) place += w.candidate[i] > mine;
      if (place < l.top) w.best[rank][place] = mine;
    }
  }
  Shared* first = &w;
  if (p.share > 1) {
    first = cluster.map_shared_rank(&w, 0);
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    __syncthreads();
    if (rank)
      for (int k = t; k < found; k += kThreads) first->best[rank][k] = w.best[rank][k];
  }
  if (t == 0) { first->all[rank] = block; first->found[rank] = found; }
  if (p.share > 1) {
    cluster.sync();
    if (rank) return;
  } else if (l.top) {
    __syncthreads();
  }
  // ---- the row's ----
  if (warp == 0) {
    if (p.share > 1) block = together<kMaxShare>(lane % kMaxShare < p.share ? w.all[lane % kMaxShare] : Sums{-INFINITY, 0.f, 0.f}, k2);
    const float log_sum = logf(block.sum);
    if (lane == 0) {
      w.top = block.top; w.log_sum = log_sum;
      if (l.entropy) l.entropy[r] = block.sum > 0.f ? log_sum - kLn2 * block.mean / block.sum : 0.f;
    }
  }
  if (!l.given && !l.top) return;
  __syncthreads();
  const float row_top = w.top, base = below_infinity(row_top), log_sum = w.log_sum;
  auto log_prob = [&](float v) {
    if (!(v > -INFINITY) || (row_top == INFINITY && v < INFINITY)) return -INFINITY;
    return (below_infinity(v) * 0.5f - base * 0.5f) / T1 * 2.f - log_sum;   // (halves: the difference may pass fp32's range, the quotient not)
  };
  if (t < l.given) l.token_log_probs[r * l.given + t] = log_prob(given);
  for (int i = t + kThreads; i < l.given; i += kThreads) {
    const int token = l.tokens[r * l.given + i];
    l.token_log_probs[r * l.given + i] = token >= 0 && token < l.vocab ? log_prob(widen<T>(s.row[token])) : -INFINITY;
  }
  int all = 0;
  for (int i = 0; i < p.share; ++i) all += w.found[i];
  for (int c = t; c < p.share * l.top; c += kThreads) {
    const int i = p.share == 1 ? 0 : c / l.top, k = c - i * l.top;
    if (k >= w.found[i]) continue;
    const unsigned long long mine = w.best[i][k];
    int place = k;
    for (int j = 0; j < p.share; ++j)
      if (j != i) {
        const int n = w.found[j];
#pragma unroll 4
        for (int m = 0; m < n; ++m) place += w.best[j][m] > mine;
      }
    if (place < l.top) {
      const uint32_t key = (uint32_t)(mine >> 32);
      l.top_tokens[r * l.top + place] = (int)~(uint32_t)mine;
      l.top_log_probs[r * l.top + place] = log_prob(__uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key));
    }
  }
  for (int k = all + t; k < l.top; k += kThreads) { l.top_tokens[r * l.top + k] = -1; l.top_log_probs[r * l.top + k] = -INFINITY; }
}

template <typename T> int launch(const LogProbs& l, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  Params p{};
  p.l = l;
  const int pieces = (l.vocab + VEC - 1) / VEC + 1;
  p.share = 1;
  while (p.share < 8 && l.rows * p.share < 148 && pieces / p.share > 2 * kThreads) p.share *= 2;
  p.batches = ((pieces + p.share - 1) / p.share + kThreads * kBatch - 1) / (kThreads * kBatch);
  const size_t smem = l.top ? sizeof(uint16_t) * (size_t)p.batches * kThreads : 0;
  auto* fn = log_probs_kernel<T>;
  static std::atomic<uint64_t> told{0};
  if (smem > kMostSmem || !once_per_device(told, [&] { return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostSmem) == cudaSuccess; })) return -2;
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
