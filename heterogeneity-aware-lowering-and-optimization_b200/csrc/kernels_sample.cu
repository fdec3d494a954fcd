// The next token of each row of logits: temperature, top-k, top-p, min-p and an inverse cumulative distribution.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>

#include "kernels.h"

namespace b200 {
namespace {
namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 8;

// Logits as keys that compare like them: whole numbers, larger for larger logits, 0 for those that are never chosen (NaN, -inf).
// -0 becomes +0: equal logits must have equal keys.
template <typename T> struct Keys;
template <> struct Keys<float> {
  using Key = uint32_t;
  static constexpr int kBits = 32;
  static __device__ __forceinline__ Key key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v > -INFINITY ? ((b >> 31) ? ~b : b | 0x80000000u) : 0u;
  }
  static __device__ __forceinline__ float value(Key k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
};
template <int INF> __device__ __forceinline__ uint16_t half_key(uint16_t b) {   // INF: the type's bits of infinity
  const uint32_t m = b & 0x7fffu;
  if (m > INF || b == (0x8000u | INF)) return 0;
  return (b >> 15) && m ? (uint16_t)~b : (uint16_t)(m | 0x8000u);
}
template <> struct Keys<__half> {
  using Key = uint16_t;
  static constexpr int kBits = 16;
  static __device__ __forceinline__ Key key(__half v) { return half_key<0x7c00>(__half_as_ushort(v)); }
  static __device__ __forceinline__ float value(Key k) { return __half2float(__ushort_as_half((k >> 15) ? k & 0x7fff : (uint16_t)~k)); }
};
template <> struct Keys<__nv_bfloat16> {
  using Key = uint16_t;
  static constexpr int kBits = 16;
  static __device__ __forceinline__ Key key(__nv_bfloat16 v) { return half_key<0x7f80>(__bfloat16_as_ushort(v)); }
  static __device__ __forceinline__ float value(Key k) { return __uint_as_float((uint32_t)((k >> 15) ? k & 0x7fff : (uint16_t)~k) << 16); }
};

constexpr int kBins = 2048, kList = 2048, kListTopK = 1024;
constexpr float kBinsPerE = 32.f;         // bins per factor e of the weight: bin 2047 holds weights below 2^-92, which are no units

struct Shared {
  double table[256];                      // 2^(j / 256)
  // The direct way: a histogram (counts, or masses), then a list of (key, ~index), and what every warp of the cluster has summed.
  union { uint32_t hist[kBins]; unsigned long long list[kList]; };
  unsigned long long weight[kListTopK];   // of the list's first, by rank (top-k)
  unsigned long long all[kMaxCluster * kWarps], below[kMaxCluster * kWarps], taken[kMaxCluster * kWarps];
  double share;
  unsigned long long before;
  double target;
  unsigned long long cut_entry;
  int n_list, found, owner, ok;
  unsigned long long warp_sum[kWarps], cta_sum, best;
  uint32_t lo[2][256], hi[2][256];        // histograms: counts in lo, or masses in both words
  unsigned long long total[256], above, in_bin;
  uint32_t bin;
  int cut, pick;
};

// exp(d * inverse) for d <= 0, with scale = inverse * 256 / ln 2: a table of 2^(j/256) and the exponential series up to the third power on
// |r| <= ln 2 / 512 (P. T. P. Tang's table-driven method, 1989); the next term is below 1.4e-13, and in a sum of many weights, of
// either size, less.  Ten operations in 64 bits, two clocks of a scheduler each, are what a weight costs; a table of 64 takes two more.
__device__ __forceinline__ double exp_below(double d, double scale, const double* table) {
  const double z = d * scale;
  if (!(z > -258000.0)) return 0.0;                            // below exp(-698)
  const double shift = 6755399441055744.0;                     // 1.5 * 2^52: adding it rounds to a whole number
  const double m = z + shift, g = z - (m - shift);
  const int n = __double2loint(m);
  constexpr double c = 0.69314718055994530942 / 256;
  double p = fma(g, c * c * c / 6, c * c / 2);
  p = fma(p, g, c) * g;
  const double t = table[n & 255], w = __hiloint2double(__double2hiint(t) + ((n >> 8) << 20), __double2loint(t));
  return fma(w, p, w);
}
// Weights are summed as whole numbers of 2^-44 of the largest: 2^18 of them stay inside 62 bits, and the sums do not depend on
// their order.
__device__ __forceinline__ unsigned long long units(double w) {
  const double whole = fma(w, 17592186044416.0, 4503599627370496.0);   // 2^44 w + 2^52, rounded to a whole number
  return (unsigned long long)__double_as_longlong(whole) & 0xfffffffffffffull;
}

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
__device__ __forceinline__ unsigned long long warp_scan(unsigned long long v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(~0u, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

struct Row {
  float temperature, top_p, min_p, uniform;
  int top_k;
};

// Sum over the block's threads before this one, and over all of them.
template <typename V> __device__ __forceinline__ V block_scan(V mine, V* warps, V& total, int lane, int warp) {
  V upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(~0u, upto, o);
    if (lane >= o) upto += u;
  }
  const V previous = __shfl_up_sync(~0u, upto, 1);
  __syncthreads();
  if (lane == 31) warps[warp] = upto;
  __syncthreads();
  V before = 0;
  total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = total;
    total += warps[w];
  }
  return lane ? before + previous : before;   // (the same sums, in the same order, as the thread in front of this one ends with)
}
// Largest first; n2 a power of two, entries from n on are zeros.
__device__ __forceinline__ void sort_list(unsigned long long* list, int n2, int tid) {
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j; j >>= 1) {
      __syncthreads();
      for (int i = tid; i < n2 / 2; i += kThreads) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const unsigned long long x = list[a], y = list[b];
        if ((x < y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
      }
    }
  __syncthreads();
}

// What nearly every row takes.  A bin is a range of logits whose weights differ by a factor of e^(1/32): one histogram over 2048 of them, of
// counts for top-k or of masses (32-bit, relative to the bin's middle: good to 2^-16) for top-p, finds the bin of the last
// kept token.
//   top-k up to 1024: all tokens down to that bin go to a list of the first CTA, which sorts it and does the rest alone.
//   otherwise: every CTA sums exact weights, over all tokens, over those in higher bins, and of the latter, warp by warp, over those that
//   min-p keeps; tokens in the bin itself go to the list.  The first CTA sorts it, finds the last token kept, and which
//   warp's stretch of the row the choice lies in; that stretch's CTA finds it there.
// The histogram of masses only proposes the bin: the exact sums have to confirm it.  Returns false, with nothing written, where that fails, the list
// is full (many equal logits), or a parameter is out of this way's range (top-k above 1024, uniform outside (0, 1), temperature, infinities).
// All CTAs of a cluster take the same branches.
template <typename T>
__device__ __forceinline__ bool direct(Shared& s, cg::cluster_group& cluster, const typename Keys<T>::Key* keys, const Row& r, typename Keys<T>::Key top_key, double scale, int vocab,
                                       int slice, int row, int* tokens) {
  using K = Keys<T>;
  using Key = typename K::Key;
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, base = rank * slice;
  const float topf = K::value(top_key), per_unit = kBinsPerE / r.temperature;
  const bool by_count = r.top_k > 0 && r.top_k < vocab, by_mass = r.top_p < 1.f;
  if (!(r.uniform > 0.f && r.uniform < 1.f) || !(fabsf(topf) < 1e30f) || !(r.temperature > 1e-4f && r.temperature < 1e4f) || (by_count && r.top_k > kListTopK)) return false;
  const double top = (double)topf;
  auto weight = [&](Key k) { return k == top_key ? 1.0 : exp_below((double)K::value(k) - top, scale, s.table); };
  Shared* first = cluster.map_shared_rank(&s, 0);
  // the bin, as a float: nearest to (top - logit) * per_unit, which grows as logits fall
  auto place = [&](Key k) { return fminf((topf - K::value(k)) * per_unit, (float)(kBins - 1)); };
  auto bin_of = [&](float at) { return (int)(__float_as_uint(at + 8388608.f) & 0x7fffffu); };
  int bin = -1;
  if (by_count || by_mass) {
    for (int i = tid; i < kBins; i += kThreads) s.hist[i] = 0;
    if (tid == 0) { s.found = -1; s.n_list = 0; }
    __syncthreads();
    struct alignas(4 * sizeof(Key)) Four { Key k[4]; };
    for (int i = tid; i < slice / 4; i += kThreads) {
      const Four f = ((const Four*)keys)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (f.k[j]) {
          const float at = place(f.k[j]);
          const int b = bin_of(at);
          uint32_t add = 1;
          if (!by_count) {   // 2^16 e^(-(at - b) / 32), |at - b| <= 1/2, to 2^-22
            const float x = ((float)b - at) * (1.f / kBinsPerE);
            add = __float_as_uint(fmaf(fmaf(fmaf(x, 1.f / 6, 0.5f), x, 1.f), x * 65536.f, 65536.f + 8388608.f)) & 0x7fffffu;
          }
          atomicAdd(&s.hist[b], add);
        }
    }
    cluster.sync();
    // each CTA adds up its share of the bins
    const int share = kBins / ranks, each = share > kThreads ? share / kThreads : 1, b0 = rank * share + tid * each;
    const bool mine = tid * each < share;
    double v[kBins / kThreads], sum = 0;
#pragma unroll
    for (int j = 0; j < kBins / kThreads; ++j) {
      v[j] = 0;
      if (mine && j < each) {
        unsigned long long n = 0;
        for (int k = 0; k < ranks; ++k) n += cluster.map_shared_rank(&s, k)->hist[b0 + j];
        v[j] = (double)n;
        if (!by_count) v[j] *= (double)exp2f((float)(b0 + j) * (-1.44269504f / kBinsPerE));
      }
      sum += v[j];
    }
    double total;
    const double before = block_scan(sum, (double*)s.warp_sum, total, lane, warp);
    if (tid == 0) s.share = total;
    cluster.sync();
    double offset = 0, everything = 0;
    for (int k = 0; k < ranks; ++k) {
      if (k == rank) offset = everything;
      everything += cluster.map_shared_rank(&s, k)->share;
    }
    const double need = by_count ? (double)r.top_k : (double)r.top_p * everything;
    double run = offset + before;
#pragma unroll
    for (int j = 0; j < kBins / kThreads; ++j) {
      if (run < need && need <= run + v[j])
        for (int k = 0; k < ranks; ++k) cluster.map_shared_rank(&s, k)->found = b0 + j;
      run += v[j];
    }
    cluster.sync();
    bin = s.found;
    if (bin < 0 || bin == kBins - 1) return false;   // (fewer tokens than k; a mark that rounding put between two bins; weights of no units)
  }
  auto push = [&](bool any, Key k, int i) {
    const uint32_t who = __ballot_sync(~0u, any);
    if (!who) return;
    int at = 0;
    if (lane == __ffs(who) - 1) at = atomicAdd(&first->n_list, __popc(who));
    at = __shfl_sync(~0u, at, __ffs(who) - 1) + __popc(who & ((1u << lane) - 1));
    if (any && at < kList) first->list[at] = ((unsigned long long)k << 32) | (uint32_t)~(uint32_t)(base + i);
  };
  const int sub = slice / kWarps, warp_base = warp * sub;
  const double least = (double)r.min_p;
  if (by_count) {
    for (int i = lane; i < sub; i += 32) {
      const Key k = keys[warp_base + i];
      push(k && bin_of(place(k)) <= bin, k, warp_base + i);
    }
  } else {
    // (below this no weight passes min-p, with room for the roundings of 32 bits)
    const float last = by_mass ? (float)(kBins - 1) : r.min_p > 0.f ? fminf(-kBinsPerE * logf(r.min_p) + 1.f, (float)(kBins - 1)) : (float)(kBins - 1);
    unsigned long long all = 0, below = 0, taken = 0;
    for (int i = lane; i < sub; i += 32) {
      const Key k = keys[warp_base + i];
      const float at = k ? place(k) : (float)kBins;
      bool listed = false;
      if (at < last) {
        const double w = weight(k);
        const unsigned long long u = units(w);
        const int b = bin_of(at);
        all += u;
        if (!by_mass || b < bin) {
          below += u;
          if (w >= least) taken += u;
        } else {
          listed = b == bin;
        }
      }
      if (by_mass) push(listed, k, warp_base + i);
    }
    all = warp_sum(all); below = warp_sum(below); taken = warp_sum(taken);
    if (lane == 0) { first->all[rank * kWarps + warp] = all; first->below[rank * kWarps + warp] = below; first->taken[rank * kWarps + warp] = taken; }
  }
  cluster.sync();
  if (by_count || by_mass) {
    const bool full = first->n_list > kList;
    cluster.sync();   // (the first CTA goes on, and the others may leave)
    if (full) return false;
  }
  // exact weights of the sorted list, four entries per thread; entries from `limit` on do not count
  unsigned long long unit[4], sum = 0, total = 0, run = 0;
  double w[4];
  auto weigh = [&](int limit) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * 4 + j;
      w[j] = i < limit ? weight((Key)(s.list[i] >> 32)) : 0.0;
      unit[j] = i < limit ? units(w[j]) : 0;
      sum += unit[j];
    }
    run = block_scan(sum, s.warp_sum, total, lane, warp);
  };
  auto sorted = [&]() {
    const int n = s.n_list;
    int n2 = 2;
    while (n2 < n) n2 *= 2;
    for (int i = n + tid; i < n2; i += kThreads) s.list[i] = 0;
    sort_list(s.list, n2, tid);
    return n;
  };
  if (by_count) {
    if (rank) return true;
    sorted();
    weigh(r.top_k);
    const double mark = by_mass ? (double)r.top_p * (double)total : 0.0;
    unsigned long long kept = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * 4 + j;
      if (i < r.top_k && (i == 0 || ((!by_mass || (double)run < mark) && w[j] >= least))) {
        kept += unit[j];
        s.weight[i] = unit[j];
      } else if (i < kListTopK) {
        s.weight[i] = 0;
      }
      run += unit[j];
    }
    block_scan(kept, s.warp_sum, total, lane, warp);
    // by index, six bits at a time: the digit at which the running sum passes the target
    const double target = (double)r.uniform * (double)total;
    uint32_t prefix = 0;
    unsigned long long before = 0;
    for (int shift = 12; shift >= 0; shift -= 6) {
      if (tid < 64) { s.lo[0][tid] = 0; s.hi[0][tid] = 0; }
      __syncthreads();
      for (int i = tid; i < r.top_k; i += kThreads) {
        const uint32_t index = ~(uint32_t)s.list[i];
        const unsigned long long u = s.weight[i];
        if (u && index >> (shift + 6) == prefix) {
          const int d = (index >> shift) & 63;
          const uint32_t lo = (uint32_t)u, old = atomicAdd(&s.lo[0][d], lo), up = (uint32_t)(u >> 32) + (old + lo < old ? 1u : 0u);
          if (up) atomicAdd(&s.hi[0][d], up);
        }
      }
      __syncthreads();
      if (warp == 0) {
        const unsigned long long x = ((unsigned long long)s.hi[0][2 * lane] << 32) + s.lo[0][2 * lane], y = ((unsigned long long)s.hi[0][2 * lane + 1] << 32) + s.lo[0][2 * lane + 1];
        const unsigned long long upto = before + warp_scan(x + y, lane), from = upto - x - y;
        const uint32_t ballot = __ballot_sync(~0u, (double)upto > target);
        if (lane == __ffs(ballot) - 1) {
          const bool second = !((double)(from + x) > target);
          s.bin = prefix << 6 | (uint32_t)(2 * lane + second);
          s.above = second ? from + x : from;
        }
      }
      __syncthreads();
      prefix = s.bin;
      before = s.above;
    }
    if (tid == 0) tokens[row] = (int)prefix;
    return true;
  }
  if (rank == 0) {
    // the sums of all warps, in index order
    const int n_warps = ranks * kWarps;
    const unsigned long long all = tid < n_warps ? s.all[tid] : 0, below = tid < n_warps ? s.below[tid] : 0;
    unsigned long long sum_all, sum_below;
    block_scan(all, s.warp_sum, sum_all, lane, warp);
    block_scan(below, s.warp_sum, sum_below, lane, warp);
    if (tid == 0) { s.ok = 1; s.cut_entry = 0; s.owner = -1; }
    if (by_mass) {
      const int n = sorted();
      weigh(n);
      const double mark = (double)r.top_p * (double)sum_all;
      run += sum_below;
      // (kept entries are the first ones; the last of them ends the kept tokens)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = tid * 4 + j;
        const bool kept = i < n && ((double)run < mark || (i == 0 && sum_below == 0));
        const bool next = i + 1 < n && (double)(run + unit[j]) < mark;
        if (kept) {
          const unsigned long long entry = s.list[i];
          if (!next) s.cut_entry = entry;
          const uint32_t index = ~(uint32_t)entry;
          if (w[j] >= least) atomicAdd(&s.taken[index / (uint32_t)sub], unit[j]);
        }
        run += unit[j];
      }
      if (tid == 0 && !((sum_below == 0 || (double)sum_below < mark) && mark <= (double)(sum_below + total))) s.ok = 0;
    }
    __syncthreads();
    const unsigned long long taken = tid < n_warps ? s.taken[tid] : 0;
    unsigned long long sum_taken;
    const unsigned long long before = block_scan(taken, s.warp_sum, sum_taken, lane, warp);
    const double target = (double)r.uniform * (double)sum_taken;
    if (!((double)before > target) && (double)(before + taken) > target)
      for (int k = 0; k < ranks; ++k) {
        Shared* o = cluster.map_shared_rank(&s, k);
        o->owner = tid; o->before = before; o->target = target;
      }
    __syncthreads();
    if (tid < ranks && tid) { Shared* o = cluster.map_shared_rank(&s, tid); o->cut_entry = s.cut_entry; o->ok = s.ok; }
  }
  cluster.sync();
  if (!s.ok) return false;
  if (s.owner / kWarps != rank) return true;
  // the stretch of one warp, now by all warps of its CTA
  const Key cut = (Key)(s.cut_entry >> 32);
  const int cut_index = by_mass ? (int)~(uint32_t)s.cut_entry : INT_MAX, stretch = (s.owner - rank * kWarps) * sub, part = (sub / kWarps + 31) & ~31;
  auto chosen = [&](int i) -> unsigned long long {
    if (i >= sub) return 0;
    const Key k = keys[stretch + i];
    if (!k || !(k > cut || (k == cut && base + stretch + i <= cut_index))) return 0;
    const double w = weight(k);
    return w >= least ? units(w) : 0;
  };
  unsigned long long mine = 0;
  for (int i = warp * part + lane; i < (warp + 1) * part; i += 32) mine += chosen(i);
  mine = warp_sum(mine);
  __syncthreads();
  if (lane == 0) s.warp_sum[warp] = mine;
  __syncthreads();
  unsigned long long before = s.before;
  for (int k = 0; k < warp; ++k) before += s.warp_sum[k];
  if ((double)before > s.target || !((double)(before + mine) > s.target)) return true;
  for (int i = warp * part; i < (warp + 1) * part; i += 32) {
    const unsigned long long upto = before + warp_scan(chosen(i + lane), lane);
    const uint32_t ballot = __ballot_sync(~0u, (double)upto > s.target);
    if (ballot) {
      if (lane == __ffs(ballot) - 1) tokens[row] = base + stretch + i + lane;
      break;
    }
    before = __shfl_sync(~0u, upto, 31);
  }
  return true;
}

// One cluster of CTAs takes one row, each CTA `slice` consecutive logits, which it reads once and keeps as keys in shared memory.
//   1. the largest key (and, of those, the lowest index);
//   2. top-k and top-p, each a search for the key t and, among the tokens with that key, the last index c that are still kept: a
//      histogram of counts, or of masses, over 8 bits of the keys at a time from the top;
//   3. the sum of what is kept, and the place where the running sum passes uniform * W.
// Sums over CTAs go through distributed shared memory in rank order; index order is rank order, then warp order.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const T* __restrict__ logits, int64_t row_stride, int vocab, int slice, int vec, const float* temperature,
                                                          const int* top_k, const float* top_p, const float* min_p, const float* uniform, int* tokens) {
  using K = Keys<T>;
  using Key = typename K::Key;
  extern __shared__ __align__(16) uint8_t dynamic[];
  Key* keys = (Key*)dynamic;
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = rank * slice;
  const Row r{temperature ? temperature[row] : 1.f, top_p ? top_p[row] : 1.f, min_p ? fminf(min_p[row], 1.f) : 0.f, uniform[row], top_k ? top_k[row] : 0};

  if (tid < 256) { s.table[tid] = exp2((double)tid / 256.0); s.lo[0][tid] = 0; s.hi[0][tid] = 0; }
  // ---- 1. keys, and the largest ----
  unsigned long long best = 0;
  const T* src = logits + (int64_t)row * row_stride + base;
  const int here = max(0, min(slice, vocab - base));
  auto put = [&](int i, T v) {
    const Key k = K::key(v);
    keys[i] = k;
    const unsigned long long b = ((unsigned long long)k << 32) | (uint32_t)~(uint32_t)(base + i);
    if (k && b > best) best = b;
  };
  constexpr int VEC = 16 / sizeof(T);
  int done = 0;
  if (vec) {
    done = here / VEC * VEC;
#pragma unroll 2
    for (int i = tid * VEC; i < done; i += kThreads * VEC) {
      const uint4 u = *(const uint4*)(src + i);
      T e[VEC];
      *(uint4*)e = u;
#pragma unroll
      for (int j = 0; j < VEC; ++j) put(i + j, e[j]);
    }
  }
  for (int i = done + tid; i < here; i += kThreads) put(i, src[i]);
  for (int i = here + tid; i < slice; i += kThreads) keys[i] = 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) { const unsigned long long v = __shfl_xor_sync(~0u, best, o); if (v > best) best = v; }
  if (lane == 0) s.warp_sum[warp] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) if (s.warp_sum[w] > best) best = s.warp_sum[w];
    s.best = best;
  }
  cluster.sync();
  best = 0;
  for (int k = 0; k < ranks; ++k) { const unsigned long long v = cluster.map_shared_rank(&s, k)->best; if (v > best) best = v; }
  const Key top_key = (Key)(best >> 32);
  if (top_key == 0 || !(r.temperature > 0.f)) {
    if (rank == 0 && tid == 0) tokens[row] = top_key == 0 ? -1 : (int)~(uint32_t)best;
    cluster.sync();   // nobody leaves while a peer may still read its shared memory
    return;
  }
  const double top = (double)K::value(top_key), scale = 369.32993046757462708 / (double)r.temperature;   // 256 / ln 2
  auto weight = [&](Key k) { return k == top_key ? 1.0 : exp_below((double)K::value(k) - top, scale, s.table); };
  if (direct<T>(s, cluster, keys, r, top_key, scale, vocab, slice, row, tokens)) return;

  // Kept so far: key > t, or key == t and index <= c.
  Key t = 1;
  int c = INT_MAX, buffer = 0;
  auto kept = [&](Key k, int i) { return k > t || (k == t && i <= c); };
  // The key at which counts, or masses, summed from the largest key down, reach the mark; `above` is the sum over the larger keys
  // and `in_bin` the sum at the key itself.
  auto search = [&](bool mass, auto reached, bool share_of, double share, unsigned long long& above_out, unsigned long long& bin_out, double& mark) -> Key {
    Key prefix = 0;
    unsigned long long above = 0, in_bin = 0;
    for (int shift = K::kBits - 8; shift >= 0; shift -= 8) {
      for (int i = tid; i < slice; i += kThreads) {
        const Key k = keys[i];
        if (k && (shift + 8 == K::kBits || (uint32_t)k >> (shift + 8) == (uint32_t)prefix) && kept(k, base + i)) {
          const int b = ((uint32_t)k >> shift) & 255;
          if (mass) {
            const unsigned long long u = units(weight(k));
            if (u) {
              const uint32_t lo = (uint32_t)u, old = atomicAdd(&s.lo[buffer][b], lo), up = (uint32_t)(u >> 32) + (old + lo < old ? 1u : 0u);
              if (up) atomicAdd(&s.hi[buffer][b], up);
            }
          } else {
            atomicAdd(&s.lo[buffer][b], 1u);
          }
        }
      }
      cluster.sync();
      if (tid < 256) {
        unsigned long long v = 0;
        for (int k = 0; k < ranks; ++k) {
          const Shared* o = cluster.map_shared_rank(&s, k);
          v += ((unsigned long long)o->hi[buffer][tid] << 32) + o->lo[buffer][tid];
        }
        s.total[tid] = v;
        s.lo[buffer ^ 1][tid] = 0;
        s.hi[buffer ^ 1][tid] = 0;
      }
      __syncthreads();
      if (warp == 0) {
        unsigned long long mine = 0;
        for (int j = 0; j < 8; ++j) mine += s.total[255 - lane * 8 - j];
        const unsigned long long upto = warp_scan(mine, lane);
        if (share_of && shift + 8 == K::kBits) mark = share * (double)__shfl_sync(~0u, upto, 31);
        unsigned long long run = above + upto - mine;
        if (!reached(run, mark) && reached(run + mine, mark))
          for (int j = 0; j < 8; ++j) {
            const unsigned long long v = s.total[255 - lane * 8 - j];
            if (reached(run + v, mark)) { s.bin = (uint32_t)(255 - lane * 8 - j); s.above = run; s.in_bin = v; break; }
            run += v;
          }
      }
      __syncthreads();
      prefix = (Key)((uint32_t)prefix << 8 | s.bin);
      above = s.above;
      in_bin = s.in_bin;
      buffer ^= 1;
    }
    above_out = above;
    bin_out = in_bin;
    return prefix;
  };
  // The index of the n-th kept token, by index, whose key is `key`.
  const int sub = slice / kWarps, warp_base = warp * sub;
  auto nth = [&](Key key, int n) -> int {
    int mine = 0;
    for (int i = lane; i < sub; i += 32) mine += keys[warp_base + i] == key && kept(key, base + warp_base + i);
    const unsigned long long count = warp_sum((unsigned long long)mine);
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = count;
    if (tid == 0) s.cut = -1;
    __syncthreads();
    if (tid == 0) {
      unsigned long long v = 0;
      for (int w = 0; w < kWarps; ++w) v += s.warp_sum[w];
      s.cta_sum = v;
    }
    cluster.sync();
    long long before = 0;
    for (int k = 0; k < rank; ++k) before += (long long)cluster.map_shared_rank(&s, k)->cta_sum;
    for (int w = 0; w < warp; ++w) before += (long long)s.warp_sum[w];
    if (before < n && before + (long long)count >= n)
      for (int i = 0; i < sub; i += 32) {
        const bool hit = keys[warp_base + i + lane] == key && kept(key, base + warp_base + i + lane);
        const uint32_t ballot = __ballot_sync(~0u, hit);
        const int upto = (int)before + __popc(ballot & (0xffffffffu >> (31 - lane)));
        if (hit && upto == n) s.cut = base + warp_base + i + lane;
        before += __popc(ballot);
        if (before >= n) break;
      }
    cluster.sync();
    int found = -1;
    for (int k = 0; k < ranks; ++k) found = max(found, cluster.map_shared_rank(&s, k)->cut);
    cluster.sync();
    return found;
  };

  // ---- 2. top-k, top-p ----
  unsigned long long above = 0, in_bin = 0;
  double mark = 0.0;
  if (r.top_k > 0 && r.top_k < vocab) {
    // (with fewer live logits than k no sum reaches the mark: everything stays)
    unsigned long long live = 0;
    {
      int mine = 0;
      for (int i = tid; i < slice; i += kThreads) mine += keys[i] != 0;
      const unsigned long long n = warp_sum((unsigned long long)mine);
      if (lane == 0) s.warp_sum[warp] = n;
      __syncthreads();
      if (tid == 0) {
        unsigned long long v = 0;
        for (int w = 0; w < kWarps; ++w) v += s.warp_sum[w];
        s.cta_sum = v;
      }
      cluster.sync();
      for (int k = 0; k < ranks; ++k) live += cluster.map_shared_rank(&s, k)->cta_sum;
      cluster.sync();
    }
    if ((unsigned long long)r.top_k < live) {
      const unsigned long long need = (unsigned long long)r.top_k;
      const Key found = search(false, [need](unsigned long long v, double) { return v >= need; }, false, 0.0, above, in_bin, mark);
      const int ties = (int)(need - above);
      const int last = (unsigned long long)ties < in_bin ? nth(found, ties) : INT_MAX;
      t = found;
      c = last;
    }
  }
  if (r.top_p < 1.f) {
    const double p = (double)fmaxf(r.top_p, 0.f);
    const Key found = search(true, [](unsigned long long v, double m) { return (double)v >= m && v > 0; }, true, p, above, in_bin, mark);
    // (the mark is known to warp 0)
    const unsigned long long w = units(weight(found));
    if (tid == 0) {
      long long j = w ? (long long)((mark - (double)above) / (double)w) : 1;
      if (j < 1) j = 1;
      while (j > 1 && (double)(above + (unsigned long long)(j - 1) * w) >= mark) --j;
      while ((double)(above + (unsigned long long)j * w) < mark) ++j;
      s.pick = (int)j;
    }
    __syncthreads();
    const int ties = s.pick;
    const int old = found == t ? c : INT_MAX;
    const int last = (unsigned long long)ties * w < in_bin ? nth(found, ties) : old;
    t = found;
    c = last;
  }

  // ---- 3. the choice ----
  const double least = (double)r.min_p;
  auto chosen_weight = [&](int i, bool& is_kept) -> unsigned long long {
    const Key k = keys[i];
    is_kept = false;
    if (!k || !kept(k, base + i)) return 0;
    const double w = weight(k);
    is_kept = w >= least;
    return is_kept ? units(w) : 0;
  };
  unsigned long long sum = 0;
  int lowest = INT_MAX, highest = -1;
  for (int i = lane; i < sub; i += 32) {
    bool is_kept;
    sum += chosen_weight(warp_base + i, is_kept);
    if (is_kept) { lowest = min(lowest, base + warp_base + i); highest = base + warp_base + i; }
  }
  sum = warp_sum(sum);
  __syncthreads();
  if (tid == 0) { s.pick = r.uniform > 0.f ? -1 : INT_MAX; s.cut = -1; }
  if (lane == 0) s.warp_sum[warp] = sum;
  __syncthreads();
  if (!(r.uniform > 0.f)) atomicMin(&s.pick, lowest);
  atomicMax(&s.cut, highest);
  if (tid == 0) {
    unsigned long long v = 0;
    for (int w = 0; w < kWarps; ++w) v += s.warp_sum[w];
    s.cta_sum = v;
  }
  cluster.sync();
  unsigned long long before = 0, all = 0;
  int first = INT_MAX, last = -1;
  for (int k = 0; k < ranks; ++k) {
    const Shared* o = cluster.map_shared_rank(&s, k);
    if (k < rank) before += o->cta_sum;
    all += o->cta_sum;
    first = min(first, o->pick);
    last = max(last, o->cut);
  }
  const double target = (double)r.uniform * (double)all;
  if (!(r.uniform > 0.f) || !((double)all > target)) {
    if (rank == 0 && tid == 0) tokens[row] = !(r.uniform > 0.f) ? first : last;
  } else {
    for (int w = 0; w < warp; ++w) before += s.warp_sum[w];
    if (!((double)before > target) && (double)(before + sum) > target)
      for (int i = 0; i < sub; i += 32) {
        bool is_kept;
        const unsigned long long upto = before + warp_scan(chosen_weight(warp_base + i + lane, is_kept), lane);
        const uint32_t ballot = __ballot_sync(~0u, (double)upto > target);
        if (ballot) {
          if (lane == __ffs(ballot) - 1) tokens[row] = base + warp_base + i + lane;
          break;
        }
        before = __shfl_sync(~0u, upto, 31);
      }
  }
  cluster.sync();
}

template <typename T>
int launch(int rows, int vocab, int64_t row, const void* logits, const float* temperature, const int* top_k, const float* top_p, const float* min_p, const float* uniform, int* tokens,
           cudaStream_t stream) {
  int ranks = 1;
  auto slice_of = [&](int n) { return ((vocab + n - 1) / n + kThreads - 1) / kThreads * kThreads; };
  while (ranks < kMaxCluster && (slice_of(ranks) * sizeof(T) > 64 * 1024 || (rows * ranks < 148 && slice_of(ranks) > 2048))) ranks *= 2;
  const int slice = slice_of(ranks);
  const size_t smem = (size_t)slice * sizeof(T);
  const int vec = (uintptr_t)logits % 16 == 0 && row * sizeof(T) % 16 == 0;
  auto* fn = sample_kernel<T>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) { cudaGetLastError(); return -2; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * (unsigned)ranks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, (const T*)logits, row, vocab, slice, vec, temperature, top_k, top_p, min_p, uniform, tokens);
  if (e != cudaSuccess) { cudaGetLastError(); return -2; }
  return 0;
}

}  // namespace

int sample(int dt, int rows, int vocab, int64_t row, const void* logits, const float* temperature, const int* top_k, const float* top_p, const float* min_p, const float* uniform,
           int* tokens, cudaStream_t stream) {
  switch (dt) {
    case DT_F32: return launch<float>(rows, vocab, row, logits, temperature, top_k, top_p, min_p, uniform, tokens, stream);
    case DT_F16: return launch<__half>(rows, vocab, row, logits, temperature, top_k, top_p, min_p, uniform, tokens, stream);
    case DT_BF16: return launch<__nv_bfloat16>(rows, vocab, row, logits, temperature, top_k, top_p, min_p, uniform, tokens, stream);
  }
  return -1;
}

}  // namespace b200
