// The next token of each row of logits: temperature, top-k, top-p, min-p and an inverse cumulative distribution.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cmath>

#include "kernels.h"

namespace b200 {
namespace {
namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 8;
constexpr int kBins = 2048, kList = 1536, kTopK = 1024, kBucket = 128, kFew = kThreads / 4;
constexpr int kSlice = 64 * kThreads;   // logits of a CTA at most: a thread names its own by the bits of one word
constexpr float kNoUnits = 2000.f;   // weights from here on, below 2^-45, are no units
constexpr float kBinsPerE = 64.f;   // bins per factor e of the weight: bin 2047 holds weights below 2^-46, which are no units

// Logits as keys that compare like them: whole numbers, larger for larger logits, 0 for those that are never chosen (NaN, -inf).
// -0 becomes +0: equal logits must have equal keys.
template <int INF> __device__ __forceinline__ uint16_t half_key(uint16_t b) {   // INF: the type's bits of infinity
  const uint32_t m = b & 0x7fffu;
  if (m > INF || b == (0x8000u | INF)) return 0;
  return (b >> 15) && m ? (uint16_t)~b : (uint16_t)(m | 0x8000u);
}
template <typename T> struct Logits;
template <> struct Logits<float> {
  using Key = uint32_t;
  static constexpr int kBits = 32;
  static __device__ __forceinline__ float dead() { return -INFINITY; }
  static __device__ __forceinline__ Key key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v > -INFINITY ? ((b >> 31) ? ~b : b | 0x80000000u) : 0u;
  }
  static __device__ __forceinline__ float value(Key k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
  static __device__ __forceinline__ float widen(float v) { return v; }
  static __device__ __forceinline__ float largest(const uint4& u) {   // of 16 bytes; a NaN loses
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
};
template <> struct Logits<__half> {
  using Key = uint16_t;
  static constexpr int kBits = 16;
  static __device__ __forceinline__ __half dead() { return __ushort_as_half(0xfc00); }
  static __device__ __forceinline__ Key key(__half v) { return half_key<0x7c00>(__half_as_ushort(v)); }
  static __device__ __forceinline__ float value(Key k) { return __half2float(__ushort_as_half((k >> 15) ? k & 0x7fff : (uint16_t)~k)); }
  static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
  static __device__ __forceinline__ float largest(const uint4& u) {
    const __half2* h = (const __half2*)&u;
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <> struct Logits<__nv_bfloat16> {
  using Key = uint16_t;
  static constexpr int kBits = 16;
  static __device__ __forceinline__ __nv_bfloat16 dead() { return __ushort_as_bfloat16(0xff80); }
  static __device__ __forceinline__ Key key(__nv_bfloat16 v) { return half_key<0x7f80>(__bfloat16_as_ushort(v)); }
  static __device__ __forceinline__ float value(Key k) { return __uint_as_float((uint32_t)((k >> 15) ? k & 0x7fff : (uint16_t)~k) << 16); }
  static __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ float largest(const uint4& u) {
    const __nv_bfloat162* h = (const __nv_bfloat162*)&u;
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
// 16 bytes of logits.
template <typename T> struct alignas(16) Piece {
  static constexpr int N = 16 / sizeof(T);
  T e[N];
};

constexpr int kTable = 32, kCopies = 16;
struct Powers { double of[kTable]; };   // 2^(j / 32)
struct alignas(16) Shared {
  double table[kTable][kCopies];          // 2^(j / 32), a copy for each pair of banks
  // The direct way: a histogram (counts, or masses), then a list of (key, ~index); what every warp of the cluster has summed.
  union { uint32_t hist[kBins]; unsigned long long list[2048]; };   // (kList entries, room for a power of two when they are sorted by exchanges)
  union {
    unsigned long long spare[kList];      // while the list is sorted
    unsigned long long weight[kTopK];     // of the list's first, by rank (top-k)
    struct {                              // the general way
      uint32_t lo[2][256], hi[2][256];    // histograms: counts in lo, or masses in both words
      unsigned long long total[256];
    };
  };
  uint32_t bucket[kBins];
  unsigned long long below[kMaxCluster * kWarps], taken[kMaxCluster * kWarps], all[kMaxCluster];
  unsigned long long warp_sum[kWarps], cta_sum, before, cut_entry, above, in_bin;
  float warp_top[kWarps], tops[kMaxCluster];
  unsigned long long shares[kMaxCluster];
  double target;
  uint32_t low_key, high_key, bin, digit_lo[64], digit_hi[64];
  int listed[kMaxCluster], found, owner, ok, crowded, token, cut, pick;
};

// exp(d * inverse) for d <= 0, with scale = inverse * 32 / ln 2: a table of 2^(j/32) and the exponential series up to the fourth power on
// |r| <= ln 2 / 64 (P. T. P. Tang's table-driven method, 1989); the next term is below 1.3e-12, a fifth of that on average over r, and in sums
// of many weights, of either size, less.  Eleven operations in 64 bits, two clocks of a scheduler each, are what a weight costs.  (A table of
// 256 entries and two operations fewer were slower: 32 lanes at random places of it meet in the same banks.)
template <bool NEAR> __device__ __forceinline__ double exp_below(double d, double scale, const Shared& s) {
  const double z = d * scale;
  if (!NEAR && !(z > -32250.0)) return 0.0;                    // below exp(-698); NEAR: known to be above
  const double shift = 6755399441055744.0;                     // 1.5 * 2^52: adding it rounds to a whole number
  const double m = z + shift, g = z - (m - shift);
  const int n = __double2loint(m);
  constexpr double c = 0.69314718055994530942 / 32;
  double p = fma(g, c * c * c * c / 24, c * c * c / 6);
  p = fma(p, g, c * c / 2);
  p = fma(p, g, c) * g;
  const double t = s.table[n & 31][threadIdx.x & 15], w = __hiloint2double(__double2hiint(t) + ((n >> 5) << 20), __double2loint(t));
  return fma(w, p, w);
}
// Weights are summed as whole numbers of 2^-44 of the largest: 2^18 of them stay inside 62 bits, and the sums do not depend on
// their order.
__device__ __forceinline__ unsigned long long units(double w) {
  const double whole = fma(w, 17592186044416.0, 4503599627370496.0);   // 2^44 w + 2^52, rounded to a whole number
  return (unsigned long long)__double_as_longlong(whole) & 0xfffffffffffffull;
}
// The same as a double; sums of up to 256 of them are exact.
__device__ __forceinline__ double units_exact(double w) { return fma(w, 17592186044416.0, 4503599627370496.0) - 4503599627370496.0; }

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

// Adds a weight to a sum of two words.
__device__ __forceinline__ void add_units(uint32_t* lo, uint32_t* hi, unsigned long long u) {
  const uint32_t l = (uint32_t)u, old = atomicAdd(lo, l), up = (uint32_t)(u >> 32) + (old + l < old ? 1u : 0u);
  if (up) atomicAdd(hi, up);
}

struct Row {
  float temperature, top_p, min_p, uniform;
  int top_k;
};

// Sum over the block's threads before this one, and over all of them (whole numbers; a block has at most as many warps as a warp has lanes).
template <typename V> __device__ __forceinline__ V block_scan(V mine, V* warps, V& total, int lane, int warp) {
  auto scan = [lane](V v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V u = __shfl_up_sync(~0u, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  const V upto = scan(mine);
  __syncthreads();
  if (lane == 31) warps[warp] = upto;
  __syncthreads();
  const V all = scan(lane < kWarps ? warps[lane] : (V)0);
  total = __shfl_sync(~0u, all, 31);
  const V before = __shfl_sync(~0u, all, (warp + kWarps - 1) % kWarps);
  return (warp ? before : 0) + upto - mine;
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

// A CTA's part of a row: `slice` logits in shared memory, of which those past the row's end never count.
template <typename T, int RANKS> struct Part {
  static constexpr int kGroups = 8, kPer = kSlice / kThreads / Piece<T>::N / kGroups;
  Shared& s;
  cg::cluster_group cluster;
  const T* logits;             // in shared memory, or, where they do not fit, the caller's
  Row r;
  float top;                   // the row's largest logit
  float group[kGroups];        // the largest of kPer pieces: of this thread's pieces tid + (g * kPer + i) * kThreads
  double scale;                // 32 / (ln 2 * temperature)
  int vocab, slice, limit, base, rank, row;   // logits[i] may be read below `limit`, whole pieces; the rest of a slice counts as dead
  int* tokens;

  using L = Logits<T>;
  using Key = typename L::Key;
  __device__ __forceinline__ Shared* peer(int k) { return RANKS == 1 ? &s : cluster.map_shared_rank(&s, k); }
  __device__ __forceinline__ void sync_row() { if (RANKS == 1) __syncthreads(); else cluster.sync(); }
  __device__ __forceinline__ T logit(int i) const { return i < limit ? logits[i] : L::dead(); }
  __device__ __forceinline__ double weight(float v) const { return exp_below<false>((double)v - (double)top, scale, s); }

  // What nearly every row takes.  A bin is a range of logits whose weights differ by a factor of e^(1/64): one histogram over 2048 of them finds
  // the bin of the last kept token.
  //   top-k up to 1024: a histogram of the largest logits of small groups, kept in registers (the k-th largest of those has at least k tokens above it, and rarely
  //   many more; of every logit where that did not hold, or the row is short).  All tokens down to that bin go to a list of the first CTA,
  //   which sorts it and does the rest alone.
  //   otherwise: a histogram of masses, 32-bit and relative to the bin's middle (good to 2^-16 each), for top-p; then every CTA sums exact weights,
  //   over all tokens, over those in higher bins, and of the latter, warp by warp, over those that min-p keeps; tokens in the bin itself
  //   go to the list.  The first CTA sorts it, finds the last token kept, and which warp's stretch of the row the choice lies in; that
  //   stretch's CTA finds it there.
  // The histogram of masses only proposes the bin: the exact sums have to confirm it.  Returns false, with nothing written, where that fails
  // (a mark so near the edge of a bin that the proposal fell on the wrong side: one of 5000 rows with top-p, and the call then takes 140 us longer at
  // 128000 tokens; listing the neighbour, too, where the mark is near an edge cost every call 1 %),
  // the list is full (many equal logits), or a parameter is out of this way's range (top-k above 1024, uniform outside (0, 1),
  // temperature, infinities, logits beside which 70 temperatures vanish).  All CTAs of a cluster take the same branches.
  __device__ __forceinline__ bool direct() {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int N = Piece<T>::N;
    const float per_unit = kBinsPerE / r.temperature;
    const bool by_count = r.top_k > 0 && r.top_k < vocab, by_mass = r.top_p < 1.f;
    if (!(r.uniform > 0.f && r.uniform < 1.f) || !(fabsf(top) < 1e30f) || !(r.temperature > 1e-4f && r.temperature < 1e4f) || (by_count && r.top_k > kTopK)) return false;
    // The logit that dead and far ones count as, 70 temperatures below the largest.  Where 32 bits round the difference to at least one step, it is
    // more than 46 temperatures (two thirds), a weight of no units; where they round it to none, this would be the largest logit itself.
    const float floor = top - 70.f * r.temperature;
    if (!by_count && !(floor < top)) return false;
    const double least = (double)r.min_p;
    const int sub = slice / kWarps, warp_base = warp * sub;   // a warp's stretch
    bool groups = by_count && vocab / (kPer * N) >= 2 * r.top_k;
    int n = 0;
    for (;;) {
      int bin = kBins;
      if (by_count || by_mass) {
        bin = find_bin(by_count, groups, per_unit, by_count ? (double)r.top_k : (double)r.top_p);
        // fewer than k tokens outside the last bin; a mark that rounding put between two bins; weights of no units
        if (bin < 0 || (!by_count && bin == kBins - 1)) {
          if (!by_count) return false;
          if (groups) {
            groups = false;
            continue;
          }
          bin = kBins - 2;   // all there are: what lies in the last bin has no units
        }
      }
      unsigned long long named = 0;
      if (by_count) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          if (!groups || bin_of(place(group[g], per_unit)) <= bin) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
              const int i = tid + (g * kPer + k) * kThreads;
              if (i < limit / N) {
                const Piece<T> x = ((const Piece<T>*)logits)[i];
                uint32_t mask = 0;
#pragma unroll
                for (int j = 0; j < N; ++j) mask |= (bin_of(place(L::widen(x.e[j]), per_unit)) <= bin ? 1u : 0u) << j;
                named |= (unsigned long long)mask << ((g * kPer + k) * N);
              }
            }
          }
      } else {
        named = add_up(per_unit, floor, by_mass, bin, sub, warp_base, lane, warp, tid);
      }
      if (by_count || by_mass) {
        n = collect(by_count ? enlist(named, tid, kThreads) : enlist(named, warp_base / N + lane, 32));
        if (n > kList) {
          if (!groups) return false;
          groups = false;
          continue;
        }
      } else {
        sync_row();
      }
      break;
    }
    if (by_count && rank) return true;
    if (rank == 0) {
      constexpr int kAll = RANKS * kWarps, kMine = kList / kThreads;
      if (by_count && n <= kFew) { choose_from_few(n); return true; }
      if (tid == 0) { s.ok = 1; s.cut_entry = 0; s.owner = -1; s.pick = 0; }
      unsigned long long sum_all = 0, sum_below = 0;
      if (!by_count) {
        // the sums of all warps, in index order
#pragma unroll
        for (int k = 0; k < RANKS; ++k) sum_all += s.all[k];
        if (by_mass) block_scan(tid < kAll ? s.below[tid] : 0ull, s.warp_sum, sum_below, lane, warp);
      }
      if (n) {
        sort(n, by_count, per_unit);
        // exact weights of the list, largest first, kMine entries per thread; those kept are the first ones
        const int count = by_count ? min(r.top_k, n) : n;
        unsigned long long unit[kMine], sum = 0, total;
        double w[kMine];
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          const int i = tid * kMine + j;
          w[j] = i < count ? weight(value_of(s.list[i])) : 0.0;
          sum += unit[j] = i < count ? units(w[j]) : 0;
        }
        unsigned long long run = sum_below + block_scan(sum, s.warp_sum, total, lane, warp);
        const double mark = (double)r.top_p * (double)(by_count ? total : sum_all);
        int n_kept = 0;
        sum = 0;
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          const int i = tid * kMine + j;
          const bool in_mass = i < count && (!by_mass || (double)run < mark || (i == 0 && sum_below == 0)), keep = in_mass && w[j] >= least;
          if (by_count) {
            if (keep) { n_kept = i + 1; sum += unit[j]; }
            if (i < kTopK) s.weight[i] = keep ? unit[j] : 0;
          } else if (in_mass) {
            const unsigned long long entry = s.list[i];
            if (!(i + 1 < n && (double)(run + unit[j]) < mark)) s.cut_entry = entry;   // the last of them ends the kept tokens
            if (keep) atomicAdd(&s.taken[~(uint32_t)entry / (uint32_t)sub], unit[j]);
          }
          run += unit[j];
        }
        if (by_count) {
          block_scan(sum, s.warp_sum, total, lane, warp);
          if (n_kept) atomicMax(&s.pick, n_kept);
          __syncthreads();
          choose_by_digits(s.pick, (double)r.uniform * (double)total, lane, warp, tid);
          return true;
        }
        if (tid == 0 && !((sum_below == 0 || (double)sum_below < mark) && mark <= (double)(sum_below + total))) s.ok = 0;
      }
      __syncthreads();
      const unsigned long long taken = tid < kAll ? s.taken[tid] : 0;
      unsigned long long sum_taken;
      const unsigned long long before = block_scan(taken, s.warp_sum, sum_taken, lane, warp);
      const double target = (double)r.uniform * (double)sum_taken;
      if (!((double)before > target) && (double)(before + taken) > target)
        for (int k = 0; k < RANKS; ++k) { Shared* o = peer(k); o->owner = tid; o->before = before; o->target = target; }
      __syncthreads();
      if (tid == 0 && s.owner < 0) s.ok = 0;
      __syncthreads();
      if (tid && tid < RANKS) { Shared* o = peer(tid); o->cut_entry = s.cut_entry; o->ok = s.ok; }
    }
    sync_row();
    if (!s.ok) return false;
    if (s.owner / kWarps != rank) return true;
    // The stretch of one warp, now by all warps of its CTA.  Its tokens and their units are those that were summed (a logit's bin follows from
    // its value, falls as it grows, and every weight of no units counts for nothing in both), so that one of the warps passes the target.
    const Key cut = (Key)(s.cut_entry >> 32);
    const int cut_index = by_mass ? (int)~(uint32_t)s.cut_entry : INT_MAX, stretch = (s.owner - rank * kWarps) * sub, part = (sub / kWarps + 31) & ~31;
    auto chosen = [&](int i) -> unsigned long long {
      if (i >= sub) return 0;
      const T x = logit(stretch + i);
      const Key k = L::key(x);
      if (!k || !(k > cut || (k == cut && base + stretch + i <= cut_index))) return 0;
      const double w = weight(L::widen(x));
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

  // The bin, as a float: nearest to (top - logit) * per_unit, which grows as logits fall; the last one for NaN and -inf.
  __device__ __forceinline__ float place(float v, float per_unit) const { return fminf((top - v) * per_unit, (float)(kBins - 1)); }
  static __device__ __forceinline__ int bin_of(float at) { return (int)(__float_as_uint(at + 8388608.f) & 0x7fffffu); }

  // The bin in which the sum over bins passes `need` (a count, or a share of the mass), or -1.
  __device__ __forceinline__ int find_bin(bool count, bool groups, float per_unit, double need) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < kBins; i += kThreads) s.hist[i] = 0;
    if (tid == 0) s.found = -1;
    __syncthreads();
    if (groups) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int b = bin_of(place(group[g], per_unit));
        if (b < kBins - 1) atomicAdd(&s.hist[b], 1u);
      }
    } else {
#pragma unroll 2
      for (int i = tid; i < limit / Piece<T>::N; i += kThreads) {
        const Piece<T> x = ((const Piece<T>*)logits)[i];
#pragma unroll
        for (int j = 0; j < Piece<T>::N; ++j) {
          const float at = place(L::widen(x.e[j]), per_unit);
          const int b = bin_of(at);
          // 2^16 e^(-(at - b) / 64), |at - b| <= 1/2, to 8e-8 and a whole number.
          const float d = ((at + 8388608.f) - 8388608.f) - at;
          constexpr float c = 1.f / kBinsPerE;
          const uint32_t add = count ? 1u : __float_as_uint(fmaf(fmaf(d, 32768.f * c * c, 65536.f * c), d, 65536.f + 8388608.f)) & 0x7fffffu;
          if (b < kBins - 1) atomicAdd(&s.hist[b], add);
        }
      }
    }
    sync_row();
    // each CTA adds up its share of the bins
    constexpr int kShare = kBins / RANKS, kEach = kShare > kThreads ? kShare / kThreads : 1;
    const int b0 = rank * kShare + tid * kEach;
    unsigned long long v[kEach], sum = 0;   // counts, or masses in units of 2^-40 (a bin holds at most 2^18 of them)
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      v[j] = 0;
      if (tid * kEach < kShare) {
        uint32_t n[RANKS];
#pragma unroll
        for (int k = 0; k < RANKS; ++k) n[k] = peer(k)->hist[b0 + j];
#pragma unroll
        for (int k = 0; k < RANKS; ++k) v[j] += n[k];
        if (!count) v[j] = (unsigned long long)((float)v[j] * exp2f((float)(b0 + j) * (-1.44269504f / kBinsPerE) + 24.f));
      }
      sum += v[j];
    }
    unsigned long long total;
    const unsigned long long before = block_scan(sum, s.warp_sum, total, lane, warp);
    if (tid < RANKS) peer(tid)->shares[rank] = total;
    sync_row();
    unsigned long long offset = 0, everything = 0;
#pragma unroll
    for (int k = 0; k < RANKS; ++k) {
      if (k == rank) offset = everything;
      everything += s.shares[k];
    }
    const double mark = count ? need : need * (double)everything;
    unsigned long long run = offset + before;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if ((double)run < mark && mark <= (double)(run + v[j]))
        for (int k = 0; k < RANKS; ++k) peer(k)->found = b0 + j;
      run += v[j];
    }
    sync_row();
    return s.found;
  }

  // Puts on this CTA's list the logits that `mask` names: bit m of thread t is element m % N of its piece m / N, pieces `first` + (m / N) * `step`.
  // The first kList bits of the row's order need not come first: the list is sorted later.  Returns how many there are.
  __device__ __forceinline__ int enlist(unsigned long long mask, int first, int step) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int all;
    int at = block_scan(__popcll(mask), (int*)s.warp_sum, all, lane, warp);
    while (mask) {
      const int m = __ffsll((long long)mask) - 1, i = (first + m / Piece<T>::N * step) * Piece<T>::N + m % Piece<T>::N;
      mask &= mask - 1;
      if (at < kList) s.list[at] = ((unsigned long long)L::key(logits[i]) << 32) | (uint32_t)~(uint32_t)(base + i);
      ++at;
    }
    return all;
  }
  // The CTAs' lists of n entries, one after the other in the first one's memory.  Returns their length; above kList they are not there.
  __device__ __forceinline__ int collect(int n) {
    const int tid = threadIdx.x;
    if (tid < RANKS) peer(tid)->listed[rank] = n;
    sync_row();
    int offset = 0, all = 0;
#pragma unroll
    for (int k = 0; k < RANKS; ++k) {
      if (k == rank) offset = all;
      all += s.listed[k];
    }
    if (all <= kList) {
      if (rank) {
        Shared* first = peer(0);
        for (int i = tid; i < n; i += kThreads) first->list[offset + i] = s.list[i];
      }
    }
    sync_row();
    return all;
  }
  // The first CTA's list, largest first.  Entries go to buckets, by their bins or, where they all share one, by key and, between equal keys, by
  // index; inside a bucket they are counted, or, where one is crowded, all are sorted by exchanges.
  __device__ __forceinline__ void sort(int n, bool by_bin, float per_unit) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    double spread = 0.0;
    uint32_t high = 0;
    if (!by_bin) {
      if (tid == 0) { s.low_key = ~0u; s.high_key = 0; }
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) { const uint32_t k = (uint32_t)(s.list[i] >> 32); atomicMin(&s.low_key, k); atomicMax(&s.high_key, k); }
      __syncthreads();
      high = s.high_key;
      spread = (double)((float)kBins / ((float)(high - s.low_key) + 1.f));   // (any number will do that all entries share)
    }
    auto place_of = [&](unsigned long long e) {
      if (by_bin) return bin_of(place(value_of(e), per_unit));
      return min(kBins - 1, (int)(((double)(high - (uint32_t)(e >> 32)) + (double)(~(uint32_t)e) * (1.0 / kMaxVocab)) * spread));
    };
    for (int i = tid; i < kBins; i += kThreads) s.bucket[i] = 0;
    if (tid == 0) s.crowded = 0;
    __syncthreads();
    unsigned long long entry[kList / kThreads];
    int b[kList / kThreads];
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j) {
      const int i = j * kThreads + tid;
      if (i < n) {
        entry[j] = s.list[i];
        b[j] = place_of(entry[j]);
        if (atomicAdd(&s.bucket[b[j]], 1u) >= kBucket) s.crowded = 1;
      }
    }
    __syncthreads();
    if (s.crowded) {
      int n2 = 2;
      while (n2 < n) n2 *= 2;
      for (int i = n + tid; i < n2; i += kThreads) s.list[i] = 0;
      sort_list(s.list, n2, tid);
      return;
    }
    uint32_t mine[kBins / kThreads], sum = 0, total;
#pragma unroll
    for (int j = 0; j < kBins / kThreads; ++j) sum += mine[j] = s.bucket[tid * (kBins / kThreads) + j];
    uint32_t run = block_scan(sum, (uint32_t*)s.warp_sum, total, lane, warp);
#pragma unroll
    for (int j = 0; j < kBins / kThreads; ++j) { s.bucket[tid * (kBins / kThreads) + j] = run; run += mine[j]; }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j)
      if (j * kThreads + tid < n) s.spare[atomicAdd(&s.bucket[b[j]], 1u)] = entry[j];
    __syncthreads();
    // (each bucket now names its end, which is the next one's beginning)
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j)
      if (j * kThreads + tid < n) {
        const uint32_t from = b[j] ? s.bucket[b[j] - 1] : 0u, to = s.bucket[b[j]];
        uint32_t rank_of = from;
        for (uint32_t i = from; i < to; ++i) rank_of += s.spare[i] > entry[j];
        s.list[rank_of] = entry[j];
      }
    __syncthreads();
  }
  __device__ __forceinline__ float value_of(unsigned long long entry) const { return L::value((Key)(entry >> 32)); }

  // The choice from a list of up to 128 entries in any order, four threads for each: three rounds in which every entry looks at all others.
  __device__ __forceinline__ void choose_from_few(int n) {
    const int tid = threadIdx.x, i = tid >> 2;
    const bool live = i < n;
    const unsigned long long entry = live ? s.list[i] : 0;
    const double w = live ? weight(value_of(entry)) : 0.0;
    const unsigned long long unit = units(w);
    if (live && (tid & 3) == 0) s.weight[i] = unit;
    if (tid == 0) s.token = INT_MAX;
    __syncthreads();
    auto quad = [](unsigned long long v) { v += __shfl_xor_sync(~0u, v, 1); return v + __shfl_xor_sync(~0u, v, 2); };
    // rank, and the weight of all larger ones; both in one sum: up to 128 of 2^44 units and of 2^56
    unsigned long long sum = 0;
    for (int j = tid & 3; j < n; j += 4)
      if (s.list[j] > entry) sum += s.weight[j] + (1ull << 56);
    sum = quad(sum);
    const int place_in = (int)(sum >> 56);
    const unsigned long long larger = sum & ((1ull << 56) - 1);
    bool keep = live && place_in < r.top_k;
    if (r.top_p < 1.f) {
      __syncthreads();
      if (live && (tid & 3) == 0 && !keep) s.weight[i] = 0;
      __syncthreads();
      unsigned long long total = 0;
      for (int j = 0; j < n; ++j) total += s.weight[j];
      keep = keep && (place_in == 0 || (double)larger < (double)r.top_p * (double)total);
    }
    keep = keep && w >= (double)r.min_p;
    __syncthreads();
    if (live && (tid & 3) == 0) s.weight[i] = keep ? unit : 0;
    __syncthreads();
    unsigned long long upto = 0, total = 0;
    for (int j = tid & 3; j < n; j += 4) {
      total += s.weight[j];
      if (~(uint32_t)s.list[j] <= ~(uint32_t)entry) upto += s.weight[j];
    }
    upto = quad(upto);
    total = quad(total);
    if (keep && (double)upto > (double)r.uniform * (double)total) atomicMin(&s.token, (int)~(uint32_t)entry);
    __syncthreads();
    if (tid == 0) tokens[row] = s.token;
  }

  // From the list's first n_kept entries, with their weights beside them: by index, six bits at a time, the digit at which the running sum
  // passes the target.
  __device__ __forceinline__ void choose_by_digits(int n_kept, double target, int lane, int warp, int tid) {
    uint32_t prefix = 0;
    unsigned long long before = 0;
    for (int shift = 12; shift >= 0; shift -= 6) {
      if (tid < 64) { s.digit_lo[tid] = 0; s.digit_hi[tid] = 0; }
      __syncthreads();
      for (int i = tid; i < n_kept; i += kThreads) {
        const uint32_t index = ~(uint32_t)s.list[i];
        const unsigned long long u = s.weight[i];
        if (u && index >> (shift + 6) == prefix) add_units(&s.digit_lo[(index >> shift) & 63], &s.digit_hi[(index >> shift) & 63], u);
      }
      __syncthreads();
      if (warp == 0) {
        const unsigned long long x = ((unsigned long long)s.digit_hi[2 * lane] << 32) + s.digit_lo[2 * lane], y = ((unsigned long long)s.digit_hi[2 * lane + 1] << 32) + s.digit_lo[2 * lane + 1];
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
  }

  // This CTA's exact sums, into the first CTA's memory; names the logits in the bin.  Logits below `floor`, NaN and -inf among them, become it.
  __device__ __forceinline__ unsigned long long add_up(float per_unit, float floor, bool by_mass, int bin, int sub, int warp_base, int lane, int warp, int tid) {
    constexpr int N = Piece<T>::N;
    Shared* first = peer(0);
    const double least = (double)r.min_p;
    unsigned long long named = 0;
    {
      // (where only min-p chooses, no weight past this place passes it, with room for the roundings of 32 bits)
      const float last = by_mass || !(r.min_p > 0.f) ? kNoUnits : fminf(-kBinsPerE * logf(r.min_p) + 1.f, kNoUnits);
      const bool every = !(r.min_p > 0.f);              // min-p keeps all
      // a thread's sums of units are exact as doubles (64 logits at most); integer additions of two words would cost as much as the weights
      double all = 0, below = 0, taken = 0;
      int shift = 0;
      for (int i = warp_base / N + lane; i < min(warp_base + sub, limit) / N; i += 32, shift += N) {
        const Piece<T> x = ((const Piece<T>*)logits)[i];
        if (place(L::largest(*(const uint4*)&x), per_unit) < last) {
          uint32_t mask = 0;
#pragma unroll
          for (int j0 = 0; j0 < N; j0 += 4) {
            double w[4];
            int b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float v = fmaxf(L::widen(x.e[j0 + j]), floor);
              b[j] = (int)__float_as_uint(__fmul_rn(top - v, per_unit) + 8388608.f) - 0x4b000000;   // (two roundings, as in the histogram)
              w[j] = exp_below<true>((double)v - (double)top, scale, s);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const double u = units_exact(w[j]);
              all += u;
              if (b[j] < bin) {
                below += u;
                if (!every && w[j] >= least) taken += u;
              }
              mask |= (b[j] == bin ? 1u : 0u) << (j0 + j);
            }
          }
          named |= (unsigned long long)mask << shift;
        }
      }
      if (every) taken = below;
      const unsigned long long sum_all = warp_sum((unsigned long long)all), sum_below = warp_sum((unsigned long long)below), sum_taken = warp_sum((unsigned long long)taken);
      if (lane == 0) { s.bucket[2 * warp] = (uint32_t)sum_all; s.bucket[2 * warp + 1] = (uint32_t)(sum_all >> 32); first->below[rank * kWarps + warp] = sum_below; first->taken[rank * kWarps + warp] = sum_taken; }
    }
    __syncthreads();
    if (tid == 0) {
      unsigned long long v = 0;
      for (int k = 0; k < kWarps; ++k) v += ((unsigned long long)s.bucket[2 * k + 1] << 32) + s.bucket[2 * k];
      first->all[rank] = v;
    }
    return named;
  }

  // Any row: one search for top-k and one for top-p, each over 8 bits of the keys at a time from the top.
  __device__ __noinline__ void general() {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ranks = RANKS;
    const Key top_key = key_of_top();
    if (tid < 256) { s.lo[0][tid] = 0; s.hi[0][tid] = 0; }
    __syncthreads();
    auto weight_of = [&](Key k) { return k == top_key ? 1.0 : exp_below<false>((double)L::value(k) - (double)top, scale, s); };
    // Kept so far: key > t, or key == t and index <= c.
    Key t = 1;
    int c = INT_MAX, buffer = 0;
    auto kept = [&](Key k, int i) { return k > t || (k == t && i <= c); };
    // The key at which counts, or masses, summed from the largest key down, reach the mark; `above` is the sum over the larger keys
    // and `in_bin` the sum at the key itself.
    auto search = [&](bool mass, auto reached, bool share_of, double share, unsigned long long& above_out, unsigned long long& bin_out, double& mark) -> Key {
      Key prefix = 0;
      unsigned long long above = 0, in_bin = 0;
      for (int shift = L::kBits - 8; shift >= 0; shift -= 8) {
        for (int i = tid; i < slice; i += kThreads) {
          const Key k = L::key(logit(i));
          if (k && (shift + 8 == L::kBits || (uint32_t)k >> (shift + 8) == (uint32_t)prefix) && kept(k, base + i)) {
            const int b = ((uint32_t)k >> shift) & 255;
            if (mass) {
              const unsigned long long u = units(weight_of(k));
              if (u) add_units(&s.lo[buffer][b], &s.hi[buffer][b], u);
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
          if (share_of && shift + 8 == L::kBits) mark = share * (double)__shfl_sync(~0u, upto, 31);
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
      for (int i = lane; i < sub; i += 32) mine += L::key(logit(warp_base + i)) == key && kept(key, base + warp_base + i);
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
          const bool hit = L::key(logit(warp_base + i + lane)) == key && kept(key, base + warp_base + i + lane);
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
        for (int i = tid; i < slice; i += kThreads) mine += L::key(logit(i)) != 0;
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
      const unsigned long long w = units(weight_of(found));
      if (tid == 0) {
        // the fewest of them with which the sum reaches the mark: the quotient, which roundings can put off by one
        const long long all = w ? (long long)(in_bin / w) : 1;
        long long j = w ? (long long)((mark - (double)above) / (double)w) : 1;
        j = j < 1 ? 1 : j > all ? all : j;
        for (int i = 0; i < 2 && j > 1 && (double)(above + (unsigned long long)(j - 1) * w) >= mark; ++i) --j;
        for (int i = 0; i < 2 && j < all && (double)(above + (unsigned long long)j * w) < mark; ++i) ++j;
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
      const Key k = L::key(logit(i));
      is_kept = false;
      if (!k || !kept(k, base + i)) return 0;
      const double w = weight_of(k);
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
  __device__ __forceinline__ Key key_of_top() const { return L::key(narrow()); }
  __device__ __forceinline__ T narrow() const { return (T)top; }
};

// One cluster of CTAs takes one row, each CTA `slice` consecutive logits, which it reads once and keeps in shared memory; where they do not fit
// (`keep` is 0) the passes after the first read them from the caller's memory again, mostly from L2.  Two CTAs share an SM, so that one
// computes while the other waits: what a row costs beside its loads and weights is a chain of barriers.  The logits are no __restrict__ constants: the
// kernel may begin while the one in front still writes them, and loads that count on memory which nobody writes are not for it.
template <typename T, int RANKS>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const T* logits, int64_t row_stride, int vocab, int slice, int vec, int keep, const __grid_constant__ Powers powers,
                                                          const float* temperature, const int* top_k, const float* top_p, const float* min_p, const float* uniform, int* tokens) {
  using L = Logits<T>;
  using P = Part<T, RANKS>;
  extern __shared__ __align__(16) uint8_t dynamic[];
  Shared& s = *(Shared*)dynamic;
  constexpr int N = Piece<T>::N;
  cg::cluster_group cluster = cg::this_cluster();
  if (RANKS > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // (its other half stands before the first access to a peer's memory)
  auto peer = [&](int k) { return RANKS == 1 ? &s : cluster.map_shared_rank(&s, k); };
  const int rank = RANKS == 1 ? 0 : (int)cluster.block_rank(), row = blockIdx.x / RANKS, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, base = rank * slice;
  const T* src = logits + (int64_t)row * row_stride + base;
  T* mine = keep ? (T*)(dynamic + sizeof(Shared)) : (T*)src;
  const int here = max(0, min(slice, vocab - base));
  asm volatile("griddepcontrol.wait;" ::: "memory");   // (launched while the kernel in front may still be writing the logits)
  float group[P::kGroups], top = -INFINITY;
  if (!vec) {   // (then the slice goes to shared memory)
    for (int i = tid; i < slice; i += kThreads) mine[i] = i < here ? src[i] : L::dead();
    __syncthreads();
  }
  const T* from = vec ? src : mine;
  const int readable = vec ? here : slice;
#pragma unroll
  for (int g = 0; g < P::kGroups; ++g) {
    group[g] = -INFINITY;
#pragma unroll
    for (int k = 0; k < P::kPer; ++k) {
      const int i = (tid + (g * P::kPer + k) * kThreads) * N;
      if (i + N <= readable) {
        const uint4 u = *(const uint4*)(from + i);
        if (vec && keep) *(uint4*)(mine + i) = u;
        group[g] = fmaxf(group[g], L::largest(u));
      } else if (vec && keep && i < slice) {   // past the row's last 16 bytes, and past the row
#pragma unroll 1
        for (int j = i; j < i + N; ++j) {
          const T x = j < here ? src[j] : L::dead();
          mine[j] = x;
          group[g] = fmaxf(group[g], L::widen(x));
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < P::kGroups; ++g) top = fmaxf(top, group[g]);
  static_assert(kTable * kCopies <= kThreads, "an entry per thread");
  if (tid < kTable * kCopies) s.table[tid / kCopies][tid % kCopies] = powers.of[tid / kCopies];
  const Row r{temperature ? temperature[row] : 1.f, top_p ? top_p[row] : 1.f, min_p ? fminf(min_p[row], 1.f) : 0.f, uniform[row], top_k ? top_k[row] : 0};
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if (lane == 0) s.warp_top[warp] = top;
  if (tid == 0) s.token = INT_MAX;
  if (RANKS > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // all CTAs of the cluster have begun
  __syncthreads();
  if (tid < RANKS) {
#pragma unroll
    for (int k = 0; k < kWarps; ++k) top = fmaxf(top, s.warp_top[k]);
    peer(tid)->tops[rank] = top;
  }
  if (RANKS == 1) __syncthreads(); else cluster.sync();
#pragma unroll
  for (int k = 0; k < RANKS; ++k) top = fmaxf(top, s.tops[k]);
  top += 0.f;   // (of two zeros the positive one)
  if (!(top > -INFINITY) || !(r.temperature > 0.f)) {
    // nothing to choose from, or the lowest index of the largest logit
    if (top > -INFINITY) {
      int at = INT_MAX;
#pragma unroll
      for (int g = 0; g < P::kGroups; ++g)
        if (group[g] == top && at == INT_MAX)
          for (int i = 0; i < P::kPer * N; ++i) {
            const int e = (tid + (g * P::kPer + i / N) * kThreads) * N + i % N;
            if (e < here && L::widen(mine[e]) == top) { at = base + e; break; }
          }
      at = __reduce_min_sync(~0u, at);
      if (lane == 0 && at < INT_MAX) atomicMin(&peer(0)->token, at);
      if (RANKS == 1) __syncthreads(); else cluster.sync();
    }
    if (rank == 0 && tid == 0) tokens[row] = top > -INFINITY ? s.token : -1;
    return;
  }
  P part{s, cluster, mine, r, top, {}, 0.0, vocab, slice, keep ? slice : here, base, rank, row, tokens};
#pragma unroll
  for (int g = 0; g < P::kGroups; ++g) part.group[g] = group[g];
  part.scale = 46.166241308446828384 / (double)r.temperature;   // 32 / ln 2
  if (part.direct()) return;
  P copy = part;   // (general() takes its address, which would put the registers of the other way in memory, too: 5000 clocks a row)
  copy.general();
}

template <typename T> auto kernel_of(int ranks) { return ranks == 1 ? sample_kernel<T, 1> : ranks == 2 ? sample_kernel<T, 2> : ranks == 4 ? sample_kernel<T, 4> : sample_kernel<T, 8>; }

template <typename T>
int launch(int rows, int vocab, int64_t row, const void* logits, const float* temperature, const int* top_k, const float* top_p, const float* min_p, const float* uniform, int* tokens,
           cudaStream_t stream) {
  // A slice goes to shared memory where it fits; it has to where a row is no number of aligned 16 bytes, because only the first pass reads
  // single logits.
  constexpr size_t kKeep = 64 * 1024;   // two CTAs to an SM
  const int vec = (uintptr_t)logits % 16 == 0 && row * sizeof(T) % 16 == 0;
  const bool must = !vec || vocab % (16 / (int)sizeof(T));
  int ranks = 1;
  auto slice_of = [&](int n) { return ((vocab + n - 1) / n + kThreads - 1) / kThreads * kThreads; };
  while (ranks < kMaxCluster && (slice_of(ranks) > kSlice || (rows * ranks < 148 && slice_of(ranks) > 2048))) ranks *= 2;
  const int slice = slice_of(ranks);
  const int keep = must || slice * sizeof(T) <= kKeep;
  const size_t smem = sizeof(Shared) + (keep ? (size_t)slice * sizeof(T) : 0);
  static const Powers powers = [] { Powers p; for (int j = 0; j < kTable; ++j) p.of[j] = std::exp2((double)j / kTable); return p; }();
  auto* fn = kernel_of<T>(ranks);
  // The kernel's limit is one for all host threads: always that of the longest slice, so that no call lowers it under another's launch.
  constexpr size_t kMost = sizeof(Shared) + kSlice * sizeof(T);
  static_assert(kMost <= 227 * 1024 && kMaxVocab <= kSlice * kMaxCluster, "any slice fits");
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost) != cudaSuccess) { cudaGetLastError(); return -2; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * (unsigned)ranks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, (const T*)logits, row, vocab, slice, vec, keep, powers, temperature, top_k, top_p, min_p, uniform, tokens);
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
