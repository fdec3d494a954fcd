// Attention of the new tokens of each sequence of a batch over a paged cache.
#include <algorithm>
#include <cstdlib>

#include "attention.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kRows = 256, kStep = 128, kRing = 4, kLoaders = 2, kThreads = 12 * 32, kMaxShare = 16;
constexpr uint32_t kBox = 16384;   // 128 rows of 128 bytes

struct Params {
  ChunkAttention a;
  int group;                       // query heads of a cache head; rows of a sequence = its new tokens * group
  int tiles, share;                // tiles of 256 rows that the batch can have; CTAs (a cluster) that share a tile's positions
  float scale_log2e;
  int box_shift;                   // keys and values arrive in boxes of 1 << box_shift positions by TMA; 0: by 16-byte copies only
  uint32_t spin_limit;
  int test_skip_stage;             // test hook, as in kernels_umma.cu: block 0's second unit is neither loaded nor announced
};

struct Shared {
  float2 stat[kRows];       // reference (a base-2 exponent) and sum of each row
  uint64_t full[kRing], empty[kRing], clean[kRing], q_full, s_full[2], p_half[2], p_full[2], o_done[2], handed, drained;
  uint32_t seen[4][4];      // which of a step's positions lie on pages that are there; a step's words are written at most two steps ahead
  uint32_t tmem;
  int abort, odd;           // odd: values that not all rows see, infinite or no numbers, were taken out of the products
  int scan[kThreads / 32], found, sequence, tile;
};

__device__ __forceinline__ float2 load_remote2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
template <int N> __device__ __forceinline__ void load_remote(uint32_t at, float (&v)[N]) {
  if constexpr (N == 4) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at) : "memory");
  else asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(at) : "memory");
}
__device__ __forceinline__ bool odd16(uint32_t u, bool bf16) {   // one of two elements is infinite or no number
  const uint32_t e = bf16 ? 0x7f80u : 0x7c00u;
  return (u & e) == e || (u >> 16 & e) == e;
}

// What a row sees of values that are infinite or no numbers, and that stay out of the products of a step that not all rows see whole: position for
// position, from memory, onto its result (a weight is not zero, so that an infinity remains one).  Rare, and slow.
template <typename T, int D> __device__ __noinline__ void add_odd(const Params& p, uint32_t row_at, bool wide, int head, const int* pages, int from, int to) {
  for (int pos = from; pos < to; ++pos) {
    const int page = pages[pos / p.a.page_size];
    if (page < 0 || page >= p.a.pages) continue;
    const uint32_t* v = (const uint32_t*)((const T*)p.a.v + page * p.a.c_page + (int64_t)(pos % p.a.page_size) * p.a.c_token + (int64_t)head * p.a.c_head);
    for (int c = 0; c < D / 2; ++c) {
      const uint32_t u = v[c];
      if (!odd16(u, Mma<T>::kBf16)) continue;
      for (int h = 0; h < 2; ++h) {
        const uint32_t e = h ? u >> 16 : u & 0xffffu;
        if (!odd16(e, Mma<T>::kBf16)) continue;
        const float x = Mma<T>::kBf16 ? __uint_as_float(e << 16) : __half2float(__ushort_as_half((unsigned short)e));
        if (wide) {
          float y;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(row_at + (2 * c + h) * 4) : "memory");
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(row_at + (2 * c + h) * 4), "f"(y + x) : "memory");
        } else {
          unsigned short y;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(row_at + (2 * c + h) * 2) : "memory");
          const float z = (Mma<T>::kBf16 ? __uint_as_float((uint32_t)y << 16) : __half2float(__ushort_as_half(y))) + x;
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(row_at + (2 * c + h) * 2), "h"((unsigned short)(Mma<T>::pack(z, 0.f) & 0xffffu)) : "memory");
        }
      }
    }
  }
}

// Up to 256 rows (token, query head of one cache head's group; two tiles of 128) of one sequence against the positions that they see, 128 at a
// time: first the prefix's, then the sequence's own.  S = Q K^T goes to tensor memory; a thread per row turns it into weights, which replace it there
// as the A operand of O += P V, and O stays in tensor memory.  A row's reference is not its running maximum but one that follows it only when it
// has been passed by more than 2^8, so that O is rarely rescaled; in fp16, which has no numbers below 2^-24, it lies 2^7 lower, so that the many small weights
// of a long context count together.
// Rows are counted token by token, the heads of the group side by side: a tile covers few tokens, and little of its last steps is hidden from it.  Up to 128
// rows leave the second tile free: it takes the same rows against every other step (`split`), and hands its sums to the first at the end.
// Where tiles are few, the CTAs of a cluster share the positions of each, by the lengths that they find, and every one joins some of the rows
// out of the others' shared memory.
// A weight of zero does not hide an infinity: in steps that some rows see less of than others, values that are infinite or no numbers are taken
// out of shared memory before the product (and positions behind the last one, whatever lies there), and added to the rows that see them at the end.
// Warps 0-3 and 4-7: softmax of a tile each; 8 and 9: loads; 10: products; 11: values of steps that not all see.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
chunk_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap keys, const __grid_constant__ CUtensorMap values) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared w;
  constexpr int kBoxes = D / 64, kPieces = D / 8;
  constexpr uint32_t kUnit = kBoxes * kBox;
  const uint32_t smem = (shared_address(smem_raw) + 1023u) & ~1023u, s_q = smem, s_ring = smem + 2 * kUnit;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x / p.share, rank = blockIdx.x - item * p.share, head = item % p.a.kv_heads;
  grid_dependency_wait();
  launch_dependents();
  // ---- the sequence that this tile is of: the last ones, which see the most, begin first ----
  {
    const int flat = p.tiles - 1 - item / p.a.kv_heads;
    int before = 0;
    if (threadIdx.x == 0) w.found = 0;
    for (int b0 = 0; b0 < p.a.batch; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      int n = 0;
      if (b < p.a.batch) {
        const int lo = max(0, min(p.a.starts[b], p.a.tokens)), hi = max(lo, min(p.a.starts[b + 1], p.a.tokens));
        n = ((hi - lo) * p.group + kRows - 1) / kRows;
      }
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
      }
      __syncthreads();
      if (lane == 31) w.scan[warp] = upto;
      __syncthreads();
      int all = 0;
      for (int i = 0; i < kThreads / 32; ++i) {
        if (i < warp) upto += w.scan[i];
        all += w.scan[i];
      }
      if (flat >= before + upto - n && flat < before + upto) { w.found = 1; w.sequence = b; w.tile = flat - (before + upto - n); }
      before += all;
      if (before > flat) break;
    }
    __syncthreads();
    if (!w.found) return;   // (all of a cluster)
  }
  const int b = w.sequence, first_row = max(0, min(p.a.starts[b], p.a.tokens)), count = max(first_row, min(p.a.starts[b + 1], p.a.tokens)) - first_row;
  const int row0 = w.tile * kRows, n_rows = min(kRows, count * p.group - row0);
  const int length = (int)min((long long)max(p.a.lengths[b], 0), (long long)p.a.table_width * p.a.page_size);
  const int* own_pages = p.a.page_table + (int64_t)b * p.a.table_width;
  // own positions that row r of the sequence sees
  auto limit_of = [&](int r) { return max(0, length - count + r / p.group + 1); };
  const int prefix_steps = (p.a.prefix_length + kStep - 1) / kStep;
  const int least = limit_of(row0), most = limit_of(row0 + n_rows - 1);   // of this tile's first and last row
  const bool split = n_rows <= 128;
  // steps of the whole tile, this CTA's share of them, and how many of those each half of the rows takes part in
  const int all_steps = prefix_steps + (most + kStep - 1) / kStep;
  const int first = (int)((int64_t)all_steps * rank / p.share), steps = (int)((int64_t)all_steps * (rank + 1) / p.share) - first;
  int takes_part[2];
  if (split) {
    takes_part[0] = (steps + 1) / 2;
    takes_part[1] = steps / 2;
  } else {
    takes_part[0] = max(0, min(steps, prefix_steps + (limit_of(row0 + 127) + kStep - 1) / kStep - first));
    takes_part[1] = steps;
  }
  // step i of this CTA: where it begins in its segment, where the segment ends (for the last row), its pages
  auto begin_of = [&](int i) { return (first + i < prefix_steps ? first + i : first + i - prefix_steps) * kStep; };
  auto end_of = [&](int i) { return first + i < prefix_steps ? p.a.prefix_length : most; };
  auto pages_of = [&](int i) { return first + i < prefix_steps ? p.a.prefix_pages : own_pages; };
  constexpr uint32_t kColumns = 512;
  if (threadIdx.x == 0) {
    if (p.box_shift) { prefetch_map(&keys); prefetch_map(&values); }
    for (int i = 0; i < kRing; ++i) { mbar_init(&w.full[i], kLoaders * 33); mbar_init(&w.empty[i], 1); mbar_init(&w.clean[i], 1); }
    mbar_init(&w.q_full, split ? 4 : 8);
    for (int t = 0; t < 2; ++t) { mbar_init(&w.s_full[t], 1); mbar_init(&w.p_half[t], 4); mbar_init(&w.p_full[t], 4); mbar_init(&w.o_done[t], 1); }
    mbar_init(&w.handed, 4);
    mbar_init(&w.drained, 1);
    w.abort = 0;
    w.odd = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_proxy();
  }
  if (warp == 8 + kLoaders) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&w.tmem)), "r"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = w.tmem;
  volatile int* abort_flag = &w.abort;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, nullptr, 0, p.spin_limit); };
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(~0u, wait(bar, parity)); };   // one answer for the warp
  constexpr uint32_t kWideRow = D * 4 + 16, kNarrowRow = D * 2 + 16;   // (16 bytes apart from each other's banks)

  if (warp < 8) {
    // ------------------------------------------------------------------- softmax ----
    const int tile = warp >> 2, quarter = warp & 3, in_tile = quarter * 32 + lane, r = split ? in_tile : tile * 128 + in_tile;
    const bool live = r < n_rows;
    const int row = row0 + (live ? r : n_rows - 1), j = row / p.group, g = row - j * p.group;
    const int limit = limit_of(row);
    // (a negative scale becomes the sign of the queries: the largest score is then the largest product)
    if (!(split && tile)) {
      const uint4* q = (const uint4*)((const T*)p.a.q + (int64_t)(first_row + j) * p.a.q_token + (int64_t)(head * p.group + g) * p.a.q_head);
      const uint32_t sign = p.scale_log2e < 0.f ? 0x80008000u : 0u;
      const uint32_t s_row = s_q + tile * kUnit + in_tile * 128;
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        uint4 u = live ? q[c] : make_uint4(0, 0, 0, 0);
        u.x ^= sign; u.y ^= sign; u.z ^= sign; u.w ^= sign;
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(s_row + (c >> 3) * kBox + (((c & 7) ^ (r & 7)) << 4)), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&w.q_full);
    }
    const float scale = fabsf(p.scale_log2e);
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, t_s = tmem + tile * 128 + lanes, t_o = tmem + 256 + tile * D + lanes;
    float reference = -INFINITY, sum = 0.f;
    bool ok = true;
    const int own_steps = takes_part[tile];
    for (int i = 0; i < own_steps; ++i) {
      const int step = split ? 2 * i + tile : i;
      if (!warp_wait(&w.s_full[tile], i & 1)) { ok = false; break; }
      tc_fence_after();
      uint32_t seen[4];
      const int sees = (first + step < prefix_steps ? p.a.prefix_length : limit) - begin_of(step);   // positions of this step, if their pages are there
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        seen[c] = *(volatile uint32_t*)&w.seen[step & 3][c];
        seen[c] &= sees >= 32 * (c + 1) ? ~0u : sees <= 32 * c ? 0u : (1u << (sees - 32 * c)) - 1u;
      }
      const bool whole = __all_sync(~0u, (seen[0] & seen[1] & seen[2] & seen[3]) == ~0u);
      float mx = -INFINITY;
      auto largest = [&](auto all) {
        uint32_t v[2][32];
        tmem_ld32(t_s, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld_wait32(v[c & 1]);
          if (c < 3) tmem_ld32(t_s + (c + 1) * 32, v[(c + 1) & 1]);
          float m4[4] = {mx, mx, mx, mx};
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float x[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = decltype(all)::value || (seen[c] >> (k + h) & 1) ? __uint_as_float(v[c & 1][k + h]) : -INFINITY;
            m4[k >> 1 & 3] = fmaxf(m4[k >> 1 & 3], fmaxf(x[0], x[1]));
          }
          mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        }
      };
      if (whole) largest(True()); else largest(False());
      mx = mx == -INFINITY ? mx : mx * scale - Mma<T>::kLift;   // (a scale of zero keeps it a number)
      const bool passed = mx > (i ? reference + 8.f : -INFINITY);
      if (__any_sync(~0u, passed)) {
        const float next = passed ? mx : reference, corr = passed ? exp2_fast(reference - mx) : 1.f;
        reference = next;
        sum *= corr;
        if (i) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t v[32];
            tmem_ld32(t_o + c * 32, v);
            tmem_ld_wait32(v);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t u[16];
#pragma unroll
              for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(__uint_as_float(v[h * 16 + k]) * corr);
              tmem_st16(t_o + c * 32 + h * 16, u);
            }
          }
          tmem_st_wait();
        }
      }
      const float base = reference == -INFINITY ? 0.f : reference;
      const uint64_t scale2 = pair_of(scale, scale), base2 = pair_of(-base, -base);
      auto weights = [&](auto all) {
        uint32_t v[2][32], u[16];
        uint64_t part = 0;   // two zeros
        tmem_ld32(t_s, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_ld_wait32(v[c & 1]);
          if (c < 3) tmem_ld32(t_s + (c + 1) * 32, v[(c + 1) & 1]);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float e[2];
            const uint64_t x = fma2(pair_of(v[c & 1][2 * k], v[c & 1][2 * k + 1]), scale2, base2);
            if (k % 4 == 3) exp2_pair(x, e); else { unpack(x, e); e[0] = exp2_fast(e[0]); e[1] = exp2_fast(e[1]); }
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (!decltype(all)::value && !(seen[c] >> (2 * k + h) & 1)) e[h] = 0.f;
            part = add2(part, pair_of(e[0], e[1]));
            u[k] = Mma<T>::pack(e[0], e[1]);
          }
          tmem_st16(t_s + c * 16, u);   // (over scores that have been read)
          if (c == 1) {   // the first half of the weights can be multiplied
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&w.p_half[tile]);
          }
        }
        float e[2];
        unpack(part, e);
        sum += e[0] + e[1];
      };
      if (whole) weights(True()); else weights(False());
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&w.p_full[tile]);
    }
    // All products done, queries and ring are free: the rows of the result go there, and each on as one copy, or to the CTAs that join them.
    if (ok && takes_part[0]) ok = warp_wait(&w.o_done[0], 0);
    if (ok && takes_part[1]) ok = warp_wait(&w.o_done[1], 0);
    tc_fence_after();
    const bool hands = split && tile, takes = split && !tile && steps > 1, shared = p.share > 1;
    const uint32_t wide_at = smem + (uint32_t)r * kWideRow;
    if (hands) w.stat[128 + in_tile] = make_float2(ok ? reference : 0.f, ok ? sum : __int_as_float(0x7fc00000));
    float mine = 1.f, theirs = 0.f;
    if (takes) {
      if (ok) ok = warp_wait(&w.handed, 0);
      if (ok) {
        const float2 st = w.stat[128 + in_tile];
        const float top = fmaxf(reference, st.x), base = top == -INFINITY ? 0.f : top;
        mine = exp2_fast(reference - base);
        theirs = exp2_fast(st.x - base);
        sum = sum * mine + st.y * theirs;
        reference = top;
      }
    }
    const float inverse = shared || hands ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
    const bool wide = hands || shared;
    // narrow rows lie behind the wide ones that the second tile hands over
    const uint32_t row_at = wide ? wide_at : smem + (split ? 128 * kWideRow : 0) + (uint32_t)r * kNarrowRow;
    if (ok && (own_steps || !hands)) {   // (nothing to hand over: the first tile does not wait, and its rows lie there)
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (own_steps) {
          tmem_ld32(t_o + c * 32, v);
          tmem_ld_wait32(v);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = 0;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float x[4] = {__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]), __uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3])};
          if (takes) {
            float y[4];
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]) : "r"(wide_at + c * 128 + k * 16) : "memory");
#pragma unroll
            for (int h = 0; h < 4; ++h) x[h] = x[h] * mine + y[h] * theirs;
          }
          if (wide) {
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(row_at + c * 128 + k * 16), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]) : "memory");
          } else {
            const uint32_t lo = Mma<T>::pack(x[0] * inverse, x[1] * inverse), hi = Mma<T>::pack(x[2] * inverse, x[3] * inverse);
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(row_at + c * 64 + k * 8), "r"(lo), "r"(hi) : "memory");
          }
        }
      }
    }
    if (hands) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&w.handed);
    } else {
      if (ok && *(volatile int*)&w.odd && live) {   // positions of this CTA's steps that this row sees and others do not
        const int from = max(least, steps ? (max(first, prefix_steps) - prefix_steps) * kStep : 0), to = min(limit, (first + steps - prefix_steps) * kStep);
        add_odd<T, D>(p, row_at, wide, head, own_pages, from, to);
      }
      if (shared) {
        w.stat[r] = make_float2(ok ? reference : 0.f, ok ? sum : __int_as_float(0x7fc00000));
      } else if (live) {
        T* y = (T*)p.a.y + (int64_t)(first_row + j) * p.a.y_token + (int64_t)(head * p.group + g) * p.a.y_head;
        if (ok) {
          fence_async_proxy();
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(y), "r"(row_at), "n"(D * 2) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        } else {
          for (int c = 0; c < kPieces; ++c) ((uint4*)y)[c] = make_uint4(~0u, ~0u, ~0u, ~0u);   // (no numbers)
        }
      }
    }
    tc_fence_before();
  } else if (warp < 8 + kLoaders) {
    // --------------------------------------------------------------------- loads ----
    const int part = warp - 8;
    const T *kc = (const T*)p.a.k + (int64_t)head * p.a.c_head, *vc = (const T*)p.a.v + (int64_t)head * p.a.c_head;
    // Page numbers are asked for one step early: of the box that this lane brings, or of the positions whose copies it knows the address of.
    constexpr int kEach = 4 / kLoaders;   // groups of 32 positions
    int page[kEach], box_page = -1;
    int64_t off[kEach];
    const int boxes = p.box_shift ? kStep >> p.box_shift : 0;
    auto position = [&](int step, int h) { return begin_of(step) + (part * kEach + h) * 32 + lane; };
    auto ask = [&](int step) {
      if (step >= steps) return;
      if (p.box_shift) {
        const int at = begin_of(step) + (lane << p.box_shift);
        box_page = lane < boxes && at < end_of(step) ? pages_of(step)[at / p.a.page_size] : -1;
      } else {
#pragma unroll
        for (int h = 0; h < kEach; ++h) page[h] = position(step, h) < end_of(step) ? pages_of(step)[position(step, h) / p.a.page_size] : -1;
      }
    };
    int box_coord = 0, box_at = 0, loaded = 0;
    ask(0);
    for (int u = 0; u < 2 * steps; loaded = ++u) {
      const int step = u >> 1;
      uint64_t* full = &w.full[u % kRing];
      const uint32_t dst = s_ring + (u % kRing) * kUnit;
      if (!warp_wait(&w.empty[u % kRing], ((u / kRing) & 1) ^ 1)) break;
      const bool skip = p.test_skip_stage && blockIdx.x == 0 && u == 1;
      if (p.box_shift) {
        if (!(u & 1)) {
          const bool there = box_page >= 0 && box_page < p.a.pages;
          box_coord = there ? box_page : p.a.pages;   // (past the last page: zeros)
          box_at = (begin_of(step) + (lane << p.box_shift)) % p.a.page_size;
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const uint32_t seen = __ballot_sync(~0u, __shfl_sync(~0u, there, (h * 32 + lane) >> p.box_shift));
            if (lane == 0 && part == 0) *(volatile uint32_t*)&w.seen[step & 3][h] = seen;
          }
          ask(step + 1);
        }
        if (skip) continue;
        mbar_arrive(full);
        if (lane == 0) { if (part == 0) mbar_expect_tx(full, kUnit); else mbar_arrive(full); }
        if (part == 0 && lane < boxes) {
#pragma unroll
          for (int c = 0; c < kBoxes; ++c) load_box(dst + c * kBox + (lane << p.box_shift) * 128, (u & 1) ? &values : &keys, full, c * 64, box_at, head, box_coord);
        }
        continue;
      }
      if (!(u & 1)) {
#pragma unroll
        for (int h = 0; h < kEach; ++h) {
          off[h] = page[h] >= 0 && page[h] < p.a.pages ? page[h] * p.a.c_page + (int64_t)(position(step, h) % p.a.page_size) * p.a.c_token : -1;
          const uint32_t seen = __ballot_sync(~0u, off[h] >= 0);
          if (lane == 0) *(volatile uint32_t*)&w.seen[step & 3][part * kEach + h] = seen;
        }
        ask(step + 1);
      }
      const T* base = (u & 1) ? vc : kc;
#pragma unroll
      for (int h = 0; h < kEach; ++h) {
        const uint32_t row0_at = dst + (part * kEach + h) * 32 * 128;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int n = i * 32 + lane, at = n / kPieces, c = n % kPieces;
          const int64_t o = __shfl_sync(~0u, off[h], at);
          copy16(row0_at + (c >> 3) * kBox + at * 128 + (((c & 7) ^ (at & 7)) << 4), base + (o < 0 ? 0 : o) + c * 8, o >= 0);
        }
      }
      // Each thread's copies announce themselves when they have landed, so that this warp goes on to the next unit at once; lane 0's own
      // arrival publishes `seen`.
      if (!skip) {
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full)) : "memory");
        if (lane == 0) mbar_arrive(full);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (*abort_flag && lane == 0)
      for (int i = 0; i < kRing; ++i) await_landing(&w.full[i], loaded > i ? (uint32_t)((loaded - 1 - i) / kRing & 1) : 1u);   // boxes in flight land before their memory goes
  } else if (warp == 8 + kLoaders && elect_one()) {
    // ------------------------------------------------------------------ products ----
    const uint32_t fmt = Mma<T>::kBf16 ? 1u : 0u, common = (1u << 4) | (fmt << 7) | (fmt << 10) | (8u << 24);
    const uint32_t idesc_s = common | ((uint32_t)(kStep >> 3) << 17), idesc_o = common | (1u << 16) | ((uint32_t)(D >> 3) << 17);   // (V lies with channels innermost)
    const uint64_t hi = (uint64_t)(((8u * 128u) >> 4) | (1u << 14) | (2u << 29)) << 32;
    // the distance between two boxes of channels is only read for V, whose 64-channel groups are a box apart
    auto desc = [&](uint32_t at, uint32_t lead) { return hi | ((uint64_t)lead << 16) | (uint64_t)((at & 0x3FFFF) >> 4); };
    // (keys and values were written by copies or stores of other threads, which the barrier has told of: the fence makes them visible to the products)
    auto landed = [&](uint64_t* bars, int u) {
      const bool there = wait(&bars[u % kRing], (u / kRing) & 1);
      fence_async_proxy();
      return there;
    };
    bool ok = steps == 0 || wait(&w.q_full, 0);
    auto scores = [&](int i, int t) {   // S_t = Q_t K_i^T
      const uint32_t k = s_ring + (2 * i % kRing) * kUnit, q = s_q + (split ? 0u : t * kUnit);
#pragma unroll
      for (int n = 0; n < D / 16; ++n)
        umma_f16(tmem + t * 128, desc(q + (n >> 2) * kBox + (n & 3) * 32, 1), desc(k + (n >> 2) * kBox + (n & 3) * 32, 1), idesc_s, n ? 1u : 0u);
      umma_commit(&w.s_full[t]);
    };
    // Every tile takes every step that its rows see any of; split, step i belongs to tile i & 1, whose next one is i + 2.
    const int ahead = split ? 2 : 1;
    auto has = [&](int i, int t) { return split ? (i & 1) == t : i < takes_part[t]; };
    for (int i = 0; i < min(ahead, steps) && ok; ++i) {
      ok = landed(w.full, 2 * i);
      if (!ok) break;
      tc_fence_after();
      for (int t = 0; t < 2; ++t) if (has(i, t)) scores(i, t);
      umma_commit(&w.empty[2 * i % kRing]);
    }
    for (int i = 0; i < steps && ok; ++i) {
      const int vu = 2 * i + 1, ku = 2 * (i + ahead), turn = split ? i >> 1 : i;
      const bool more = i + ahead < steps;
      ok = landed(w.clean, vu);
      bool keys_there = false;
      for (int t = 0; t < 2 && ok; ++t) {
        if (!has(i, t)) continue;
        const uint32_t v = s_ring + (vu % kRing) * kUnit;
#pragma unroll
        for (int h = 0; h < 2; ++h) {   // half of the weights while the other half is worked out
          ok = ok && wait(h ? &w.p_full[t] : &w.p_half[t], turn & 1);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int n = h * 4; n < h * 4 + 4; ++n)
            umma_tmem_a(tmem + 256 + t * D, tmem + t * 128 + n * 8, desc(v + n * 2048, kBox >> 4), idesc_o, (turn || n) ? 1u : 0u);
        }
        if (!ok) break;
        if (t == 1 || split) umma_commit(&w.empty[vu % kRing]);
        if (!more || !has(i + ahead, t)) { umma_commit(&w.o_done[t]); continue; }
        if (!keys_there) { ok = landed(w.full, ku); keys_there = true; }
        if (!ok) break;
        tc_fence_after();
        scores(i + ahead, t);
        if (t == 1 || split) umma_commit(&w.empty[ku % kRing]);
      }
    }
    if (!ok) { umma_commit(&w.drained); await_landing(&w.drained, 0); }   // products in flight end before their memory goes
  } else if (warp == 9 + kLoaders) {
    // ------------------------------------------- values of steps that not all rows see ----
    for (int i = 0; i < steps; ++i) {
      const int u = 2 * i + 1;
      if (!warp_wait(&w.full[u % kRing], (u / kRing) & 1)) break;
      const int from = (first + i < prefix_steps ? p.a.prefix_length : least) - begin_of(i), end = end_of(i) - begin_of(i);   // seen by all; by any
      if (from < kStep) {
        const uint32_t at = s_ring + (u % kRing) * kUnit;
        bool any = false;
        for (int n = max(from, 0) * kPieces + lane; n < kStep * kPieces; n += 32) {
          const int pos = n / kPieces, c = n % kPieces;
          const uint32_t to = at + (c >> 3) * kBox + pos * 128 + (((c & 7) ^ (pos & 7)) << 4);
          uint32_t x[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(to) : "memory");
          bool store = pos >= end;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (pos >= end) x[k] = 0;
            else if (odd16(x[k], Mma<T>::kBf16)) {
              store = any = true;
              x[k] &= (odd16(x[k] & 0xffffu, Mma<T>::kBf16) ? 0u : 0xffffu) | (odd16(x[k] >> 16, Mma<T>::kBf16) ? 0u : 0xffff0000u);
            }
          }
          if (store) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
        }
        if (any) *(volatile int*)&w.odd = 1;
        fence_async_proxy();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&w.clean[u % kRing]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8 + kLoaders) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
  if (p.share > 1) {
    // ---- each CTA joins the rows that are its own modulo the cluster's size ----
    cluster_sync_all();
    constexpr int N = D / 32;
    const uint32_t stat = smem_u32(w.stat);
    for (int r = rank + p.share * warp; r < n_rows; r += p.share * (kThreads / 32)) {
      float2 st[kMaxShare];
      float top = -INFINITY, sum = 0.f, acc[N];
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = 0.f;
#pragma unroll
      for (int i = 0; i < kMaxShare; ++i)
        if (i < p.share) {
          st[i] = load_remote2(map_to_cta(stat + r * 8, i));
          top = fmaxf(top, st[i].x);
        }
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int i = 0; i < kMaxShare; ++i)
        if (i < p.share && st[i].y != 0.f) {   // (a share without positions wrote no row)
          float x[N];
          load_remote<N>(map_to_cta(smem + (uint32_t)r * kWideRow + lane * (N * 4), i), x);
          const float f = exp2_fast(st[i].x - base);
          sum += f * st[i].y;
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += f * x[k];
        }
      const int row = row0 + r, j = row / p.group, g = row - j * p.group;
      T* y = (T*)p.a.y + (int64_t)(first_row + j) * p.a.y_token + (int64_t)(head * p.group + g) * p.a.y_head + lane * N;
      const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int k = 0; k < N; k += 2) *(uint32_t*)(y + k) = Mma<T>::pack(acc[k] * inverse, acc[k + 1] * inverse);
    }
    cluster_sync_all();   // (what the others read stays until they have)
  }
}

template <typename T, int D> int launch(Params& p, cudaStream_t stream) {
  constexpr size_t smem = (size_t)(2 + kRing) * (D / 64) * kBox + 1024;
  CUtensorMap keys{}, values{};
  p.box_shift = 0;
  int shift = 0;
  while (shift < 7 && p.a.page_size % (2 << shift) == 0) ++shift;
  if (shift >= 3 && box_map(&keys, p.a, p.a.k, 1 << shift) && box_map(&values, p.a, p.a.v, 1 << shift)) p.box_shift = shift;
  auto* fn = chunk_kernel<T, D>;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) { cudaGetLastError(); return -2; }
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) { cudaGetLastError(); return -2; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.tiles * p.a.kv_heads * p.share));
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
  if (cudaLaunchKernelEx(&cfg, fn, p, keys, values) == cudaSuccess) return 0;
  cudaGetLastError();
  return -2;
}

}  // namespace

int chunk_attention(const ChunkAttention& a, cudaStream_t stream) {
  Params p{};
  p.a = a;
  p.group = a.heads / a.kv_heads;
  // (a sequence's last tile has one row at least)
  p.tiles = (int)(((int64_t)a.tokens * p.group + (int64_t)std::min(a.batch, a.tokens) * (kRows - 1)) / kRows);
  const int64_t steps = ((int64_t)a.table_width * a.page_size + kStep - 1) / kStep + (a.prefix_length + kStep - 1) / kStep;
  p.share = 1;
  while (p.share < kMaxShare && (int64_t)p.tiles * a.kv_heads * p.share * 2 <= 148 && steps >= 4 * p.share) p.share *= 2;
  p.scale_log2e = a.scale * kLog2e;
  p.spin_limit = kSpinLimit;
  p.test_skip_stage = getenv("ODLA_B200_TEST_SKIP_STAGE") != nullptr;
  if (const char* e = getenv("ODLA_B200_TEST_SPIN_LIMIT")) { const long v = atol(e); if (v >= 64 && v <= (1l << 18)) p.spin_limit = (uint32_t)v; }
  if (a.dt == DT_F16) return a.channels == 64 ? launch<__half, 64>(p, stream) : launch<__half, 128>(p, stream);
  return a.channels == 64 ? launch<__nv_bfloat16, 64>(p, stream) : launch<__nv_bfloat16, 128>(p, stream);
}

}  // namespace b200
