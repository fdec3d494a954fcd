// Attention of the new tokens of each sequence of a batch over a paged cache.
#include <algorithm>
#include <cstddef>
#include <cstdlib>

#include "attention.cuh"
#include "kernels.h"
#include "per_device.h"

namespace b200 {
namespace {

constexpr int kRows = 256, kStep = 128, kSoftmax = 8, kLoaders = 2, kThreads = (kSoftmax + kLoaders + 2) * 32, kMaxShare = 16, kMostRing = 5, kSeen = 8;
template <int D> constexpr int kRing = D == 128 ? 2 : 4;   // units of 128 keys, and as many of values; one more of values where a tile has no second half

constexpr uint32_t kBox = 16384;   // 128 rows of 128 bytes

struct Params {
  ChunkAttention a;
  int group;                       // query heads of a cache head; rows of a sequence = its new tokens * group
  int capacity;                    // positions that a sequence's table has room for
  int tile_rows, tiles, share;     // rows of a tile (half_rows or twice as many); tiles that the batch can have; CTAs (a cluster) that share a tile's positions
  float scale_log2e;
  uint32_t group_factor, group_shift, page_factor, page_shift;   // n / group = n * factor >> shift for n < 2^30, n / page_size likewise
  int box_shift;                   // keys and values arrive in boxes of 1 << box_shift positions by TMA; 0: by 16-byte copies only
  int half_rows;                   // rows of half a tile: those of as many whole tokens as fit into 128, where they leave few of them empty
  int row_boxes;                   // queries and results of half a tile move as boxes
  uint32_t group_bytes, half_bytes;   // in a unit: from eight positions to the next eight, from 64 channels to the next 64
  int fold;                        // boxes bring all 128 channels: 1: pages and heads are counted together, 2: pages and positions are; 0: they bring 64
  uint32_t spin_limit;
  int test_skip_stage;             // test hook, as in kernels_umma.cu: block 0's second unit is neither loaded nor announced
  int test_late;                   // test hook: the warp that hides values comes to each step some steps' time late
};

constexpr int kBarriers = 4 * kMostRing + 15 + kSeen;
struct Shared {
  float2 stat[kRows];       // reference (a base-2 exponent) and sum of each row
  uint64_t k_full[kMostRing], v_full[kMostRing], k_empty[kMostRing], v_empty[kMostRing], q_full, s_full[2], s_read[2], p_most[2], p_full[2], o_done[2], handed, all_done, clean[kSeen], drained[2];
  uint32_t seen[kSeen][4];  // which of a step's positions lie on pages that are there; written at most a ring ahead of the step that is read
  uint32_t tmem;
  int abort, odd;           // odd: values that not all rows see, infinite or no numbers, were taken out of the products
  int scan[kThreads / 32], found, sequence, tile, first_row, count, length;
};

__device__ __forceinline__ int token_of(const Params& p, int row) { return (int)((uint64_t)(uint32_t)row * p.group_factor >> p.group_shift); }
__device__ __forceinline__ int page_of(const Params& p, int n) { return (int)((uint64_t)(uint32_t)n * p.page_factor >> p.page_shift); }
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
// A row without any weight (`none`) is zeros, whatever it sees: a weight of zero did not hide that from its sums.  (In line, this costs the steps their registers:
// 8192 tokens behind 8192 took 5 % longer, with the call 1 %.)
template <typename T, int D> __device__ __noinline__ void add_odd(const Params& p, uint32_t row_at, bool wide, int swizzle, uint32_t second_half, int head, const int* pages, int from, int to, bool none) {
  if (none) {
    for (int c = 0; c < (wide ? D / 4 : D / 8); ++c)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(row_at + (wide ? c * 16 : (c >= 8 ? second_half : 0u) + ((c ^ swizzle) << 4))), "r"(0) : "memory");
    return;
  }
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
          const uint32_t at = row_at + (c >= 32 ? second_half : 0u) + (uint32_t)(((c >> 2) ^ swizzle) << 4) + (uint32_t)((2 * c + h) & 7) * 2;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(at) : "memory");
          const float z = (Mma<T>::kBf16 ? __uint_as_float((uint32_t)y << 16) : __half2float(__ushort_as_half(y))) + x;
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((unsigned short)(Mma<T>::pack(z, 0.f) & 0xffffu)) : "memory");
        }
      }
    }
  }
}

// All 128 channels of a box's positions: eight positions of the first 64 channels, the same of the others, the next eight positions ...
__device__ __forceinline__ void load_box_all(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int eight, int outer) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %3, %4, %5}], [%2];" ::"r"(dst), "l"((uint64_t)map),
               "r"(smem_u32(bar)), "r"(0), "r"(eight), "r"(outer)
               : "memory");
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  asm("max.f32 %0, %0, %1, %2;" : "+f"(x) : "f"(y), "f"(z));
  return x;
}
// Half a tile's rows of 64 channels: whole tokens of the heads of a group.
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int channel, int head, int token) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"((uint64_t)map),
               "r"(smem_u32(bar)), "r"(channel), "r"(head), "r"(token)
               : "memory");
}
__device__ __forceinline__ void store_rows(uint32_t src, const CUtensorMap* map, int channel, int head, int token) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"((uint64_t)map), "r"(src), "r"(channel), "r"(head), "r"(token) : "memory");
}
__device__ __forceinline__ void tie32(uint32_t (&r)[32]) {   // (no read of these registers comes before what stands in front)
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

// Up to 256 rows (token, query head of one cache head's group; two tiles of 128) of one sequence against the positions that they see, 128 at a
// time: first the prefix's, then the sequence's own.  S = Q K^T goes to tensor memory, a thread per row takes it into registers and turns it into
// weights, which go back as the A operand of O += P V, and O stays in tensor memory.  A row's reference is not its running maximum but one that
// follows it only when it has been passed by more than 2^8, so that O is rarely rescaled; in fp16, which has no numbers below 2^-24, it lies 2^7
// lower, so that the many small weights of a long context count together.
// Tensor memory (512 columns, 128 channels): weights of the first tile 64, scores 128, weights of the second 64, O 128 each.  Both tiles use the same
// columns for their scores, one after the other: they are free again as soon as they are in registers, so that the next scores never
// wait for a softmax or for the products with its weights.  (Weights over each tile's own scores, two reads of them, no wait for registers: 3500
// clocks a step of 2 x 128 x 128, 1420 of them a softmax warp's wait for scores that stood behind the last products.)
// Rows are counted token by token, the heads of the group side by side: a tile covers few tokens, and little of its last steps is hidden from it.  Up to half
// a tile's rows leave the second half free: it takes the same rows against every other step (`split`), and hands its sums to the first at the end.
// Where tiles are few, the CTAs of a cluster share the positions of each, by the lengths that they find, and every one joins some of the rows
// out of the others' shared memory.
// A weight of zero does not hide an infinity: in steps that some rows see less of than others, values that are infinite or no numbers are taken
// out of shared memory before the product (and positions behind the last one, whatever lies there), and added to the rows that see them at the end.
// Warps 0-3 and 4-7: softmax of a tile each; 8 and 9: loads; 10: products for scores; 11: products with values, and
// what they must not see.  A row's scores are 128 of the 168
// registers that twelve warps leave a thread.
// 8192 tokens behind 8192, 32 / 8 heads of 128: 1.36 to 1.61 ms by the clock, 1.02 to 1.21 PFLOP/s; a step takes 3300 clocks, its products 2092: what is left is the
// scores' way through one set of columns, 1450 clocks for each tile in turn.  Tiles cost 6 us around their steps: 2048 tokens of an empty cache take 49 to 55 us.
// The running reference is the published online soft-max (M. Milakov and N. Gimelshein, "Online normalizer calculation for softmax", 2018); that it lags behind
// by a threshold is a known refinement of fused attention.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
chunk_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap keys, const __grid_constant__ CUtensorMap values, const __grid_constant__ CUtensorMap queries,
             const __grid_constant__ CUtensorMap results) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared w;
  constexpr int kBoxes = D / 64, kPieces = D / 8;
  constexpr uint32_t kUnit = kBoxes * kBox, kColumns = 512, tmem = 0;   // (all columns: they begin at the first, whatever a look at the allocation's word says, and when)
  const uint32_t smem = (shared_address(smem_raw) + 1023u) & ~1023u, s_q = smem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = p.share == 1 ? blockIdx.x : blockIdx.x / p.share, rank = blockIdx.x - item * p.share, head = item % p.a.kv_heads;
  if (warp == kSoftmax + kLoaders) {
    // (early: it takes a microsecond, which nobody but this warp waits for.  No other block that holds tensor memory fits beside this one, whose threads take all registers.)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&w.tmem)), "r"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 0) {   // a barrier for each lane, and how often it is arrived at
    static_assert(offsetof(Shared, drained) + sizeof(w.drained) - offsetof(Shared, k_full) == 8 * kBarriers, "barriers lie side by side");
    if (lane == 0) { w.abort = 0; w.odd = 0; w.found = 0; }
    for (int i = lane; i < kBarriers; i += 32) {
      uint64_t* bar = &w.k_full[0] + i;
      mbar_init(bar, bar < w.k_empty ? (p.box_shift ? 33 : kLoaders * 33) : bar == &w.q_full ? (p.row_boxes ? 1 : kSoftmax) : bar >= w.v_empty && bar < &w.q_full ? (p.box_shift ? 2 : 1) : (bar >= w.s_read && bar < w.o_done) || bar == &w.handed ? 4 : 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_proxy();
    if (lane == 0 && p.box_shift) { prefetch_map(&keys); prefetch_map(&values); }
    if (lane == 0 && p.row_boxes) { prefetch_map(&queries); prefetch_map(&results); }
  }
  grid_dependency_wait();
  launch_dependents();
  // ---- the sequence that this tile is of: the last ones, which see the most, begin first ----
  {
    const int flat = p.tiles - 1 - item / p.a.kv_heads;
    int before = 0;
    for (int b0 = 0; b0 < p.a.batch; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      int n = 0, lo = 0, hi = 0, length = 0;
      if (b < p.a.batch) {
        lo = max(0, min(p.a.starts[b], p.a.tokens));
        hi = max(lo, min(p.a.starts[b + 1], p.a.tokens));
        length = min(max(p.a.lengths[b], 0), p.capacity);
        n = ((hi - lo) * p.group + p.tile_rows - 1) / p.tile_rows;
      }
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
      }
      if (b0) __syncthreads();   // (the sums of the last turn have been read)
      if (lane == 31) w.scan[warp] = upto;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) {
        if (i < warp) upto += w.scan[i];
        all += w.scan[i];
      }
      if (flat >= before + upto - n && flat < before + upto) {
        w.found = 1; w.sequence = b; w.tile = flat - (before + upto - n);
        w.first_row = lo; w.count = hi - lo; w.length = length;
      }
      before += all;
      if (before > flat) break;
    }
    __syncthreads();
    if (!w.found) {   // (all of a cluster)
      if (warp == kSoftmax + kLoaders) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
      return;
    }
  }
  const int first_row = w.first_row, count = w.count, length = w.length;
  const int row0 = w.tile * p.tile_rows, n_rows = min(p.tile_rows, count * p.group - row0);
  const int* own_pages = p.a.page_table + (int64_t)w.sequence * p.a.table_width;
  // own positions that row r of the sequence sees
  auto limit_of = [&](int r) { return max(0, length - count + token_of(p, r) + 1); };
  const int prefix_steps = (p.a.prefix_length + kStep - 1) / kStep;
  const int least = limit_of(row0), most = limit_of(row0 + n_rows - 1);   // of this tile's first and last row
  const bool split = n_rows <= p.half_rows;
  // Keys and values have rings of their own: whoever waits for one of them follows every turn of its place.
  constexpr int kKeys = kRing<D>;
  const int n_values = kRing<D> + split;
  const uint32_t s_keys = smem + (split ? kUnit : 2 * kUnit), s_values = s_keys + kKeys * kUnit;
  struct Place { int slot; uint32_t turn; };   // in a ring; the parity of the turn
  auto next = [](Place& at, int ring) { if (++at.slot == ring) { at.slot = 0; at.turn ^= 1u; } };
  // steps of the whole tile, this CTA's share of them, and how many of those each half of the rows takes part in
  const int all_steps = prefix_steps + (most + kStep - 1) / kStep;
  const int first = p.share == 1 ? 0 : all_steps * rank / p.share, steps = (p.share == 1 ? all_steps : all_steps * (rank + 1) / p.share) - first;   // (2^23 steps at most)
  const int takes0 = split ? (steps + 1) / 2 : max(0, min(steps, prefix_steps + (limit_of(row0 + p.half_rows - 1) + kStep - 1) / kStep - first)), takes1 = split ? steps / 2 : steps;
  // step i of this CTA: where it begins in its segment, where the segment ends (for the last row), its pages
  auto begin_of = [&](int i) { return (first + i < prefix_steps ? first + i : first + i - prefix_steps) * kStep; };
  auto end_of = [&](int i) { return first + i < prefix_steps ? p.a.prefix_length : most; };
  auto pages_of = [&](int i) { return first + i < prefix_steps ? p.a.prefix_pages : own_pages; };
  volatile int* abort_flag = &w.abort;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, nullptr, 0, p.spin_limit); };
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(~0u, wait(bar, parity)); };   // one answer for the warp
  constexpr uint32_t kWideRow = D * 4 + 16;   // (16 bytes apart from each other's banks)
  const uint32_t wide_base = split ? s_keys : smem;

  // Values that some rows of this tile do not see: of step i, those that are infinite or no numbers, and all behind the last position, go out of the unit where they
  // have landed.
  auto seen_by_all = [&](int i) { return (first + i < prefix_steps ? p.a.prefix_length : least) - begin_of(i); };
  auto hides_any = [&](int i) { return seen_by_all(i) < kStep; };
  auto hide = [&](int i, int slot) {
    const int seen_by_any = end_of(i) - begin_of(i);
    const uint32_t unit = s_values + slot * kUnit;
    auto place = [&](int n) {   // of piece n of 16 bytes, position after position
      const int pos = n / kPieces, c = n % kPieces;
      return unit + (c >> 3) * p.half_bytes + (pos >> 3) * p.group_bytes + (pos & 7) * 128 + (((c & 7) ^ (pos & 7)) << 4);
    };
    const int n0 = max(seen_by_all(i), 0) * kPieces, n1 = min(seen_by_any, kStep) * kPieces;
    // (times zero, an infinity and what is no number stay no numbers: one instruction for two values)
    uint32_t none = 0;
    for (int n = n0 + lane; n < n1; n += 128) {
      uint32_t x[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[k][0]), "=r"(x[k][1]), "=r"(x[k][2]), "=r"(x[k][3]) : "r"(place(n + 32 * k < n1 ? n + 32 * k : n)));
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) none = Mma<T>::times_zero(x[k][e], none);
    }
    if (__any_sync(~0u, none & 0x7fff7fffu)) {
      for (int n = n0 + lane; n < n1; n += 32) {
        uint32_t x[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(place(n)) : "memory");
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (odd16(x[k], Mma<T>::kBf16)) x[k] &= (odd16(x[k] & 0xffffu, Mma<T>::kBf16) ? 0u : 0xffffu) | (odd16(x[k] >> 16, Mma<T>::kBf16) ? 0u : 0xffff0000u);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(n)), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
      }
      *(volatile int*)&w.odd = 1;
    }
    for (int n = n1 + lane; n < kStep * kPieces; n += 32) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(place(n)), "r"(0) : "memory");
    fence_async_proxy();
  };

  if (warp < kSoftmax) {
    // ------------------------------------------------------------------- softmax ----
    const int tile = warp >> 2, quarter = warp & 3, in_tile = quarter * 32 + lane, r = split ? in_tile : tile * p.half_rows + in_tile;
    const int n_live = min(p.half_rows, n_rows - (split ? 0 : tile * p.half_rows));   // rows of this half
    const bool live = in_tile < n_live, any_live = in_tile - lane < n_live;   // this thread's, its warp's first
    if (p.row_boxes) {
      if (threadIdx.x == 0) {   // (rows behind the sequence's last are other sequences', or zeros, and stay without effect)
        mbar_expect_tx(&w.q_full, (split ? 1 : 2) * kBoxes * p.half_rows * 128);
        for (int t = 0; t < (split ? 1 : 2); ++t)
          for (int c = 0; c < kBoxes; ++c) load_rows(s_q + t * kUnit + c * kBox, &queries, &w.q_full, c * 64, head * p.group, first_row + token_of(p, row0 + p.half_rows * t));
      }
    } else {
      // queries: sixteen (or eight) threads for a row.  A negative scale becomes the sign of the queries, the largest score is then the largest product; a scale
      // of zero makes all products zero.
      const uint32_t sign = p.scale_log2e < 0.f ? 0x80008000u : 0u, any = p.scale_log2e == 0.f ? 0u : ~0u;
      const int per = split ? 16 : 32, c = lane % kPieces;
      uint4 u[32 * kPieces / 32];
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int at = i * (32 / kPieces) + lane / kPieces, q_row = warp * per + at, n = (q_row >> 7) * p.half_rows + (q_row & 127), row = row0 + n, j = token_of(p, row);
        u[i] = make_uint4(0, 0, 0, 0);
        if (at < per && (q_row & 127) < p.half_rows && n < n_rows)
          u[i] = *((const uint4*)((const T*)p.a.q + (int64_t)(first_row + j) * p.a.q_token + (int64_t)(head * p.group + row - j * p.group) * p.a.q_head) + c);
      }
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int at = i * (32 / kPieces) + lane / kPieces, q_row = warp * per + at;
        if (at < per)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(s_q + (q_row >> 7) * kUnit + (c >> 3) * kBox + (q_row & 127) * 128 + (((c & 7) ^ (q_row & 7)) << 4)),
                       "r"((u[i].x ^ sign) & any), "r"((u[i].y ^ sign) & any), "r"((u[i].z ^ sign) & any), "r"((u[i].w ^ sign) & any) : "memory");
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&w.q_full);
    }
    const int row = row0 + (live ? r : n_rows - 1), j = token_of(p, row), limit = limit_of(row);
    const float scale = p.scale_log2e == 0.f ? 1.f : fabsf(p.scale_log2e);
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, t_s = lanes + 64, t_p = lanes + tile * 192, t_o = lanes + 256 + tile * D;
    float reference = -INFINITY, sum = 0.f;
    bool ok = true;
    const int own_steps = tile ? takes1 : takes0;
    Place ku{0, 0}, vu{0, 0};
    if (split && tile) next(ku, kKeys);
    const bool frees = (split || tile) && quarter == 0 && lane == 0;
    for (int i = 0; i < own_steps; ++i) {
      const int step = split ? 2 * i + tile : i;
      if (!warp_wait(&w.s_full[tile], i & 1)) { ok = false; break; }
      tc_fence_after();
      if (frees) mbar_arrive(&w.k_empty[ku.slot]);   // (the last scores with these keys)
      next(ku, kKeys);
      if (split) next(ku, kKeys);
      uint32_t v[4][32];
      if (any_live) {
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, v[c]);
        tmem_ld_wait32(v[0]);
#pragma unroll
        for (int c = 1; c < 4; ++c) tie32(v[c]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&w.s_read[tile]);
      if (any_live) {
        // positions of this step that the row sees, if their pages are there
        const int sees = (first + step < prefix_steps ? p.a.prefix_length : limit) - begin_of(step);
        uint32_t seen[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          seen[c] = *(volatile uint32_t*)&w.seen[step % kSeen][c];
          seen[c] &= sees >= 32 * (c + 1) ? ~0u : sees <= 32 * c ? 0u : (1u << (sees - 32 * c)) - 1u;
        }
        if (!__all_sync(~0u, (seen[0] & seen[1] & seen[2] & seen[3]) == ~0u)) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!(seen[c] >> k & 1)) v[c][k] = 0xff800000u;
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; k += 2) m4[k >> 1 & 3] = max3(m4[k >> 1 & 3], __uint_as_float(v[c][k]), __uint_as_float(v[c][k + 1]));
        float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        mx = mx * scale - Mma<T>::kLift;
        const bool passed = mx > (i ? reference + 8.f : -INFINITY);
        // the last products with this tile's weights are done: theirs are the columns that the next weights go to
        if (i) {
          if (!warp_wait(&w.o_done[tile], (i - 1) & 1)) { ok = false; break; }
          if (frees && !split) mbar_arrive(&w.v_empty[vu.slot]);
          next(vu, n_values);
        }
        if (__any_sync(~0u, passed)) {
          const float next = passed ? mx : reference, corr = passed ? exp2_fast(reference - mx) : 1.f;
          reference = next;
          sum *= corr;
          if (i) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(t_o + c * 16, o);
              tmem_ld_wait_regs<16>(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
              tmem_st16(t_o + c * 16, o);
            }
          }
        }
        const float base = reference == -INFINITY ? 0.f : reference;
        const uint64_t scale2 = pair_of(scale, scale), base2 = pair_of(-base, -base);
        uint64_t part[2] = {0, 0};
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t u[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float e[2];
            const uint64_t x = fma2(pair_of(v[c][2 * k], v[c][2 * k + 1]), scale2, base2);
            unpack(x, e);
            e[0] = exp2_fast(e[0]);
            e[1] = exp2_fast(e[1]);
            part[k & 1] = add2(part[k & 1], pair_of(e[0], e[1]));
            u[k] = Mma<T>::pack(e[0], e[1]);
          }
          tmem_st16(t_p + c * 16, u);
          if (c == 2) {   // three quarters of the weights can be multiplied
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&w.p_most[tile]);
          }
        }
        float e[2];
        unpack(add2(part[0], part[1]), e);
        sum += e[0] + e[1];
        tmem_st_wait();
      } else {
        if (i && !warp_wait(&w.o_done[tile], (i - 1) & 1)) { ok = false; break; }
        if (lane == 0) mbar_arrive(&w.p_most[tile]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&w.p_full[tile]);
    }
    // This tile's products are done, its queries' memory is free: the rows of the result go there, and on in whole rows; or, as 32 bits, to the CTAs that
    // join them or the other tile, once all products are done.
    const bool hands = split && tile, takes = split && !tile && takes1, shared = p.share > 1, wide = hands || shared;
    if (ok && own_steps) ok = warp_wait(&w.o_done[tile], (own_steps - 1) & 1);
    else if (ok) ok = warp_wait(&w.q_full, 0);   // (nobody else may have waited for queries without positions: neither boxes nor another warp's rows must land on the zeros)
    if (ok && wide && steps) ok = warp_wait(&w.all_done, 0);   // (the other tile's o_done has phases that this one does not follow)
    tc_fence_after();
    const uint32_t wide_at = wide_base + (uint32_t)r * kWideRow;
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
    const float inverse = wide ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
    // rows of whole channels, 16-byte pieces swizzled; or, for a tile that leaves as boxes, of 64 channels as boxes have them
    const bool boxed = !wide && p.row_boxes && n_live == p.half_rows;
    const uint32_t row_at = wide ? wide_at : s_q + tile * kUnit + (uint32_t)in_tile * (boxed ? 128 : D * 2), second_half = boxed ? kBox - 128 : 0;
    if (ok && any_live && (own_steps || !hands)) {   // (nothing to hand over: the first tile does not wait, and its rows lie there)
      uint32_t v[D / 32][32];
      if (own_steps) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) tmem_ld32(t_o + c * 32, v[c]);
        tmem_ld_wait32(v[0]);
#pragma unroll
        for (int c = 1; c < D / 32; ++c) tie32(v[c]);
      } else {
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k) v[c][k] = 0;
      }
      if (takes) {
#pragma unroll
        for (int k = 0; k < D / 4; ++k) {
          float y[4];
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]) : "r"(wide_at + k * 16));
#pragma unroll
          for (int h = 0; h < 4; ++h) v[k >> 3][(k & 7) * 4 + h] = __float_as_uint(__uint_as_float(v[k >> 3][(k & 7) * 4 + h]) * mine + y[h] * theirs);
        }
      }
      if (wide) {
        // (lanes behind a half's last row have the places of the other half's first ones)
#pragma unroll
        for (int k = 0; k < D / 4; ++k)
          if (live) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_at + k * 16), "r"(v[k >> 3][(k & 7) * 4]), "r"(v[k >> 3][(k & 7) * 4 + 1]), "r"(v[k >> 3][(k & 7) * 4 + 2]),
                       "r"(v[k >> 3][(k & 7) * 4 + 3]) : "memory");
      } else {
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          uint32_t u[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) u[h] = Mma<T>::pack(__uint_as_float(v[k >> 2][(k & 3) * 8 + 2 * h]) * inverse, __uint_as_float(v[k >> 2][(k & 3) * 8 + 2 * h + 1]) * inverse);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_at + (k >> 3) * second_half + ((k ^ (lane & 7)) << 4)), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
        }
      }
    }
    if (hands) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&w.handed);
    } else {
      if (ok && live && (sum == 0.f || *(volatile int*)&w.odd)) {   // positions of this CTA's steps that this row sees and others do not
        const int from = max(least, (max(first, prefix_steps) - prefix_steps) * kStep), to = min(limit, (first + steps - prefix_steps) * kStep);
        add_odd<T, D>(p, row_at, wide, lane & 7, second_half, head, own_pages, from, to, sum == 0.f);
      }
      if (shared) {
        if (live) w.stat[r] = make_float2(ok ? reference : 0.f, ok ? sum : __int_as_float(0x7fc00000));
      } else if (boxed) {
        fence_async_proxy();
        asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + tile) : "memory");   // (the tile's four warps)
        if (*abort_flag) {
          T* y = (T*)p.a.y + (int64_t)(first_row + j) * p.a.y_token + (int64_t)(head * p.group + row - j * p.group) * p.a.y_head;
          if (live)
            for (int c = 0; c < kPieces; ++c) ((uint4*)y)[c] = make_uint4(~0u, ~0u, ~0u, ~0u);   // (no numbers)
        } else if (quarter == 0 && lane == 0) {
          for (int c = 0; c < kBoxes; ++c) store_rows(s_q + tile * kUnit + c * kBox, &results, c * 64, head * p.group, first_row + token_of(p, row0 + p.half_rows * tile));
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
      } else if (any_live) {
        __syncwarp();
        const int64_t y_at = (int64_t)(first_row + j) * p.a.y_token + (int64_t)(head * p.group + row - j * p.group) * p.a.y_head;
        const int c = lane % kPieces;
        uint32_t u[kPieces][4];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int at = i * (32 / kPieces) + lane / kPieces;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u[i][0]), "=r"(u[i][1]), "=r"(u[i][2]), "=r"(u[i][3]) : "r"(row_at + (uint32_t)(at - lane) * (D * 2) + ((c ^ (at & 7)) << 4)));
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int at = i * (32 / kPieces) + lane / kPieces;
          const int64_t to = __shfl_sync(~0u, y_at, at);
          if (!ok) u[i][0] = u[i][1] = u[i][2] = u[i][3] = ~0u;   // (no numbers)
          if (in_tile - lane + at < n_live) *(uint4*)((T*)p.a.y + to + c * 8) = make_uint4(u[i][0], u[i][1], u[i][2], u[i][3]);
        }
      }
    }
    tc_fence_before();
  } else if (warp == kSoftmax + 1 && p.box_shift) {
    // one warp asks for boxes; the other looks at the values of steps that not all rows see.  It follows them all, and a place is filled again only when it has
    // been here, too: two turns further the barrier's parity would be the same.
    Place at{0, 0};
    int hidden = 0;
    for (int i = 0; i < steps; ++i, next(at, n_values)) {
      if (p.test_late) __nanosleep(20000);
      if (!warp_wait(&w.v_full[at.slot], at.turn)) break;
      if (hides_any(i)) {
        hide(i, at.slot);
        __syncwarp();
        if (lane == 0) mbar_arrive(&w.clean[hidden % kSeen]);
        ++hidden;
      }
      if (lane == 0) mbar_arrive(&w.v_empty[at.slot]);
    }
  } else if (warp < kSoftmax + kLoaders) {
    // --------------------------------------------------------------------- loads ----
    const int part = warp - kSoftmax;
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
        box_page = lane < boxes && at < end_of(step) ? pages_of(step)[page_of(p, at)] : -1;
      } else {
#pragma unroll
        for (int h = 0; h < kEach; ++h) page[h] = position(step, h) < end_of(step) ? pages_of(step)[page_of(p, position(step, h))] : -1;
      }
    };
    int box_coord = 0, box_at = 0;
    Place ku{0, 0}, vu{0, 0};
    ask(0);
    for (int u = 0; u < 2 * steps; ++u) {
      const int step = u >> 1;
      const Place at = (u & 1) ? vu : ku;
      uint64_t* full = (u & 1) ? &w.v_full[at.slot] : &w.k_full[at.slot];
      const uint32_t dst = ((u & 1) ? s_values : s_keys) + at.slot * kUnit;
      if (!warp_wait((u & 1) ? &w.v_empty[at.slot] : &w.k_empty[at.slot], at.turn ^ 1u)) break;
      if (u & 1) next(vu, n_values); else next(ku, kKeys);
      const bool skip = p.test_skip_stage && blockIdx.x == 0 && u == 1;
      if (p.box_shift) {
        if (!(u & 1)) {
          const bool there = box_page >= 0 && box_page < p.a.pages;
          box_coord = there ? box_page : p.a.pages;   // (past the last page: zeros)
          {
            const int at = begin_of(step) + (lane << p.box_shift);
            box_at = at - page_of(p, at) * p.a.page_size;
          }
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const uint32_t seen = __ballot_sync(~0u, __shfl_sync(~0u, there, (h * 32 + lane) >> p.box_shift));
            if (lane == 0) *(volatile uint32_t*)&w.seen[step % kSeen][h] = seen;
          }
          ask(step + 1);
        }
        if (skip) continue;
        mbar_arrive(full);
        if (lane == 0) mbar_expect_tx(full, kUnit);
        if (lane < boxes) {
          const CUtensorMap* map = (u & 1) ? &values : &keys;
          const uint32_t to = dst + ((uint32_t)lane << p.box_shift >> 3) * p.group_bytes;
          if (p.fold == 1) load_box_all(to, map, full, box_at >> 3, box_coord == p.a.pages ? p.a.pages * p.a.kv_heads : box_coord * p.a.kv_heads + head);
          else if (p.fold == 2) load_box_all(to, map, full, box_coord * (p.a.page_size >> 3) + (box_at >> 3), head);
          else {
#pragma unroll
            for (int c = 0; c < kBoxes; ++c) load_box(to + c * p.half_bytes, map, full, c * 64, box_at, head, box_coord);
          }
        }
        continue;
      }
      if (!(u & 1)) {
#pragma unroll
        for (int h = 0; h < kEach; ++h) {
          off[h] = page[h] >= 0 && page[h] < p.a.pages ? page[h] * p.a.c_page + (int64_t)(position(step, h) - page_of(p, position(step, h)) * p.a.page_size) * p.a.c_token : -1;
          const uint32_t seen = __ballot_sync(~0u, off[h] >= 0);
          if (lane == 0) *(volatile uint32_t*)&w.seen[step % kSeen][part * kEach + h] = seen;
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
    if (*abort_flag && lane == 0) {   // boxes in flight land before their memory goes
      await_stages(w.k_full, kKeys, ku.slot, ku.turn ^ 1u);
      await_stages(w.v_full, n_values, vu.slot, vu.turn ^ 1u);
    }
  } else {
    // ------------------------------------------------------------------ products ----
    // One thread issues those for scores, one of another warp those with values: what each does between its products would otherwise keep the tensor cores
    // waiting (one thread for both: 2750 clocks a step with a softmax that computes nothing).
    const uint32_t fmt = Mma<T>::kBf16 ? 1u : 0u, common = (1u << 4) | (fmt << 7) | (fmt << 10) | (8u << 24);
    // the distance between groups of eight rows; the distance between 64 channels and the next 64 is only read for values, which lie with channels innermost
    auto desc = [&](uint32_t at, uint32_t lead, uint32_t group) {
      return (uint64_t)((group >> 4) | (1u << 14) | (2u << 29)) << 32 | (uint64_t)(lead >> 4) << 16 | (uint64_t)((at & 0x3FFFF) >> 4);
    };
    // (16-byte copies of other threads, which the barrier has told of: the fence makes them visible to the products; boxes are)
    auto landed = [&](uint64_t* full, const Place& at) {
      const bool there = wait(&full[at.slot], at.turn);
      if (!p.box_shift) fence_async_proxy();
      return there;
    };
    // Split, a tile has every other step.
    if (warp == kSoftmax + kLoaders) {
      if (elect_one()) {
        const uint32_t idesc = common | ((uint32_t)(kStep >> 3) << 17), half = p.half_bytes >> 4;   // (64 channels further)
        const uint64_t q_desc = desc(s_q, 16, 1024), k_desc = desc(s_keys, 16, p.group_bytes);
        int last = -1, last_turn = 0;   // the tile whose scores came last: these wait until they are in registers
        Place at{0, 0};
        bool ok = steps == 0 || wait(&w.q_full, 0);
        for (int i = 0; i < steps && ok; ++i, next(at, kKeys)) {
          ok = landed(w.k_full, at);
          const uint64_t k = k_desc + (uint32_t)at.slot * (kUnit >> 4);
          for (int t = split ? i & 1 : i < takes0 ? 0 : 1; t < 2 && ok; t += split ? 2 : 1) {
            if (last >= 0) ok = wait(&w.s_read[last], last_turn & 1);
            if (!ok) break;
            tc_fence_after();
            const uint64_t q = q_desc + (split ? 0u : t * (kUnit >> 4));
#pragma unroll
            for (int n = 0; n < D / 16; ++n)   // S = Q_t K^T
              umma_f16(tmem + 64, q + (n >> 2) * (kBox >> 4) + (n & 3) * 2, k + (n >> 2) * half + (n & 3) * 2, idesc, n ? 1u : 0u);
            umma_commit(&w.s_full[t]);   // (softmax warps tell the loaders, where they know, that keys and values have been used)
            last = t;
            last_turn = split ? i >> 1 : i;
          }
        }
        if (!ok) {   // products and queries in flight end before their memory goes
          umma_commit(&w.drained[0]);
          await_landing(&w.drained[0], 0);
          if (p.row_boxes) await_landing(&w.q_full, 0);
        }
      }
    } else {
      const uint32_t idesc = common | (1u << 16) | ((uint32_t)(D >> 3) << 17), sixteen = p.group_bytes >> 3;   // (16 positions further, in units of 16 bytes)
      const uint64_t v_desc = desc(s_values, p.half_bytes, p.group_bytes);
      const bool issues = elect_one();
      int hidden = 0;   // steps that hid values
      Place at{0, 0};
      bool ok = true;
      // (all lanes go through all steps, and leave together: the one that issues skips what is left when a wait has run out)
      for (int i = 0; i < steps; ++i, next(at, n_values)) {
        const bool hides = hides_any(i);
        if (hides && !p.box_shift) {
          __syncwarp();
          if (!warp_wait(&w.v_full[at.slot], at.turn)) { ok = false; break; }
          hide(i, at.slot);
          __syncwarp();
        }
        if (issues && ok) {
          ok = hides && p.box_shift ? wait(&w.clean[hidden % kSeen], hidden / kSeen & 1) : landed(w.v_full, at);
          hidden += hides;
          const uint64_t v = v_desc + (uint32_t)at.slot * (kUnit >> 4);
          const int turn = split ? i >> 1 : i;
          for (int t = split ? i & 1 : i < takes0 ? 0 : 1; t < 2 && ok; t += split ? 2 : 1) {
#pragma unroll
            for (int n = 0; n < 8; ++n) {   // O_t += P_t V
              if (n == 0 || n == 6) {   // (most of them while the last quarter of the weights is worked out)
                ok = ok && wait(n ? &w.p_full[t] : &w.p_most[t], turn & 1);
                if (!ok) break;
                tc_fence_after();
              }
              umma_tmem_a(tmem + 256 + t * D, tmem + t * 192 + n * 8, v + n * sixteen, idesc, (turn || n) ? 1u : 0u);
            }
            if (!ok) break;
            umma_commit(&w.o_done[t]);
            if (split && i + n_values < steps) umma_commit(&w.v_empty[at.slot]);
          }
        }
      }
      if (issues) {
        uint64_t* last = ok ? &w.all_done : &w.drained[1];
        umma_commit(last);
        await_landing(last, 0);   // (no arrival is under way when the block ends)
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftmax + kLoaders) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
  if (p.share > 1) {
    // ---- each CTA joins the rows that are its own modulo the cluster's size ----
    cluster_sync_all();
    if (warp < kSoftmax) {
      constexpr int N = D / 32;
      const uint32_t stat = smem_u32(w.stat);
      for (int r = rank + p.share * warp; r < n_rows; r += p.share * kSoftmax) {
        float2 st = make_float2(-INFINITY, 0.f);
        if (lane < p.share) st = load_remote2(map_to_cta(stat + r * 8, lane));
        float top = st.x, sum = 0.f, acc[N];
#pragma unroll
        for (int o = kMaxShare / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        top = __shfl_sync(~0u, top, 0);
        const float f = st.y != 0.f ? exp2_fast(st.x - (top == -INFINITY ? 0.f : top)) : 0.f;   // (a share without positions wrote no row)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = 0.f;
#pragma unroll 4
        for (int i = 0; i < p.share; ++i) {
          const float fi = __shfl_sync(~0u, f, i), si = __shfl_sync(~0u, st.y, i);
          if (si == 0.f) continue;
          float x[N];
          load_remote<N>(map_to_cta(wide_base + (uint32_t)r * kWideRow + lane * (N * 4), i), x);
          sum += fi * si;
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += fi * x[k];
        }
        const int row = row0 + r, j = token_of(p, row);
        T* y = (T*)p.a.y + (int64_t)(first_row + j) * p.a.y_token + (int64_t)(head * p.group + row - j * p.group) * p.a.y_head + lane * N;
        const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int k = 0; k < N; k += 2) *(uint32_t*)(y + k) = Mma<T>::pack(acc[k] * inverse, acc[k + 1] * inverse);
      }
    }
    cluster_sync_all();   // (what the others read stays until they have)
  }
}
// Boxes of all 128 channels of 8 << shift positions of one head and page.  A tensor map has five dimensions: 64 channels, eight positions, the two halves of
// the channels, eights of positions, and one for both heads and pages, which dense caches allow: pages of heads are counted through, or, where the heads of a position
// lie together, pages of positions.
int whole_box_map(CUtensorMap* m, const ChunkAttention& a, const void* base, int shift) {
  if (!load_driver_entry_points()) return 0;
  const int fold = a.c_page == a.kv_heads * a.c_head || a.pages == 1 || a.kv_heads == 1 ? 1 : a.c_page == a.page_size * a.c_token ? 2 : 0;
  if (!fold || a.c_token == 0 || (int64_t)a.pages * std::max(a.kv_heads, a.page_size) >= (1ll << 31) || (a.kv_heads > 1 && a.c_head == 0)) return 0;
  const int64_t eights = a.page_size / 8, outer = fold == 1 ? (a.kv_heads > 1 ? a.c_head : a.pages > 1 ? a.c_page : a.channels) : a.kv_heads > 1 ? a.c_head : a.channels;
  const cuuint64_t dims[5] = {64, 8, 2, (cuuint64_t)(fold == 1 ? eights : eights * a.pages), (cuuint64_t)(fold == 1 ? (int64_t)a.pages * a.kv_heads : a.kv_heads)};
  const cuuint64_t strides[4] = {(cuuint64_t)a.c_token * 2, 128, (cuuint64_t)a.c_token * 16, (cuuint64_t)outer * 2};
  for (cuuint64_t s : strides) if (s == 0 || s >= (1ull << 40)) return 0;
  const cuuint32_t box[5] = {64, 8, 2, 1u << shift, 1}, step[5] = {1, 1, 1, 1, 1};
  return g_encode_tiled(m, a.dt == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, (void*)base, dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? fold : 0;
}

// Boxes of 64 channels of half a tile's rows: a group's heads of whole tokens.
bool row_map(CUtensorMap* m, const Params& p, const void* base, int64_t token, int64_t head) {
  if (!load_driver_entry_points()) return false;
  auto bytes = [](int64_t stride, int extent) { return extent == 1 && stride == 0 ? (cuuint64_t)16 : (cuuint64_t)stride * 2; };
  const cuuint64_t dims[3] = {(cuuint64_t)p.a.channels, (cuuint64_t)p.a.heads, (cuuint64_t)p.a.tokens};
  const cuuint64_t strides[2] = {bytes(head, p.a.heads), bytes(token, p.a.tokens)};
  for (cuuint64_t s : strides) if (s == 0 || s >= (1ull << 40)) return false;
  const cuuint32_t box[3] = {64, (cuuint32_t)p.group, (cuuint32_t)(p.half_rows / p.group)}, step[3] = {1, 1, 1};
  return g_encode_tiled(m, p.a.dt == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void*)base, dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Fit {
  int clusters[kMaxShare + 1];   // of each size, that run at the same time
};

template <typename T, int D> int launch(Params& p, cudaStream_t stream) {
  constexpr size_t smem = (size_t)(2 + 2 * kRing<D>) * (D / 64) * kBox + 1024;
  auto* fn = chunk_kernel<T, D>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  static std::atomic<uint64_t> told{0};
  if (!once_per_device(told, [&] {
        return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess &&
               cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
      }))
    return -2;
  // How many clusters of each size fit: GPUs of one kind have the same number of SMs, but not in the same groups.
  static PerDevice<Fit> fits;
  const Fit fit = fits([&] {
    Fit f{};
    cfg.numAttrs = 1;
    for (int i = 1; i <= kMaxShare; ++i) {
      cfg.gridDim = dim3((unsigned)(i * 148));
      attr[0].val.clusterDim.x = (unsigned)i;
      if (cudaOccupancyMaxActiveClusters(&f.clusters[i], fn, &cfg) != cudaSuccess) { cudaGetLastError(); f.clusters[i] = 0; }
    }
    f.clusters[1] = std::max(f.clusters[1], 1);
    return f;
  });
  // Rows of a tile and CTAs that share it: the shortest estimate of waves of steps (1.9 us, 1.2 for half a tile's rows) and of what a CTA does before and after them
  // (6 us, 2 more to join).  Lengths are not known here: the table's width stands for them.
  const int64_t steps = ((int64_t)p.a.table_width * p.a.page_size + kStep - 1) / kStep + (p.a.prefix_length + kStep - 1) / kStep;
  double best = 1e30;
  for (int rows = 2 * p.half_rows; rows >= p.half_rows; rows -= p.half_rows) {
    // (a sequence's last tile has one row at least)
    const int64_t tiles = ((int64_t)p.a.tokens * p.group + (int64_t)std::min(p.a.batch, p.a.tokens) * (rows - 1)) / rows, clusters = tiles * p.a.kv_heads;
    for (int share = 1; share <= kMaxShare; ++share) {
      if (fit.clusters[share] < 1 || (share > 1 && steps < 2 * share)) continue;
      const int64_t waves = (clusters + fit.clusters[share] - 1) / fit.clusters[share];
      const double us = (double)waves * ((double)((steps + share - 1) / share) * (rows > p.half_rows ? 1.9 : 1.2) + (share > 1 ? 8.0 : 6.0));
      if (us < best) { best = us; p.tile_rows = rows; p.tiles = (int)tiles; p.share = share; }
    }
  }
  CUtensorMap keys{}, values{}, queries{}, results{};
  p.box_shift = 0;
  p.group_bytes = 1024;
  p.half_bytes = kBox;
  int shift = 0;
  while (shift < 7 && p.a.page_size % (2 << shift) == 0) ++shift;
  // (an SM's boxes begin some 85 clocks after one another: 64 of eight positions and 64 channels held a step at 5460 clocks)
  if (D == 128 && shift >= 3 && (p.fold = whole_box_map(&keys, p.a, p.a.k, shift - 3)) != 0 && whole_box_map(&values, p.a, p.a.v, shift - 3)) {
    p.box_shift = shift;
    p.group_bytes = 2048;
    p.half_bytes = 1024;
  } else if (shift >= 3 && box_map(&keys, p.a, p.a.k, 1 << shift) && box_map(&values, p.a, p.a.v, 1 << shift)) {
    p.box_shift = shift;
    p.fold = 0;
  }
  p.row_boxes = p.scale_log2e > 0.f && p.half_rows % p.group == 0 && row_map(&queries, p, p.a.q, p.a.q_token, p.a.q_head) && row_map(&results, p, p.a.y, p.a.y_token, p.a.y_head);
  cfg.gridDim = dim3((unsigned)(p.tiles * p.a.kv_heads * p.share));
  attr[0].val.clusterDim.x = (unsigned)p.share;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, fn, p, keys, values, queries, results) == cudaSuccess) return 0;
  cudaGetLastError();
  return -2;
}

// n / of = n * factor >> shift for n < 2^30: factor * of exceeds 2^shift by at most of <= 2^(shift - 30).
void quotient(int of, uint32_t& factor, uint32_t& shift) {
  shift = 0;
  while ((1ll << shift) < of) ++shift;
  shift += 30;
  factor = (uint32_t)((1ull << shift) / of + 1);
}

}  // namespace

int chunk_attention(const ChunkAttention& a, cudaStream_t stream) {
  Params p{};
  p.a = a;
  p.group = a.heads / a.kv_heads;
  p.half_rows = p.group <= 128 && 128 / p.group * p.group >= 112 ? 128 / p.group * p.group : 128;
  p.capacity = a.table_width * a.page_size;   // (below 2^30)
  quotient(p.group, p.group_factor, p.group_shift);
  quotient(a.page_size, p.page_factor, p.page_shift);
  p.scale_log2e = a.scale * kLog2e;
  p.spin_limit = kSpinLimit;
  p.test_skip_stage = getenv("ODLA_B200_TEST_SKIP_STAGE") != nullptr;
  p.test_late = getenv("ODLA_B200_TEST_LATE_WARP") != nullptr;
  if (const char* e = getenv("ODLA_B200_TEST_SPIN_LIMIT")) { const long v = atol(e); if (v >= 64 && v <= (1l << 18)) p.spin_limit = (uint32_t)v; }
  if (a.dt == DT_F16) return a.channels == 64 ? launch<__half, 64>(p, stream) : launch<__half, 128>(p, stream);
  return a.channels == 64 ? launch<__nv_bfloat16, 64>(p, stream) : launch<__nv_bfloat16, 128>(p, stream);
}

}  // namespace b200
