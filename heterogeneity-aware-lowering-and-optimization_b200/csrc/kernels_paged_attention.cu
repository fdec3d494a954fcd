// Attention over a paged cache whose sequences share their first positions.
#include <algorithm>
#include <climits>
#include <cstdlib>

#include "attention.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kRows = 16, kStep = 32;   // rows of a tile; positions a warp takes at a time
constexpr int kRing = 3;                                                    // units of kStep rows of keys or of values, for each warp

struct Params {
  PagedAttention a;
  const void *k, *v, *q;
  const int *prefix_pages, *page_table, *lengths;
  void* y;
  float* part;                       // [rows][slots][channels], then float2 [rows][slots]: maximum (of base-2 exponents) and sum
  float2* stat;
  int group, rows;                   // query heads of a cache head; rows of one cache head = batch * queries * group
  int prefix_chunk, prefix_chunks, own_chunk, own_chunks, slots;
  int team;                          // 1, 2 or 4 tiles of 16 rows that a block of tile_kernel takes
  int prefix_tiles, own_tiles;       // its blocks of rows: over all rows, and over those of one sequence
  // The tensor-core kernel's tiles of 256 rows: over all rows, for the prefix, and over those of one sequence, for the own positions that all
  // its queries see (the last queries - 1 positions remain for tile_kernel, in the last slot).  0: tile_kernel takes them all.
  int wide_tiles, own_wide_tiles, own_wide_chunks, own_wide_chunk;
  float scale_log2e;
  uint32_t page_factor, page_shift;  // n / page_size = n * page_factor >> page_shift for n < 2^30
  int join_warps;                    // 4 or 1: warps that share a row's slots
  int wide_first;                    // no tile_kernel in front
  int box_shift;                     // keys and values arrive in boxes of 1 << box_shift positions by TMA; 0: by 16-byte copies only
  uint32_t spin_limit;
  int test_skip_stage;               // test hook, as in kernels_umma.cu: block 0's second unit is neither loaded nor announced
};

template <bool TRANS> __device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ int capped(const Params& p, int n) {
  const long long cap = (long long)p.a.table_width * p.a.page_size;
  return n < 0 ? 0 : n > cap ? (int)cap : n;
}
__device__ __forceinline__ int own_length(const Params& p, int b) { return capped(p, p.lengths[b]); }

__device__ __forceinline__ int page_of(const Params& p, int n) { return (int)((uint64_t)(uint32_t)n * p.page_factor >> p.page_shift); }

// Own positions that every query of the sequence sees.
__device__ __forceinline__ int common_length(const Params& p, int length) { return max(0, length - p.a.queries + 1); }

// Up to TEAM tiles of 16 rows (query, query head) of one cache head against one chunk of positions, of the prefix or of one sequence.
// The cache's bytes are the least it has to do: 16 rows do 16 products for each two bytes read, far below what the tensor cores could do.  What
// bounds it is a warp's chain of latencies, about 2000 clocks for a step of 32 positions of 128 channels (loads asked for 500, Q K^T 400, softmax 450,
// P V 420), with the two warps per scheduler that 250 registers allow: 128 sequences of up to 900 positions, 236 MB, take 50 us, 4.7 TB/s.
// With one tile each warp has positions and a ring of its own: no warp waits for another until
// the end.  The ring's units alternate keys and values of 32 positions; two of the three are always in flight.  With more tiles the warps that take
// them over the same positions are a team, which shares its warps' rings, loads and a barrier for each unit, so that a sequence's
// cache is read once (64 rows of 8 sequences of up to 2500 positions: 35.6 us, a tile for each block 43.9; 24 of 32 of up to 1500: 26.8 and 30).
// Copies of 16 bytes by all lanes, not one bulk copy for each position: of those an SM starts one in some 25 clocks (73 us).
// Softmax runs over positions with maximum and sum per row; the weights are rounded to the cache's type for the second product, and the
// sum is taken of the rounded ones, so that the result is an average of values with weights that add up to one.
template <typename T, int D, int TEAM>
__global__ void __launch_bounds__(kThreads, 2) tile_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kPieces = D / 8, kUnit = kStep * D * 2;   // 16-byte pieces of a row; bytes of a unit
  constexpr int kTeams = kWarps / TEAM, kSlots = kRing * TEAM;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, team = warp / TEAM, member = warp % TEAM, head = blockIdx.y;
  // The kernel in front may still be writing the cache; the wide kernel may start once every block here knows that it is not.
  grid_dependency_wait();
  launch_dependents();
  // what this block works on
  int item = blockIdx.x;
  const int prefix_items = p.prefix_tiles * p.prefix_chunks;
  const bool own = item >= prefix_items;
  const int* pages;
  int row0, n_rows, begin, end, slot, length = 0, b_own = 0;
  if (!own) {
    const int chunk = item / p.prefix_tiles, tile = item - chunk * p.prefix_tiles;
    row0 = tile * (kRows * TEAM);
    n_rows = min(kRows * TEAM, p.rows - row0);
    begin = chunk * p.prefix_chunk;
    end = min(begin + p.prefix_chunk, p.a.prefix_length);
    pages = p.prefix_pages;
    slot = chunk;
  } else {
    item -= prefix_items;
    b_own = item % p.a.batch;
    const int rest = item / p.a.batch, chunk = rest / p.own_tiles, tile = rest - chunk * p.own_tiles;
    const int per = p.a.queries * p.group;
    row0 = b_own * per + tile * (kRows * TEAM);
    n_rows = min(kRows * TEAM, per - tile * (kRows * TEAM));
    begin = chunk * p.own_chunk;
    if (p.own_wide_tiles) begin += common_length(p, own_length(p, b_own));
    end = (int)min((int64_t)begin + p.own_chunk, (int64_t)p.a.table_width * p.a.page_size);   // (until the length is there)
    pages = p.page_table + (int64_t)b_own * p.a.table_width;
    slot = p.prefix_chunks + p.own_wide_chunks + chunk;
  }
  // The length, the first page numbers and the queries are asked for at once; page numbers after that a step early.
  if (own) length = p.lengths[b_own];
  auto ask = [&](int step) {
    const int pos = begin + step * kStep + lane;
    return lane < kStep && pos < end ? pages[page_of(p, pos)] : -1;
  };
  int page = ask(team);
  // this warp's rows, and those of them that this lane has a share of: row + lane / 4 and + 8
  const int row_w = row0 + member * kRows, rows_w = min(kRows, n_rows - member * kRows);   // (none or less: it loads with the others, no more)
  int limit[2];
  uint32_t qa[D / 16][4];
  // (the scale's sign becomes that of the queries: the largest score is then the largest product; without a scale all products are zero)
  const uint32_t sign = p.scale_log2e < 0.f ? 0x80008000u : 0u, any = p.scale_log2e == 0.f ? 0u : ~0u;
  const float scale = p.scale_log2e == 0.f ? 1.f : fabsf(p.scale_log2e);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = (lane >> 2) + 8 * h;
    const bool live = r < rows_w;
    const int row = live ? row_w + r : row0, g = row % p.group, j = row / p.group % p.a.queries, b = row / (p.group * p.a.queries);
    limit[h] = !live ? INT_MIN : j;
    const T* q = (const T*)p.q + b * p.a.q_batch + j * p.a.q_token + (int64_t)(head * p.group + g) * p.a.q_head;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qa[k][h] = live ? (*(const uint32_t*)(q + k * 16 + (lane & 3) * 2) ^ sign) & any : 0u;
      qa[k][h + 2] = live ? (*(const uint32_t*)(q + k * 16 + 8 + (lane & 3) * 2) ^ sign) & any : 0u;
    }
  }
  if (own) {
    length = capped(p, length);
    end = min(end, length);
    if (begin >= end) return;   // (the sum over slots knows)
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) limit[h] = limit[h] == INT_MIN ? 0 : own ? length - p.a.queries + limit[h] + 1 : p.a.prefix_length;
  // positions below `all` are seen by every row of the tile
  const int all = own ? length - p.a.queries + row_w / p.group % p.a.queries + 1 : p.a.prefix_length;
  const int n_steps = (end - begin + kStep - 1) / kStep;
  const uint32_t ring = shared_address(smem) + team * (kSlots * kUnit);

  const T *kc = (const T*)p.k + (int64_t)head * p.a.c_head, *vc = (const T*)p.v + (int64_t)head * p.a.c_head;
  int64_t off = -1;
  // unit u: keys (u even) or values (u odd) of this team's step u / 2, of which each of its warps brings a part; returns which of the 32 positions can
  // be seen at all
  auto issue = [&](int u) -> uint32_t {
    uint32_t seen = 0;
    const int step = team + (u >> 1) * kTeams;
    if (step < n_steps) {
      if (!(u & 1)) {
        const int pos = begin + step * kStep + lane;
        off = -1;
        if (lane < kStep && pos < end && page >= 0 && page < p.a.pages) off = page * p.a.c_page + (int64_t)(pos - page_of(p, pos) * p.a.page_size) * p.a.c_token;
        seen = __ballot_sync(~0u, off >= 0);
        page = ask(step + kTeams);
      }
      const T* base = (u & 1) ? vc : kc;
      const uint32_t dst = ring + (u % kSlots) * kUnit;
#pragma unroll
      for (int i = 0; i < kPieces * kStep / 32 / TEAM; ++i) {
        const int n = (member * (kPieces * kStep / 32 / TEAM) + i) * 32 + lane, r = n / kPieces, c = n % kPieces;
        const int64_t o = __shfl_sync(~0u, off, r);
        copy16(dst + r * (D * 2) + ((c ^ (r & 7)) << 4), base + (o < 0 ? 0 : o) + c * 8, o >= 0);
      }
    }
    copies_commit();
    return seen;
  };

  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
  // Masks of the steps whose keys are on their way, the next one first.  A warp of its own refills a unit as soon as it has read it; a team
  // behind the barrier that tells that the next one is there, which is also where all have read it.
  constexpr int kAhead = TEAM == 1 ? 2 : kSlots / 2;
  uint32_t ahead[kAhead];
#pragma unroll
  for (int u = 0; u < (TEAM == 1 ? kSlots : kSlots - 1); ++u) {
    const uint32_t seen = issue(u);
    if (!(u & 1)) ahead[u / 2] = seen;
  }
  auto await = [&]() {
    copies_wait<TEAM == 1 ? 2 : kSlots - 2>();
    if (TEAM == 1) __syncwarp(); else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * TEAM) : "memory");
  };
  auto push = [&](uint32_t seen) {
#pragma unroll
    for (int k = 0; k + 1 < kAhead; ++k) ahead[k] = ahead[k + 1];
    ahead[kAhead - 1] = seen;
  };
  for (int i = 0, step = team; step < n_steps; ++i, step += kTeams) {
    const int at = begin + step * kStep;
    const uint32_t seen = ahead[0];
    await();
    if (TEAM > 1) issue(2 * i + kSlots - 1);
    const uint32_t ku = ring + (2 * i % kSlots) * kUnit, vu = ring + ((2 * i + 1) % kSlots) * kUnit;
    uint32_t pa[kStep / 16][4];
    if (TEAM == 1 || rows_w > 0) {
    float s[kStep / 8][4];
#pragma unroll
    for (int n = 0; n < kStep / 8; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[n][k] = 0.f;
    // (four sums side by side: each of a sum's products waits for the one before it)
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      uint32_t b[kStep / 8][4];
#pragma unroll
      for (int n = 0; n < kStep / 8; ++n) {   // 8 positions x 32 channels
        const int r = n * 8 + (lane & 7), c = k * 4 + (lane >> 3);
        ldmatrix4<false>(b[n], ku + r * (D * 2) + ((c ^ (r & 7)) << 4));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < kStep / 8; ++n) Mma<T>::run(s[n], qa[2 * k + h], b[n][2 * h], b[n][2 * h + 1]);
    }
    if (TEAM == 1) {
      __syncwarp();
      issue(2 * i + 3);
    }
    // a position that is not seen has no score
    if (seen != ~0u >> (32 - kStep) || at + kStep > all) {
#pragma unroll
      for (int n = 0; n < kStep / 8; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int pos = n * 8 + (lane & 3) * 2 + (k & 1);
          if (!(seen >> pos & 1) || at + pos >= limit[k >> 1]) s[n][k] = -INFINITY;
        }
    }
    float base[2], mx[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = m[h];
#pragma unroll
      for (int n = 0; n < kStep / 8; ++n) mx[h] = fmaxf(mx[h], fmaxf(s[n][2 * h], s[n][2 * h + 1]));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(~0u, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(~0u, mx[h], 2));
      base[h] = mx[h] == -INFINITY ? 0.f : mx[h] * scale;
    }
    if (__any_sync(~0u, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float corr = exp2_fast(m[h] * scale - base[h]);   // 0 at first
        m[h] = mx[h];
        l[h] *= corr;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) { o[n][2 * h] *= corr; o[n][2 * h + 1] *= corr; }
      }
    }
#pragma unroll
    for (int n = 0; n < kStep / 8; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        pa[n >> 1][(n & 1) * 2 + h] = Mma<T>::pack(exp2_fast(s[n][2 * h] * scale - base[h]), exp2_fast(s[n][2 * h + 1] * scale - base[h]), l[h]);
    }
    await();
    if (TEAM > 1) push(issue(2 * i + kSlots));
    if (TEAM > 1 && rows_w <= 0) continue;
    if (at + kStep <= all || !own) {
#pragma unroll
      for (int k = 0; k < kStep / 16; ++k)
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {   // 16 positions x 16 channels
          uint32_t b[4];
          const int r = k * 16 + (lane & 15), c = n * 2 + (lane >> 4);
          ldmatrix4<true>(b, vu + r * (D * 2) + ((c ^ (r & 7)) << 4));
          Mma<T>::run(o[2 * n], pa[k], b[0], b[1]);
          Mma<T>::run(o[2 * n + 1], pa[k], b[2], b[3]);
        }
    } else {
      // Positions that later queries of the tile see and earlier ones do not: a weight of zero does not hide an infinity there, so each
      // query has its product with the values that it sees, and the other rows take nothing of it.
      const int q0 = row_w / p.group, q1 = (row_w + rows_w - 1) / p.group;
      for (int qi = q0; qi <= q1; ++qi) {
        const int lim = length - p.a.queries + qi % p.a.queries + 1 - at;
        const bool mine[2] = {(row_w + (lane >> 2)) / p.group == qi, (row_w + (lane >> 2) + 8) / p.group == qi};
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k) {
          const int pos = k * 16 + (lane & 3) * 2;
          const uint32_t keep0 = (pos < lim ? 0xffffu : 0u) | (pos + 1 < lim ? 0xffff0000u : 0u), keep1 = (pos + 8 < lim ? 0xffffu : 0u) | (pos + 9 < lim ? 0xffff0000u : 0u);
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            uint32_t b[4];
            const int r = k * 16 + (lane & 15), c = n * 2 + (lane >> 4);
            ldmatrix4<true>(b, vu + r * (D * 2) + ((c ^ (r & 7)) << 4));
            float t[2][4] = {};
            Mma<T>::run(t[0], pa[k], b[0] & keep0, b[1] & keep1);
            Mma<T>::run(t[1], pa[k], b[2] & keep0, b[3] & keep1);
#pragma unroll
            for (int x = 0; x < 8; ++x)
              if (mine[(x & 3) >> 1]) o[2 * n + (x >> 2)][x & 3] += t[x >> 2][x & 3];
          }
        }
      }
    }
    if (TEAM == 1) {
      __syncwarp();
      push(issue(2 * i + 4));
    }
  }
  copies_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(~0u, l[h], 1);
    l[h] += __shfl_xor_sync(~0u, l[h], 2);
  }
  // ---- the teams' results become one ----
  __syncthreads();
  float* so = (float*)smem;                                 // [warp][16 rows][D + 4]: the padding spreads rows over the banks
  float2* sm = (float2*)(so + kWarps * kRows * (D + 4));    // [warp][16]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = (lane >> 2) + 8 * h;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) *(float2*)&so[(warp * kRows + r) * (D + 4) + n * 8 + (lane & 3) * 2] = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    if ((lane & 3) == 0) sm[warp * kRows + r] = make_float2(m[h] * scale, l[h]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_rows * (D / 4); i += kThreads) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;   // (rows lie [team][member][16])
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kTeams; ++w) top = fmaxf(top, sm[w * (TEAM * kRows) + r].x);
    const float base = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < kTeams; ++w) {
      const float2 st = sm[w * (TEAM * kRows) + r];
      const float f = exp2_fast(st.x - base);
      const float4 x = *(const float4*)&so[(w * (TEAM * kRows) + r) * (D + 4) + c];
      sum += f * st.y;
      acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
    }
    const int row = row0 + r;
    const int64_t at = ((int64_t)head * p.rows + row) * p.slots + slot;
    *(float4*)(p.part + at * D + c) = acc;
    if (c == 0) p.stat[at] = make_float2(top, sum);
  }
}

// ---------------------------------------------------------- the prefix on the tensor cores ----
// Up to 256 rows (query, query head) of one cache head against one chunk of the prefix, 128 positions at a time: two tiles of
// 128 rows, so that the products of one tile run under the softmax of the other.  S = Q K^T goes to tensor memory; a thread per
// row turns it into weights, which replace it there as the A operand of O += P V.  O stays in tensor memory over the whole chunk: a
// row's reference is not its running maximum but one that follows it only when it has been passed by more than 2^8, so that O is rarely
// rescaled; weights up to 2^8 have the same relative rounding, and the sums are fp32.  fp16 has no numbers below 2^-24, and
// the thousands of positions of the largest one's chunk count together although each weighs less: there the reference lies 2^7 below, and the largest
// weights are 2^7 to 2^15.  At 256 rows a step of 128 positions
// is 4 products of 128 x 128 x D (about 2000 clocks for D = 128) and 32768 exponentials (2048 clocks); it takes 3100 to 3200: a softmax warp
// works for 2000 and waits 1100 for the next scores, which stand behind the last products with its weights (512 rows behind 32768 positions, 8 cache
// heads: 73 us, 940 TFLOP/s).  Up to 128 rows leave the second tile free: it takes the same rows against every other step (`split`), and hands its
// sums to the first at the end.
// Warps 0-3 and 4-7: softmax of a tile each; 8 and 9: loads; 10: products (twelve warps leave a thread 168 registers).  Keys and values lie as
// the products read them (rows of 64 channels, 128-byte swizzle); the ring alternates units of 128 keys and 128 values.  They arrive by
// TMA in boxes of as many positions as divide both a page and a step, where those are at least the swizzle's eight; pages of other
// sizes, and the last step of a range, whose unseen values have to be zeros, by 16-byte asynchronous copies with an address for each
// position (as the only way they held a step at 4500 clocks).
constexpr int kWideRows = 256, kWideStep = 128, kWideRing = 4, kLoaders = 2, kWideThreads = 12 * 32;
constexpr uint32_t kBox = 16384;   // 128 rows of 128 bytes

struct WideShared {
  float2 stat[128];         // split: reference and sum of the second tile's rows
  uint64_t full[kWideRing], empty[kWideRing], q_full, s_full[2], p_half[2], p_full[2], o_done[2], handed, drained;
  uint32_t seen[4][4];   // which of a step's positions can be seen; a step's words are written at most two steps ahead
  uint32_t tmem;
  int abort;
};
template <typename T, int D>
__global__ void __launch_bounds__(kWideThreads, 1)
wide_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap keys, const __grid_constant__ CUtensorMap values) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ WideShared w;
  constexpr int kBoxes = D / 64, kPieces = D / 8;
  constexpr uint32_t kUnit = kBoxes * kBox;
  const uint32_t smem = (shared_address(smem_raw) + 1023u) & ~1023u, s_q = smem, s_ring = smem + 2 * kUnit;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.y;
  if (p.wide_first) grid_dependency_wait();
  launch_dependents();
  int row0, n_rows, begin, end, slot;
  const int* pages;
  if ((int)blockIdx.x < p.wide_tiles * p.prefix_chunks) {
    const int chunk = blockIdx.x / p.wide_tiles;
    row0 = (blockIdx.x - chunk * p.wide_tiles) * kWideRows;
    n_rows = min(kWideRows, p.rows - row0);
    begin = chunk * p.prefix_chunk;
    end = min(begin + p.prefix_chunk, p.a.prefix_length);
    pages = p.prefix_pages;
    slot = chunk;
  } else {
    const int item = blockIdx.x - p.wide_tiles * p.prefix_chunks, b = item % p.a.batch, rest = item / p.a.batch;
    const int chunk = rest / p.own_wide_tiles, tile = rest - chunk * p.own_wide_tiles, per = p.a.queries * p.group;
    row0 = b * per + tile * kWideRows;
    n_rows = min(kWideRows, per - tile * kWideRows);
    begin = chunk * p.own_wide_chunk;
    end = min(begin + p.own_wide_chunk, common_length(p, own_length(p, b)));
    if (begin >= end) { grid_dependency_wait(); return; }
    pages = p.page_table + (int64_t)b * p.a.table_width;
    slot = p.prefix_chunks + chunk;
  }
  const int steps = (end - begin + kWideStep - 1) / kWideStep;
  const bool split = n_rows <= 128;
  constexpr uint32_t kColumns = 512;
  if (threadIdx.x == 0) {
    if (p.box_shift) { prefetch_map(&keys); prefetch_map(&values); }
    for (int i = 0; i < kWideRing; ++i) { mbar_init(&w.full[i], kLoaders * 33); mbar_init(&w.empty[i], 1); }
    mbar_init(&w.q_full, split ? 4 : 8);
    for (int t = 0; t < 2; ++t) { mbar_init(&w.s_full[t], 1); mbar_init(&w.p_half[t], 4); mbar_init(&w.p_full[t], 4); mbar_init(&w.o_done[t], 1); }
    mbar_init(&w.handed, 4);
    mbar_init(&w.drained, 1);
    w.abort = 0;
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

  if (warp < 8) {
    // ------------------------------------------------------------------- softmax ----
    const int tile = warp >> 2, quarter = warp & 3, in_tile = quarter * 32 + lane, r = split ? in_tile : tile * 128 + in_tile;
    {
      const bool live = r < n_rows;
      const int row = row0 + (live ? r : 0), g = row % p.group, j = row / p.group % p.a.queries, b = row / (p.group * p.a.queries);
      // (a negative scale becomes the sign of the queries: the largest score is then the largest product)
      if (!(split && tile)) {
        const uint4* q = (const uint4*)((const T*)p.q + b * p.a.q_batch + j * p.a.q_token + (int64_t)(head * p.group + g) * p.a.q_head);
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
      const int own_steps = split ? (steps - tile + 1) / 2 : steps;
      for (int i = 0; i < own_steps; ++i) {
        const int step = split ? 2 * i + tile : i;
        if (!warp_wait(&w.s_full[tile], i & 1)) { ok = false; break; }
        tc_fence_after();
        uint32_t seen[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) seen[c] = *(volatile uint32_t*)&w.seen[step & 3][c];
        const bool whole = (seen[0] & seen[1] & seen[2] & seen[3]) == ~0u;
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
      // All products done, queries and ring are free: the rows of the result go there (16 bytes apart from each other's banks), and each on as one
      // copy (a thread's own stores, 16 bytes of 32 rows at a time, took 3.6 us).
      if (ok) ok = warp_wait(&w.o_done[0], 0);
      if (ok && (!split || steps > 1)) ok = warp_wait(&w.o_done[1], 0);
      tc_fence_after();
      constexpr uint32_t kRow = D * 4 + 16;
      const uint32_t row_at = smem + (uint32_t)r * kRow;
      const bool hands = split && tile, takes = split && !tile && steps > 1;
      if (hands) w.stat[in_tile] = make_float2(ok ? reference : 0.f, ok ? sum : __int_as_float(0x7fc00000));
      float mine = 1.f, theirs = 0.f;
      if (takes) {
        if (ok) ok = warp_wait(&w.handed, 0);
        if (ok) {
          const float2 st = w.stat[in_tile];
          const float top = fmaxf(reference, st.x), base = top == -INFINITY ? 0.f : top;
          mine = exp2_fast(reference - base);
          theirs = exp2_fast(st.x - base);
          sum = sum * mine + st.y * theirs;
          reference = top;
        }
      }
      if (ok && own_steps) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[32];
          tmem_ld32(t_o + c * 32, v);
          tmem_ld_wait32(v);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t to = row_at + c * 128 + k * 16;
            float x[4] = {__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]), __uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3])};
            if (takes) {
              float y[4];
              asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]) : "r"(to) : "memory");
#pragma unroll
              for (int h = 0; h < 4; ++h) x[h] = x[h] * mine + y[h] * theirs;
            }
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]) : "memory");
          }
        }
      }
      if (hands) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&w.handed);
      } else if (live) {
        const int64_t at = ((int64_t)head * p.rows + row) * p.slots + slot;
        p.stat[at] = make_float2(ok ? reference : 0.f, ok ? sum : __int_as_float(0x7fc00000));
        if (ok) {
          fence_async_proxy();
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.part + at * D), "r"(row_at), "n"(D * 4) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
      }
      tc_fence_before();
    }
  } else if (warp < 8 + kLoaders) {
    // --------------------------------------------------------------------- loads ----
    const int part = warp - 8;
    const T *kc = (const T*)p.k + (int64_t)head * p.a.c_head, *vc = (const T*)p.v + (int64_t)head * p.a.c_head;
    // Page numbers are asked for one step early: of the box that this lane brings, or of the positions whose copies it knows the address of.
    constexpr int kEach = 4 / kLoaders;   // groups of 32 positions
    int page[kEach], box_page = -1;
    int64_t off[kEach];
    const int boxes = p.box_shift ? kWideStep >> p.box_shift : 0;
    auto by_box = [&](int step) { return p.box_shift && begin + (step + 1) * kWideStep <= end; };
    auto position = [&](int step, int h) { return begin + step * kWideStep + (part * kEach + h) * 32 + lane; };
    auto ask = [&](int step) {
      if (by_box(step)) {
        if (lane < boxes) box_page = pages[(begin + step * kWideStep + (lane << p.box_shift)) / p.a.page_size];
      } else {
#pragma unroll
        for (int h = 0; h < kEach; ++h) page[h] = position(step, h) < end ? pages[position(step, h) / p.a.page_size] : -1;
      }
    };
    int box_coord = 0, box_at = 0, loaded = 0;
    ask(0);
    for (int u = 0; u < 2 * steps; loaded = ++u) {
      const int step = u >> 1;
      uint64_t* full = &w.full[u % kWideRing];
      const uint32_t dst = s_ring + (u % kWideRing) * kUnit;
      if (!warp_wait(&w.empty[u % kWideRing], ((u / kWideRing) & 1) ^ 1)) break;
      const bool skip = p.test_skip_stage && blockIdx.x == 0 && u == 1;
      if (by_box(step)) {
        if (!(u & 1)) {
          const bool there = box_page >= 0 && box_page < p.a.pages;
          box_coord = there ? box_page : p.a.pages;   // (past the last page: zeros)
          box_at = (begin + step * kWideStep + (lane << p.box_shift)) % p.a.page_size;
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
          const int n = i * 32 + lane, r = n / kPieces, c = n % kPieces;
          const int64_t o = __shfl_sync(~0u, off[h], r);
          copy16(row0_at + (c >> 3) * kBox + r * 128 + (((c & 7) ^ (r & 7)) << 4), base + (o < 0 ? 0 : o) + c * 8, o >= 0);
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
      for (int i = 0; i < kWideRing; ++i) await_landing(&w.full[i], loaded > i ? (uint32_t)((loaded - 1 - i) / kWideRing & 1) : 1u);   // boxes in flight land before their memory goes
  } else if (warp == 8 + kLoaders && elect_one()) {
    // ------------------------------------------------------------------ products ----
    const uint32_t fmt = Mma<T>::kBf16 ? 1u : 0u, common = (1u << 4) | (fmt << 7) | (fmt << 10) | (8u << 24);
    const uint32_t idesc_s = common | ((uint32_t)(kWideStep >> 3) << 17), idesc_o = common | (1u << 16) | ((uint32_t)(D >> 3) << 17);   // (V lies with channels innermost)
    const uint64_t hi = (uint64_t)(((8u * 128u) >> 4) | (1u << 14) | (2u << 29)) << 32;
    // the distance between two boxes of channels is only read for V, whose 64-channel groups are a box apart
    auto desc = [&](uint32_t at, uint32_t lead) { return hi | ((uint64_t)lead << 16) | (uint64_t)((at & 0x3FFFF) >> 4); };
    // (keys and values were written by copies of other threads, which the barrier has told of: the fence makes them visible to the products)
    auto landed = [&](int u) {
      const bool there = wait(&w.full[u % kWideRing], (u / kWideRing) & 1);
      fence_async_proxy();
      return there;
    };
    bool ok = wait(&w.q_full, 0);
    auto scores = [&](int i, int t) {   // S_t = Q_t K_i^T
      const uint32_t k = s_ring + (2 * i % kWideRing) * kUnit, q = s_q + (split ? 0u : t * kUnit);
#pragma unroll
      for (int n = 0; n < D / 16; ++n)
        umma_f16(tmem + t * 128, desc(q + (n >> 2) * kBox + (n & 3) * 32, 1), desc(k + (n >> 2) * kBox + (n & 3) * 32, 1), idesc_s, n ? 1u : 0u);
      umma_commit(&w.s_full[t]);
    };
    // Every tile takes every step; split, step i belongs to tile i & 1, whose next one is i + 2.
    const int ahead = split ? 2 : 1;
    for (int i = 0; i < min(ahead, steps) && ok; ++i) {
      ok = landed(2 * i);
      if (!ok) break;
      tc_fence_after();
      if (split) scores(i, i); else for (int t = 0; t < 2; ++t) scores(i, t);
      umma_commit(&w.empty[2 * i % kWideRing]);
    }
    for (int i = 0; i < steps && ok; ++i) {
      const int vu = 2 * i + 1, ku = 2 * (i + ahead), t0 = split ? i & 1 : 0, t1 = split ? t0 : 1, turn = split ? i >> 1 : i;
      const bool more = i + ahead < steps;
      for (int t = t0; t <= t1 && ok; ++t) {
        if (t == t0) ok = landed(vu);
        const uint32_t v = s_ring + (vu % kWideRing) * kUnit;
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
        if (t == t1) umma_commit(&w.empty[vu % kWideRing]);
        if (!more) { umma_commit(&w.o_done[t]); continue; }
        if (t == t0) ok = landed(ku);
        if (!ok) break;
        tc_fence_after();
        scores(i + ahead, t);
        if (t == t1) umma_commit(&w.empty[ku % kWideRing]);
      }
    }
    if (!ok) { umma_commit(&w.drained); await_landing(&w.drained, 0); }   // products in flight end before their memory goes
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8 + kLoaders) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
  grid_dependency_wait();   // the end of this grid is the end of tile_kernel's, which it may have started under
}

// The sum over a row's slots, by a warp or, for more than sixteen slots, by the four of a block.  Statistics and partial results are asked for at
// once, before it is known which slots were written: the kernel is a chain of latencies.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ Params p) {
  constexpr int N = D / 32;
  __shared__ float shared_acc[kWarps][D];
  __shared__ float2 shared_stat[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = p.join_warps, part_of = share == 1 ? 0 : warp;
  const int64_t id = share == 1 ? (int64_t)blockIdx.x * kWarps + warp : blockIdx.x;   // head * rows + row
  const bool live = id < (int64_t)p.rows * p.a.kv_heads;
  const int head = live ? (int)(id / p.rows) : 0, row = live ? (int)(id - (int64_t)head * p.rows) : 0;
  const int g = row % p.group, j = row / p.group % p.a.queries, b = row / (p.group * p.a.queries);
  grid_dependency_wait();
  if (!live) return;   // (whole blocks where a block shares a row)
  const int length = own_length(p, b);
  // slots part_of, part_of + share, ...
  const float2* stat = p.stat + id * p.slots;
  const float* part = p.part + id * p.slots * D + lane * N;
  float x[8][N];
  auto fetch = [&](int from) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float* src = part + (int64_t)min((from + e) * share + part_of, p.slots - 1) * D;
      if constexpr (N == 4) { const float4 v = *(const float4*)src; x[e][0] = v.x; x[e][1] = v.y; x[e][2] = v.z; x[e][3] = v.w; }
      else { const float2 v = *(const float2*)src; x[e][0] = v.x; x[e][1] = v.y; }
    }
  };
  float top = -INFINITY, sum = 0.f, acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  if (p.slots) {
    float2 st = stat[min(lane * share + part_of, p.slots - 1)];
    fetch(0);
    // slots that were written: all of the prefix's, as many of the sequence's as it has positions for, and that of the last positions
    const int span = p.own_wide_tiles ? common_length(p, length) : length, chunk = p.own_wide_tiles ? p.own_wide_chunk : p.own_chunk;
    const int first = p.prefix_chunks + (span > 0 ? (span + chunk - 1) / chunk : 0);
    const bool tail = p.own_wide_tiles && p.own_chunks && length > span;
    const int last = p.prefix_chunks + p.own_wide_chunks, all = ((tail ? last + 1 : first) + share - 1) / share;
    for (int i0 = 0; i0 < all; i0 += 32) {
      const int i = (i0 + lane) * share + part_of;
      const bool written = i < first || (tail && i == last);
      if (i0) st = stat[min(i, p.slots - 1)];
      float mx = written ? fmaxf(top, st.x) : top;
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
      const float base = mx == -INFINITY ? 0.f : mx, f = written ? exp2_fast(st.x - base) : 0.f, corr = exp2_fast(top - base);
      top = mx;
      float s = written ? f * st.y : 0.f;
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
      sum = sum * corr + s;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] *= corr;
      const uint32_t there = __ballot_sync(~0u, written);
      for (int m = 0; m < min(32, all - i0); m += 8) {
        if (i0 + m) fetch(i0 + m);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = __shfl_sync(~0u, f, m + e);
          if (there >> (m + e) & 1) {
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] += w * x[e][k];
          }
        }
      }
    }
  }
  if (share > 1) {
#pragma unroll
    for (int k = 0; k < N; ++k) shared_acc[warp][lane * N + k] = acc[k];
    if (lane == 0) shared_stat[warp] = make_float2(top, sum);
    __syncthreads();
    if (warp) return;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, shared_stat[w].x);
    const float base = mx == -INFINITY ? 0.f : mx;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 st = shared_stat[w];
      const float f = exp2_fast(st.x - base);
      sum += f * st.y;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += f * shared_acc[w][lane * N + k];
    }
  }
  T* y = (T*)p.y + b * p.a.y_batch + j * p.a.y_token + (int64_t)(head * p.group + g) * p.a.y_head + lane * N;
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int k = 0; k < N; k += 2) *(uint32_t*)(y + k) = Mma<T>::pack(acc[k] * inverse, acc[k + 1] * inverse);
}

constexpr int kChunkLeast = 128, kChunkMost = 4096;                // positions of a chunk
constexpr int kEnoughTiles = 5 * 148, kEnoughTeams = 2 * 148;      // blocks from which on chunks are not cut further
constexpr int64_t kPrefixSlots = 1 << 17, kPrefixChunks = 16;      // the wide kernel's partial results of the prefix: as many in all, or for each row
int64_t pieces(int64_t n, int64_t of) { return (n + of - 1) / of; }

// Partial results (of one row of one head each) that the workspace has room for: at least as many as plan() chooses, and no fewer for a larger
// batch, table or prefix or for more queries or heads.  What plan() chooses does not grow like that, because fewer sequences are cut into more chunks;
// but where it halves chunks it had less than `enough` blocks before, and has less than twice as many then.
int64_t room_for(const PagedAttention& a) {
  const int64_t per = (int64_t)a.queries * (a.heads / a.kv_heads), rows = a.batch * per, all = rows * a.kv_heads, own = (int64_t)a.table_width * a.page_size;
  int64_t prefix = 0;
  if (a.prefix_length) {
    const int64_t least = pieces(a.prefix_length, kChunkLeast), most = pieces(a.prefix_length, kChunkMost), few = std::min<int64_t>(rows, kRows);
    prefix = std::min(few * a.kv_heads * least, std::max(few * a.kv_heads * most, few * 2 * kEnoughTiles));
    if (rows > kRows) prefix = std::max(prefix, std::min(all * std::min<int64_t>(least, 64), std::max(kPrefixSlots, kPrefixChunks * all)));
  }
  // a block has up to 16 rows of a sequence, a team's up to 64, the wide kernel's up to 256
  const int64_t cut = std::max(std::min<int64_t>(per, kRows) * 2 * kEnoughTiles, std::min<int64_t>(per, kWideRows) * 2 * kEnoughTeams);
  const int64_t tail = a.queries > 1 && per > 4 * kRows && own > kWideStep ? all : 0;
  return prefix + std::min(all * pieces(own, kChunkLeast), std::max(all * pieces(own, kChunkMost), cut)) + tail;
}

Params plan(const PagedAttention& a) {
  Params p{};
  p.a = a;
  p.group = a.heads / a.kv_heads;
  p.rows = a.batch * a.queries * p.group;
  p.scale_log2e = a.scale * kLog2e;
  while ((1ll << p.page_shift) < a.page_size) ++p.page_shift;
  p.page_shift += 30;
  p.page_factor = (uint32_t)((1ull << p.page_shift) / a.page_size + 1);   // factor * page_size exceeds 2^shift by at most page_size <= 2^(shift - 30)
  p.prefix_tiles = (p.rows + kRows - 1) / kRows;
  const int64_t per = (int64_t)a.queries * p.group;
  p.team = per <= kRows ? 1 : per <= 2 * kRows ? 2 : 4;
  p.own_tiles = (int)((per + kRows * p.team - 1) / (kRows * p.team));
  const int64_t own_max = (int64_t)a.table_width * a.page_size;
  // Chunks for tile_kernel: two and a half blocks for each of the 296 that run at once even out ragged lengths (128 sequences of up to 900
  // positions, 4 rows: whole 55.9 us, 512 57.7); of teams, whose block takes four times as long over a chunk, one (16 sequences of up to 2500
  // positions, 35 rows: 512 positions 32 us, 256 35; 40 rows of one: 128 14.9, 512 25).
  auto chunk_of = [&](int64_t positions, int64_t tiles) {
    int64_t chunk = kChunkMost;
    while (chunk > kChunkLeast && tiles * a.kv_heads * pieces(positions, chunk) < (p.team == 1 ? kEnoughTiles : kEnoughTeams)) chunk /= 2;
    return (int)chunk;
  };
  if (a.prefix_length && p.rows > kRows) {
    // Blocks of equal work on 148 SMs: the number of chunks with the shortest estimate of waves of steps (1.9 us each, 1.1 us split; 5 us at both ends) and of
    // the partial results' way to memory and back; up to 64, for many rows less, to bound the workspace (by the estimate that costs at most 5 %, and
    // only from 3000 rows of all heads and 97000 positions on).
    p.wide_tiles = (p.rows + kWideRows - 1) / kWideRows;
    const int tiles = p.wide_tiles * a.kv_heads, all = (a.prefix_length + kWideStep - 1) / kWideStep;
    const int64_t most = std::min<int64_t>(64, std::max(kPrefixChunks, kPrefixSlots / ((int64_t)p.rows * a.kv_heads)));
    double best = 1e30;
    for (int c = 1; c <= all && c <= most; ++c) {
      const int steps = (all + c - 1) / c;
      const double us = (double)((tiles * (int64_t)c + 147) / 148) * (steps * (p.rows > 128 ? 1.9 : 1.1) + 5.0) + (double)c * p.rows * a.kv_heads * a.channels * 8 / 5e6;
      if (us < best) { best = us; p.prefix_chunk = steps * kWideStep; }
    }
    p.prefix_tiles = 0;
  } else {
    p.prefix_chunk = chunk_of(a.prefix_length, p.prefix_tiles);
  }
  p.prefix_chunks = (a.prefix_length + p.prefix_chunk - 1) / p.prefix_chunk;
  // (up to four tiles of 16 rows take a team less time than the wide kernel's blocks need to begin and end: 35 rows as above 32 us and 47; 64 to
  // 256 rows fill its tiles)
  if (per > 4 * kRows && own_max > kWideStep) {
    p.own_wide_tiles = (int)((per + kWideRows - 1) / kWideRows);
    const int64_t all = (own_max + kWideStep - 1) / kWideStep, tiles = (int64_t)p.own_wide_tiles * a.batch * a.kv_heads;
    int64_t steps = kChunkMost / kWideStep;
    while (steps > 4 && tiles * pieces(all, steps) < kEnoughTeams) steps /= 2;
    p.own_wide_chunk = (int)steps * kWideStep;
    p.own_wide_chunks = (int)((all + steps - 1) / steps);
    p.own_chunk = (a.queries - 1 + kStep - 1) / kStep * kStep;
    p.own_chunks = a.queries > 1 ? 1 : 0;
  } else {
    p.own_chunk = chunk_of(own_max, (int64_t)p.own_tiles * a.batch);
    p.own_chunks = (int)((own_max + p.own_chunk - 1) / p.own_chunk);
  }
  p.slots = p.prefix_chunks + p.own_wide_chunks + p.own_chunks;
  p.join_warps = p.slots > 16 ? kWarps : 1;   // (10 slots of 4096 rows: one warp 118 us for the whole call, four 124.6)
  return p;
}

int64_t tile_items(const Params& p) { return (int64_t)p.prefix_tiles * p.prefix_chunks + (int64_t)p.a.batch * p.own_tiles * p.own_chunks; }
int64_t wide_tile_items(const Params& p) { return (int64_t)p.wide_tiles * p.prefix_chunks + (int64_t)p.a.batch * p.own_wide_tiles * p.own_wide_chunks; }

// Up to three launches: tiles of 16 rows, wide tiles, the sum.  All may start while the kernel in front still runs, and wait where they need its
// results: the first at its start; the wide kernel, which reads nothing that the first writes, only before it ends (a grid that waited has
// ended after all in front of it); the sum at its start.
template <typename T, int D> int launch(Params& p, cudaStream_t stream) {
  const int64_t items = tile_items(p), wide_items = wide_tile_items(p);
  constexpr size_t ring = (size_t)kWarps * kRing * kStep * D * 2, merge = (size_t)kWarps * kRows * (D + 4) * 4 + kWarps * kRows * 8, smem = ring > merge ? ring : merge;
  constexpr size_t wide = (size_t)(2 + kWideRing) * (D / 64) * kBox + 1024;
  const unsigned heads = (unsigned)p.a.kv_heads;
  auto* tiles = p.team == 1 ? tile_kernel<T, D, 1> : p.team == 2 ? tile_kernel<T, D, 2> : tile_kernel<T, D, 4>;
  if (items && !start(tiles, dim3((unsigned)items, heads), kThreads, smem, stream, p)) return -2;
  if (wide_items) {
    p.wide_first = items == 0;
    CUtensorMap keys{}, values{};
    p.box_shift = 0;
    int shift = 0;
    while (shift < 7 && p.a.page_size % (2 << shift) == 0) ++shift;
    if (shift >= 3 && box_map(&keys, p.a, p.k, 1 << shift) && box_map(&values, p.a, p.v, 1 << shift)) p.box_shift = shift;
    if (!start(wide_kernel<T, D>, dim3((unsigned)wide_items, heads), kWideThreads, wide, stream, p, keys, values)) return -2;
  }
  const int64_t ids = (int64_t)p.rows * p.a.kv_heads;
  return start(join_kernel<T, D>, dim3((unsigned)(p.join_warps == 1 ? (ids + kWarps - 1) / kWarps : ids)), kThreads, 0, stream, p) ? 0 : -2;
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttention& a) {
  if (a.batch == 0) return 0;
  const Params p = plan(a);
  if (tile_items(p) >= (1ll << 31) || wide_tile_items(p) >= (1ll << 31)) return -1;   // more blocks than a grid has
  return room_for(a) * ((int64_t)a.channels * 4 + 8);
}

int paged_attention(const PagedAttention& a, const void* key_cache, const void* value_cache, const void* q, const int* prefix_pages, const int* page_table, const int* lengths,
                    void* y, void* workspace, cudaStream_t stream) {
  Params p = plan(a);
  p.k = key_cache; p.v = value_cache; p.q = q; p.y = y;
  p.prefix_pages = prefix_pages; p.page_table = page_table; p.lengths = lengths;
  p.spin_limit = kSpinLimit;
  p.test_skip_stage = getenv("ODLA_B200_TEST_SKIP_STAGE") != nullptr;
  if (const char* e = getenv("ODLA_B200_TEST_SPIN_LIMIT")) { const long v = atol(e); if (v >= 64 && v <= (1l << 18)) p.spin_limit = (uint32_t)v; }
  p.part = (float*)workspace;
  p.stat = (float2*)(p.part + (int64_t)p.rows * a.kv_heads * p.slots * a.channels);
  if (a.dt == DT_F16) return a.channels == 64 ? launch<__half, 64>(p, stream) : launch<__half, 128>(p, stream);
  return a.channels == 64 ? launch<__nv_bfloat16, 64>(p, stream) : launch<__nv_bfloat16, 128>(p, stream);
}

}  // namespace b200
