// What the kernels of attention over a paged cache share: two-byte types, asynchronous copies, tensor memory, exponentials, boxes of a cache, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"
#include "tensor_maps.h"
#include "umma_ptx.cuh"

namespace b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Mma;
template <> struct Mma<__half> {
  static constexpr bool kBf16 = false;
  static constexpr float kLift = 7.f;   // (see wide_kernel)
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const uint32_t*)&h;
  }
  static __device__ __forceinline__ uint32_t times_zero(uint32_t x, uint32_t sum) {   // of two values, plus the sum
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u));
    return sum;
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y, float& sum) {   // adds the values as rounded
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    sum += f.x + f.y;
    return *(const uint32_t*)&h;
  }
};
template <> struct Mma<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *(const uint32_t*)&h;
  }
  static __device__ __forceinline__ uint32_t times_zero(uint32_t x, uint32_t sum) {
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u));
    return sum;
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y, float& sum) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const uint32_t u = *(const uint32_t*)&h;
    sum += __uint_as_float(u << 16) + __uint_as_float(u & 0xffff0000u);
    return u;
  }
};

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes, or zeros (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool any) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(any ? 16 : 0) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
  return x;
}
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void umma_tmem_a(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
               "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}
// The wait for a load, naming its registers so that no read of them is scheduled above it.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                 "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Two floats in one register pair.
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(uint32_t x, uint32_t y) { return pair_of(__uint_as_float(x), __uint_as_float(y)); }
__device__ __forceinline__ void unpack(uint64_t p, float (&e)[2]) { asm("mov.b64 {%0, %1}, %2;" : "=f"(e[0]), "=f"(e[1]) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x for two x <= 15 on the multiply-add pipes, for a quarter of all exponentials (256 rows behind 32768 positions: 92 -> 88.5 us; half of them: 94):
// x = n + f with n whole, |f| <= 1/2; the series of 2^f up to the fifth power, whose rest is below 2.5e-6 (a two-hundredth of half a step
// of fp16), times 2^n.  Below 2^-126.5, where 2^n has no exponent left, a weight is zero; NaN stays NaN.
__device__ __forceinline__ void exp2_pair(uint64_t x, float (&e)[2]) {
  float t[2];
  unpack(x, t);
#pragma unroll
  for (int h = 0; h < 2; ++h) asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(t[h]));   // -127
  x = pair_of(t[0], t[1]);
  // the sum's lowest bits are n + 127: shifted into place, 2^n
  const uint64_t shift = pair_of(12582912.f + 127.f, 12582912.f + 127.f), back = pair_of(-12582912.f - 127.f, -12582912.f - 127.f), minus = pair_of(-1.f, -1.f);
  const uint64_t n = add2(x, shift), f = fma2(add2(n, back), minus, x);
  constexpr float l = 0.69314718056f;
  uint64_t r = fma2(f, pair_of(l * l * l * l * l / 120, l * l * l * l * l / 120), pair_of(l * l * l * l / 24, l * l * l * l / 24));
  r = fma2(r, f, pair_of(l * l * l / 6, l * l * l / 6));
  r = fma2(r, f, pair_of(l * l / 2, l * l / 2));
  r = fma2(r, f, pair_of(l, l));
  r = fma2(r, f, pair_of(1.f, 1.f));
  float m[2];
  unpack(n, m);
  unpack(mul2(r, pair_of(__float_as_uint(m[0]) << 23, __float_as_uint(m[1]) << 23)), e);
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int channel, int position, int head, int page) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"((uint64_t)map),
               "r"(smem_u32(bar)), "r"(channel), "r"(position), "r"(head), "r"(page)
               : "memory");
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

struct True { static constexpr bool value = true; };
struct False { static constexpr bool value = false; };

template <typename F, typename... Args> bool start(F* fn, dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  if (smem > 48 * 1024 && cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) { cudaGetLastError(); return false; }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, fn, args...) == cudaSuccess) return true;
  cudaGetLastError();
  return false;
}

// Boxes of 64 channels and `positions` positions of one head and page.  False where the strides are none that TMA takes.
template <typename A> bool box_map(CUtensorMap* m, const A& a, const void* base, int positions) {
  if (!load_driver_entry_points()) return false;
  // (the stride of a dimension of one entry is never used, but has to be valid)
  auto bytes = [](int64_t stride, int extent) { return extent == 1 && stride == 0 ? (cuuint64_t)16 : (cuuint64_t)stride * 2; };
  const cuuint64_t dims[4] = {(cuuint64_t)a.channels, (cuuint64_t)a.page_size, (cuuint64_t)a.kv_heads, (cuuint64_t)a.pages};
  const cuuint64_t strides[3] = {bytes(a.c_token, a.page_size), bytes(a.c_head, a.kv_heads), bytes(a.c_page, a.pages)};
  for (cuuint64_t s : strides) if (s == 0 || s >= (1ull << 40)) return false;
  const cuuint32_t box[4] = {64, (cuuint32_t)positions, 1, 1}, step[4] = {1, 1, 1, 1};
  return g_encode_tiled(m, a.dt == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, (void*)base, dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace b200
