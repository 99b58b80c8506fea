// The instructions that the attention kernels are built on: mbarriers, tile copies (TMA), and the fifth-generation
// tensor cores with their accumulators in tensor memory (tcgen05).
//
// Every wait on an mbarrier is bounded: where it runs out, the kernel sets a status word in host memory (the next call and
// csw_device_status look at it), its warps leave their loops, and it fills its results with NaN, frees its tensor memory
// and returns.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "values.cuh"

namespace csw {
namespace tc {

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---- mbarriers ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
__device__ __forceinline__ bool bar_wait_on(uint32_t bar, uint32_t parity, long long patience) {
  const long long start = clock64();
  do {
    if (bar_try(bar, parity)) return true;
  } while (clock64() - start < patience);
  return false;
}
// true once the phase of this parity is over; false where it does not end within `patience` clocks or so
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, long long patience) {
  return bar_try(bar, parity) || bar_wait_on(bar, parity, patience);
}
__device__ __forceinline__ void init_visible() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
// shared memory written by ordinary stores, before the tensor cores or a tile copy see it
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- copies into shared memory -------------------------------------------------------------------------------------
// a tile of [dim, token, head, batch] coordinates; dim is a multiple of 8 two-byte values (16 bytes)
__device__ __forceinline__ void copy_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int dim, int token, int head,
                                          int batch) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(dim), "r"(token), "r"(head), "r"(batch)
      : "memory");
}
// bytes (a multiple of 16) from a 16-byte boundary
__device__ __forceinline__ void copy_bytes(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// ---- copies out of shared memory -----------------------------------------------------------------------------------
// what of the tile lies behind the tensor is left out
__device__ __forceinline__ void store_tile(const CUtensorMap* map, uint32_t src, int dim, int token, int head, int batch) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map),
               "r"(src), "r"(dim), "r"(token), "r"(head), "r"(batch)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// the source of this thread's stores may be written again
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// Some warps of a CTA that meet again and again, on an mbarrier with an arrival for each of them.  Its wait is bounded,
// where a bar.sync with a warp that has given up would never end.  A meeting cannot end before all have come to it, so
// that nobody is two ahead and the parity tells.
struct Meeting {
  uint32_t bar;
  long long patience;
  uint32_t met = 0;
  // false where the others have not come
  __device__ __forceinline__ bool operator()() {
    __syncwarp();  // what all lanes have written is in front of the arrival
    if (threadIdx.x % 32 == 0) bar_arrive(bar);
    return __all_sync(0xffffffffu, bar_wait(bar, met++ & 1, patience));
  }
};

// ---- work ----------------------------------------------------------------------------------------------------------
// Asks for a CTA of this grid that has not started: it will not start, and its work is the caller's.  The answer (16
// bytes) arrives at `bar`.  Not to be asked again after a refusal.
__device__ __forceinline__ void take_next(uint32_t answer, uint32_t bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer),
      "r"(bar)
      : "memory");
}
// the index of the CTA that was taken, -1 for a refusal
__device__ __forceinline__ int taken_index(uint32_t answer) {
  int index;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}"
      : "=r"(index)
      : "r"(answer)
      : "memory");
  return index;
}

// ---- tensor memory -------------------------------------------------------------------------------------------------
// by one whole warp; the address arrives at *at in shared memory
template <int COLUMNS>
__device__ __forceinline__ void tmem_alloc(uint32_t at) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at), "n"(COLUMNS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLUMNS>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLUMNS));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define CSW_R4(a, i) a(i), a(i + 1), a(i + 2), a(i + 3)
#define CSW_R16(a, i) CSW_R4(a, i), CSW_R4(a, i + 4), CSW_R4(a, i + 8), CSW_R4(a, i + 12)
#define CSW_R32(a, i) CSW_R16(a, i), CSW_R16(a, i + 16)
#define CSW_OUT(i) "=r"(r[i])
#define CSW_IN(i) "r"(r[i])
#define CSW_BOTH(i) "+r"(r[i])
// 32 columns of the lane that is this thread's (lane 32 (warp % 4) + thread % 32; `at` names the warp's first lane)
__device__ __forceinline__ void load32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : CSW_R32(CSW_OUT, 0)
      : "r"(at));
}
// All loads are there; the 32 values depend on it, so that nothing that uses them can stand in front.
__device__ __forceinline__ void wait_loads(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : CSW_R32(CSW_BOTH, 0)::"memory");
}
// what has been computed up to here is not put off
__device__ __forceinline__ void settle(float& a, float& b, float& c, float& d) {
  asm volatile("" : "+f"(a), "+f"(b), "+f"(c), "+f"(d));
}
__device__ __forceinline__ void store32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::CSW_R32(CSW_IN, 0),
      "r"(at)
      : "memory");
}
__device__ __forceinline__ void store16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::CSW_R16(CSW_IN, 0),
      "r"(at)
      : "memory");
}
#undef CSW_R4
#undef CSW_R16
#undef CSW_R32
#undef CSW_OUT
#undef CSW_IN
#undef CSW_BOTH

// ---- products ------------------------------------------------------------------------------------------------------
// Tiles in shared memory are rows of 128 bytes, swizzled over 8 rows as the tile copies leave them.  Read along its
// rows (the reduction runs along a row), 16 two-byte values of the reduction are 32 bytes further in the row; read
// across them (the reduction runs over rows), they are 16 rows, 2048 bytes, further on.
// (The address field holds units of 16 bytes, so that steps are added to the whole word.)
__device__ __forceinline__ uint64_t tile_desc(uint32_t at, uint32_t lbo) {
  return (uint64_t)((at & 0x3ffff) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// 128 x N products of two-byte values, sums in float32.  across: the second operand's tile is read across its rows.
__host__ __device__ constexpr uint32_t product_desc(bool bf16, int n, bool across, bool negate) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (negate ? 1u << 13 : 0u) | (across ? 1u << 16 : 0u) |
         (uint32_t)(n / 8) << 17 | (uint32_t)(128 / 16) << 24;
}
// One lane of a warp whose lanes are together, the same one every time.  What the products take lies in registers that a
// warp shares; code that a whole warp runs, up to the instruction itself, computes there, where a lane on its own has to
// move every operand over (a step of a product then took some 100 clocks to issue instead of its 32 to 64).
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes;
}
// one reduction step of 16: both operands in shared memory
__device__ __forceinline__ void mma(uint32_t acc, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(acc),
      "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
      : "memory");
}
// the first operand in tensor memory, two values a column
__device__ __forceinline__ void mma_tmem(uint32_t acc, uint32_t a, uint64_t b, uint32_t desc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(acc),
      "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
      : "memory");
}
// arrives at `bar` when all products issued before have ended
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Maxima that a NaN among their operands makes NaN.
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x without the unit for it: 2^n for the whole part n is put together as a number, 2^f for the rest, -1/2 ... 1/2, is a
// polynomial of degree 5 (fitted for the least relative error, 1.6 10^-7).  x up to 127; from -126.5 down it gives 0, and
// NaN for a NaN: the exponent is multiplied in, since added to the bits of a NaN it would make a number of them.
__device__ __forceinline__ Pair exp2_poly(Pair x) {
  constexpr float kMagic = 12582912.0f;  // 1.5 2^23: a sum with it is rounded to a whole number, its low bits
  x.x = max2(x.x, -127.0f), x.y = max2(x.y, -127.0f);
  const Pair t = add2(x, {kMagic, kMagic});
  const Pair n = add2(t, {-kMagic, -kMagic});
  const Pair f = fma2(n, {-1.0f, -1.0f}, x);
  Pair p = fma2(f, {0.0013276472454890609f, 0.0013276472454890609f}, {0.009675540961325169f, 0.009675540961325169f});
  p = fma2(p, f, {0.05550713092088699f, 0.05550713092088699f});
  p = fma2(p, f, {0.24022120237350464f, 0.24022120237350464f});
  p = fma2(p, f, {0.6931469440460205f, 0.6931469440460205f});
  p = fma2(p, f, {1.0000001192092896f, 1.0000001192092896f});
  const Pair power = {__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                      __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)};
  return mul2(p, power);
}

}  // namespace tc
}  // namespace csw
