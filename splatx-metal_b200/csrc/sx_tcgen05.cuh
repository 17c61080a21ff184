// sx_tcgen05.cuh — the sm_100a instructions the tensor-core kernels are made of: mbarriers with
// bounded waits, TMA tile loads, tcgen05 matrix products with tensor memory, and their descriptors.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "sx_two.cuh"

namespace sx {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---- mbarriers ----
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Whether the phase of `parity` is complete; the warp sleeps until it is, or for about 0.1 ms.
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(100000)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {  // without waiting
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
constexpr long long kWaitCycles = 4000000000ll;  // two seconds at the highest clock

// Waits, as a whole warp, for the barrier's phase of `parity`. Gives up after two seconds, or once
// another warp of the CTA has: returns false then, the same for every lane, with *failed set. The
// waiting is left to the hardware: warps that poll take issue slots from those that compute.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* failed) {
    if (__all_sync(0xffffffffu, bar_test(bar, parity))) return true;
    const long long start = clock64();
    for (;;) {
        if (__all_sync(0xffffffffu, bar_try(bar, parity))) return true;
        if (__any_sync(0xffffffffu, *failed != 0 || clock64() - start > kWaitCycles)) {
            *failed = 1;
            return false;
        }
    }
}
// The same wait whatever *failed says: for copies and products still in flight when a kernel gives up.
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
    const long long start = clock64();
    while (!__all_sync(0xffffffffu, bar_try(bar, parity)) && !__any_sync(0xffffffffu, clock64() - start > kWaitCycles)) {
    }
}

// ---- TMA ----
// A box of a 4-axis tensor map (innermost axis first) into shared memory, counted on `bar`.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// `bytes` (a multiple of 16) of global memory into shared memory, both 16-byte aligned.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void fence_smem_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory ----
__device__ __forceinline__ void tmem_alloc(uint32_t to_smem, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to_smem), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define SX_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define SX_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 consecutive columns of the thread's lane.
__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : SX_R8(r, 0), SX_R8(r, 8), SX_R8(r, 16), SX_R8(r, 24)
        : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(at), SX_W8(r, 0), SX_W8(r, 8), SX_W8(r, 16), SX_W8(r, 24)
        : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(at), SX_W8(r, 0), SX_W8(r, 8)
        : "memory");
}
#define SX_T8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
// Waits for the thread's loads. The registers are named as changed behind the wait, so that the
// compiler moves no use of them before it.
__device__ __forceinline__ void changed(uint32_t (&r)[32]) {
    asm volatile("" : SX_T8(r, 0), SX_T8(r, 8));
    asm volatile("" : SX_T8(r, 16), SX_T8(r, 24));
}
template <typename... R>
__device__ __forceinline__ void wait_ld(R&... r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    (changed(r), ...);
}

// ---- matrix products ----
// Shared-memory operand in rows of 128 bytes with the 128-byte swizzle, as TMA writes them: 64
// 16-bit values a row, rows in groups of 8 (1024 bytes). `lead` (bytes) is the distance of the next
// 64 values of the row axis for an operand whose rows run along its M or N axis; an operand whose
// rows run along K does not use it.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
    return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | static_cast<uint64_t>((lead >> 4) & 0x3fff) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
template <typename T>
struct Format;
template <>
struct Format<__half> {
    static constexpr uint32_t code = 0;
};
template <>
struct Format<__nv_bfloat16> {
    static constexpr uint32_t code = 1;
};
// 128 x N product of T with 32-bit sums; `b_along_n`: B's rows in shared memory run along N.
template <typename T>
__host__ __device__ constexpr uint32_t shape(int n, bool b_along_n) {
    return 1u << 4 | Format<T>::code << 7 | Format<T>::code << 10 | (b_along_n ? 1u << 16 : 0u) |
           static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(128 >> 4) << 24;
}
// One lane of a converged warp, always the same one. The products are issued by the whole warp under
// this lane's predicate: their operands then stay in uniform registers. Behind a branch that one lane
// takes, each product waited some 80 cycles for its operands to get there.
__device__ __forceinline__ uint32_t elect() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
// D (tensor memory) = A B + (add ? D : 0) over 16 values of K, issued by the lane with `one`.
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add)), "r"(one)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(shape), "r"(static_cast<uint32_t>(add)), "r"(one)
        : "memory");
}
// Arrives on `bar` once every product that the lane with `one` has issued is complete.
__device__ __forceinline__ void commit(uint32_t one, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(one)
        : "memory");
}

// ---- registers ----
// A warpgroup's threads take more or fewer registers; the sum over the CTA stays within its launch's.
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// 32 bytes in one access (32-byte aligned): whole memory sectors.
__device__ __forceinline__ void store32(void* p, const uint32_t (&x)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), SX_W8(x, 0) : "memory");
}

// ---- values ----
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The largest; NaN where one of them is (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x on the multiply-add pipes, for x up to 127 (0 below -126.5, -inf among it: a masked key has no
// weight at all): x = n + f with n the nearest whole number, 2^f by a polynomial fitted for the least
// relative error on [-1/2, 1/2] (2.2e-7 in 32 bits), times 2^n. The low bits of x + 1.5 2^23 + 127 are
// n + 127, which is 2^n once they stand in the exponent's place, and zero for n = -127. The
// special-function unit gives 16 values a cycle and SM, half of what the products of 64-value rows leave
// time for.
__device__ __forceinline__ void exp2_poly(Two x, float& lo, float& hi) {
    float a, b;
    split(x, a, b);
    x = two(max_nan(a, -127.f), max_nan(b, -127.f));  // NaN stays, as it does in exp2_approx
    const Two magic = two(12583039.f, 12583039.f), back = two(-12583039.f, -12583039.f), minus = two(-1.f, -1.f);
    const Two t = add2(x, magic);
    const Two f = fma2(add2(t, back), minus, x);
    Two p = two(0x1.5c08e4p-10f, 0x1.5c08e4p-10f);
    p = fma2(p, f, two(0x1.3d0c52p-7f, 0x1.3d0c52p-7f));
    p = fma2(p, f, two(0x1.c6b6e4p-5f, 0x1.c6b6e4p-5f));
    p = fma2(p, f, two(0x1.ebf918p-3f, 0x1.ebf918p-3f));
    p = fma2(p, f, two(0x1.62e428p-1f, 0x1.62e428p-1f));
    p = fma2(p, f, two(0x1.000002p+0f, 0x1.000002p+0f));
    float n0, n1;
    split(t, n0, n1);
    split(mul2(p, two(__uint_as_float(__float_as_uint(n0) << 23), __uint_as_float(__float_as_uint(n1) << 23))), lo, hi);
}

}  // namespace tc
}  // namespace sx
