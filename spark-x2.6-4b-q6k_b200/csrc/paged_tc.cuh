// paged_tc.cuh — what the paged attention kernels on the tensor cores share: warp election, commits and fences, bounded
// waits that sleep, the rows' types.
#pragma once
#include "paged.cuh"

namespace spk {
namespace paged {
namespace {

__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// One thread of a warp that is together, always the same one.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The phase of that parity is over; sleeps up to a while before it says no, so that 20 waiting warps leave
// the issue slots to those that work.
__device__ __forceinline__ bool mbar_sleep(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
constexpr unsigned long long WAIT_NS = 4000000000ull;   // the longest wait
// Bounded wait. The first one that runs out records the error and marks the CTA dead; from then on
// waits return at once, copies and MMAs are no longer issued, and every warp still walks its range, so
// that none is left at a barrier.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, int *dead, int *err) {
    if (mbar_sleep(bar, parity)) return true;
    const unsigned long long t0 = now_ns();
    while (!(dead && *(volatile int *)dead)) {
        if (mbar_sleep(bar, parity)) return true;
        if (now_ns() - t0 > WAIT_NS) {
            if (dead) *(volatile int *)dead = 1;
            if (err) atomicExch(err, DEV_WAIT_TIMEOUT);
            break;
        }
    }
    return false;
}
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

}  // namespace
}  // namespace paged
}  // namespace spk
