/*
 * Transaction barriers and bulk copies into shared memory (sm_90+), with
 * bounded waits.
 */
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

__device__ __forceinline__ uint32_t kmb_smem(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ void kmb_mbar_init(uint64_t *bar, uint32_t arrivals) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(kmb_smem(bar)), "r"(arrivals) : "memory");
}
/* makes the initialised barriers visible to the copies' completion */
__device__ __forceinline__ void kmb_mbar_init_fence() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
/* one arrival that also announces `bytes` of copies */
__device__ __forceinline__ void kmb_mbar_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(kmb_smem(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void kmb_mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(kmb_smem(bar)) : "memory");
}
__device__ __forceinline__ bool kmb_mbar_done(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(kmb_smem(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}
/* Waits for the phase with `parity`, at most about 2^31 cycles; then *error
 * is set.  False when it gave up.  While *error is set every wait that is not
 * over after 16 looks gives up, of later launches too, until the host clears
 * the word: a caller that gave up lets its copies land before it ends
 * (kmb_mbar_done). */
__device__ __forceinline__ bool kmb_mbar_wait(uint64_t *bar, uint32_t parity, int *error) {
    long long t0 = 0;
    for (int n = 1; !kmb_mbar_done(bar, parity); ++n) {
        if (n % 16) continue;
        const long long t = clock64();
        if (n == 16) t0 = t;
        const bool late = t - t0 > (1ll << 31);
        if (late) atomicExch(error, 1);
        if (late || *reinterpret_cast<volatile int *>(error)) return false;
    }
    return true;
}

/* Kernels that follow one another in a call: the second is launched with
 * kmb_launch_after and begins with kmb_wait_before, which returns when the
 * first has ended and what it wrote is visible; the launch itself is then no
 * longer in between: 2 to 3 us a pair (layer norm backward 4096 x 1024 bf16
 * 18.1 -> 15.6 us).  kmb_let_after in the first: the second's CTAs may come
 * to wait on the SM as soon as every CTA of the first has been there. */
__device__ __forceinline__ void kmb_wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void kmb_let_after() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P>
cudaError_t kmb_launch_after(bool after, void (*k)(P...), dim3 grid, dim3 block, size_t shared, cudaStream_t s,
                             P... args) {
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = shared;
    cfg.stream = s;
    cfg.attrs = &at;
    cfg.numAttrs = after ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

/* `bytes` (a multiple of 16, both addresses 16-byte aligned) from global to
 * this CTA's shared memory, counted on bar. */
__device__ __forceinline__ void kmb_bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     kmb_smem(dst)),
                 "l"(src), "r"(bytes), "r"(kmb_smem(bar))
                 : "memory");
}
