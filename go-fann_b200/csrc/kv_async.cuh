// kv_async.cuh — mbarriers and bulk copies of the cache operators.  Every
// wait is bounded: a kernel whose wait runs out sets the status word to
// GOFANN_ERR_TIMEOUT and ends.
#pragma once

#include "kv_common.cuh"

namespace gofann {

__device__ __forceinline__ uint32_t shared_addr(const void* p)
{
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_fence()
{
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Waits for the phase of `parity`; false when the limit of some 2 s ran out.
constexpr long long kWaitCycles = 4ll << 30;
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity)
{
    if (barrier_try(bar, parity)) return true;
    const long long start = clock64();
    while (!barrier_try(bar, parity))
        if (clock64() - start > kWaitCycles) return false;
    return true;
}
// Contiguous global -> shared copy; both addresses and the size multiples of 16.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// Programmatic launches: the next kernel of the stream may start, and wait
// for the work of the one before.  Every thread of a kernel launched that way
// waits before it returns, one with nothing to do too: what follows in the
// stream is ordered behind that kernel only, so it must not end first.  What
// the kernel before wrote is read with __ldcg: neither the read-only path nor a
// line that its blocks left in this SM's L1 may serve it.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void kv_timeout(const gofann_kv_batch& b)
{
    if (b.status) atomicExch(b.status, GOFANN_ERR_TIMEOUT);
}

}  // namespace gofann
