// The bounded waits on mbarriers of a CTA whose roles give up together.  A whole warp calls them, converged, and the
// verdict is the warp's: what follows a wait is warp-collective (TMEM accesses, elections, votes, shuffles), so no lane may
// leave while its neighbours go on.  A lane whose test has passed passes it again: a barrier's next phase needs the
// arrivals of the warps that wait for this one.
// Included by tcgen05.cuh, behind mbar_test_wait; nothing here needs more than the names below, so that the votes can be
// tried on the host: mbar_test_wait, mbar_try_wait_hint, smem_u32, kWaitBudgetCycles, clock64, atomicOr and the votes.
#pragma once

namespace pplb200 {

constexpr uint32_t kWholeWarp = 0xffffffffu;

// Gives up as soon as another warp of the CTA has given up, or the budget is spent.  The common case, a phase that has
// completed already, costs one test and a vote; the polling loop is kept out of line.
static __device__ __noinline__ bool wait_or_abort_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                                       uint32_t* status, uint32_t code) {
    const long long t0 = clock64();
    for (uint32_t i = 0;; i += 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (__all_sync(kWholeWarp, PPLB200_PREFILL_WAIT(bar, parity))) {
                return true;
            }
        }
        if ((i & 255u) == 252u) {
            if (__any_sync(kWholeWarp, *abort_flag != 0)) {
                return false;
            }
            if (__any_sync(kWholeWarp, clock64() - t0 > kWaitBudgetCycles)) {
                break;
            }
        }
    }
    *abort_flag = 1;
    atomicOr(status, code);
    return false;
}
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                              uint32_t* status, uint32_t code) {
    if (__all_sync(kWholeWarp, PPLB200_PREFILL_WAIT(bar, parity))) {
        return true;
    }
    return wait_or_abort_slow(bar, parity, abort_flag, status, code);
}

// The same for a warp that is in no hurry: parked by the hardware instead of polling, so that it leaves the issue slots
// to the others.
__device__ __forceinline__ bool wait_or_abort_parked(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                                     uint32_t* status, uint32_t code) {
    const uint32_t addr = smem_u32(bar);
    if (__all_sync(kWholeWarp, mbar_try_wait_hint(addr, parity, PPLB200_WAIT_HINT_NS))) {
        return true;
    }
    const long long t0 = clock64();
    while (!__all_sync(kWholeWarp, mbar_try_wait_hint(addr, parity, PPLB200_WAIT_HINT_NS))) {
        if (__any_sync(kWholeWarp, *abort_flag != 0)) {
            return false;
        }
        if (__any_sync(kWholeWarp, clock64() - t0 > kWaitBudgetCycles)) {
            *abort_flag = 1;
            atomicOr(status, code);
            return false;
        }
    }
    return true;
}

}  // namespace pplb200
