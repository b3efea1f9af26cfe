"""The bounded waits of the tensor-core kernels (csrc/warp_wait.cuh), tried on the host: 32 threads are the lanes of a warp,
and a script says when each lane's test of the barrier passes, when another warp gives up, and how fast its clock runs."""
import shutil
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parent.parent / "ppl.nn_b200" / "csrc" / "warp_wait.cuh"

HARNESS = r"""
#include <atomic>
#include <barrier>
#include <cstdint>
#include <cstdio>
#include <thread>
#include <vector>
#define __device__
#define __noinline__
#define __forceinline__ inline
#define PPLB200_PREFILL_WAIT mbar_test_wait
#define PPLB200_WAIT_HINT_NS 1

struct Script { int pass_at[32]; int abort_at; int abort_lane; long long tick[32]; };
static Script script;
static thread_local int lane, polls;
static thread_local long long now;
static volatile int abort_word;
static uint32_t status_word;
static std::barrier<> meet(32);
static std::atomic<int> votes[2];

namespace pplb200 {
constexpr long long kWaitBudgetCycles = 100000;
inline bool poll() {
    const int n = polls++;
    if (n == script.abort_at && lane == script.abort_lane) abort_word = 1;
    return n >= script.pass_at[lane];
}
inline bool mbar_test_wait(uint64_t*, uint32_t) { return poll(); }
inline bool mbar_try_wait_hint(uint32_t, uint32_t, uint32_t) { return poll(); }
inline uint32_t smem_u32(const void*) { return 0; }
inline long long clock64() { return now += script.tick[lane]; }
inline uint32_t atomicOr(uint32_t* p, uint32_t v) { return __atomic_fetch_or(p, v, __ATOMIC_SEQ_CST); }
inline int count_true(bool p) {
    static thread_local int turn = 0;
    const int t = turn++ & 1;
    if (p) votes[t].fetch_add(1);
    meet.arrive_and_wait();
    const int n = votes[t].load();
    meet.arrive_and_wait();
    if (lane == 0) votes[t].store(0);
    return n;
}
inline bool __all_sync(uint32_t, bool p) { return count_true(p) == 32; }
inline bool __any_sync(uint32_t, bool p) { return count_true(p) > 0; }
}
#include "WAITS"

int main(int argc, char** argv) {
    // case, parked
    const int which = argv[1][0] - '0';
    const bool parked = argv[2][0] == '1';
    for (int l = 0; l < 32; ++l) { script.pass_at[l] = 1 << 30; script.tick[l] = 1; }
    script.abort_at = -1;
    script.abort_lane = 0;
    if (which == 0) for (int l = 0; l < 32; ++l) script.pass_at[l] = 7 * l;              // late, one after the other
    if (which == 1) { script.pass_at[5] = 0; script.abort_at = 300; }                    // one passes, another warp gives up
    if (which == 2) { for (int l = 0; l < 32; ++l) script.pass_at[l] = l < 16 ? 3 : 400; script.abort_at = 100; script.abort_lane = 20; }
    if (which == 3) { script.pass_at[9] = 0; script.tick[3] = 60000; }                    // one lane's clock is ahead
    if (which == 4) for (int l = 0; l < 32; ++l) script.pass_at[l] = 0;                   // complete already
    bool result[32];
    uint64_t bar = 0;
    std::vector<std::thread> lanes;
    for (int l = 0; l < 32; ++l) {
        lanes.emplace_back([&, l] {
            lane = l;
            result[l] = parked ? pplb200::wait_or_abort_parked(&bar, 0, &abort_word, &status_word, 2)
                               : pplb200::wait_or_abort(&bar, 0, &abort_word, &status_word, 2);
        });
    }
    for (auto& t : lanes) t.join();
    int passed = 0;
    for (bool r : result) passed += r;
    printf("%d %d %u\n", passed, static_cast<int>(abort_word), status_word);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    folder = tmp_path_factory.mktemp("warp_wait")
    (folder / "main.cc").write_text(HARNESS.replace("WAITS", str(HEADER)))
    subprocess.run([gxx, "-std=c++20", "-O1", "-pthread", "-Wno-unknown-pragmas", "-o", str(folder / "main"), str(folder / "main.cc")],
                   check=True)
    return folder / "main"


@pytest.mark.parametrize("parked", [0, 1])
@pytest.mark.parametrize("case,expect", [
    (0, "32 0 0"),  # every lane sees the phase complete, late ones later
    (1, "0 1 0"),   # one lane's test has passed when another warp gives up: the warp gives up, and reports nothing more
    (2, "0 1 0"),   # so it does where half of the lanes have passed
    (3, "0 1 2"),   # the budget of one lane is spent: the warp gives up, raises the flag and reports
    (4, "32 0 0"),
])
def test_a_warp_goes_on_or_gives_up_as_one(program, case, expect, parked):
    out = subprocess.run([str(program), str(case), str(parked)], check=True, capture_output=True, text=True, timeout=60)
    assert out.stdout.strip() == expect
