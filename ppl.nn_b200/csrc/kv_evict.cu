// Eviction from the KV cache: the choice of the positions to keep, and the in-place compaction of their rows.
//
// Select.  For one (sequence, kv head) with n cached positions and a budget of k, the last r = min(recent, k)
// positions stay, then the first s = min(sink, k - r), and of the positions [s, n - r) the k - r - s of highest
// accumulated weight, ties going to the lowest position.  The order of fp32 weights is the order of a 32-bit key
// (order_key below).  One CTA per list, and one read of the weights:
//   1. A sample of 4096 keys brackets the key of the last candidate taken: [low, high] around the sample's quantile,
//      four standard deviations wide on either side.  (Up to kListCap candidates need no sample: all go to the list.)
//   2. Every weight is read once.  A key above the bracket sets its position's bit in a mask in shared memory, a key
//      inside it joins a list in shared memory.
//   3. A radix descent over that list (four rounds of 8 bits) gives the exact key of the last one taken; the list's
//      keys above it set their bits, the equal ones theirs in a second mask.
//   4. The masks are walked in order of position: bits of the first mask, and the first so many of the second.
// Should the bracket miss (too many keys above, or too few down to its end) or the list overflow (many equal weights),
// the radix descent runs over the weights themselves, and so it does for lists too long for the masks.
// Measured: 128 lists of 32768 to 131072 positions, 4096 kept: 40 us (49 us a call), of which the longest list takes 7 us
// for the sample, 21 for the scan, 5 for the descent and 3 for the output.  A read of the weights alone would take 7 us:
// a list is one CTA's, because its mask and list fill an SM's shared memory, and 128 CTAs of unequal length fill the chip
// 60 %.
//
// Compact.  Row base + kept[i] moves to row base + i.  kept is strictly ascending, so kept[i] >= i; an entry below its
// index, outside its sequence or not above every such entry before it is skipped, so that the rows that do move are
// strictly ascending in any list.  A list is cut into
// segments; a segment reads all its sources before it writes.  Its destinations may still be the sources of EARLIER
// segments (kept[i'] = i with i' < i), never of later ones, so a segment raises a flag once it has read, and before it
// writes waits for the flags of those earlier segments whose sources lie among its destinations -- few, and long done
// where many positions were dropped.  A list ends at its first negative entry, whatever follows.  A kernel of its own looks
// at all the entries (a twentieth of the bytes) and leaves that end, and for each segment the entries that move and the
// earlier segments to wait for.  The highest positions that move before each segment do not fall, whatever the list holds,
// so those are found by bisection.  Persistent CTAs draw their segments from a counter in an order in which a list's
// earlier segments come first.  Nobody waits before it has raised the flags of the segments it has begun, so the lowest
// flag not yet up always belongs to a CTA that can go on.
// Measured: 16 sequences of up to 16384 positions, 2048 kept per kv head, weights too (176 MB): 47 us behind 6 for the
// lists, 55 a call (3.2 TB/s); 4 of up to 131072, paged, 16001 kept (347 MB): 100 behind 9, 112 a call (3.1 TB/s); the
// accepted paths of 32 sequences in 32 layers (26 MB): 7 us behind 4, 19 a call.  DRAM is 43 to 46 % busy, about the bytes
// that have to move; the first stall is the barrier: a CTA begins no copy of its next segment before the stores of this
// one are on their way.
#include <type_traits>

#include "common.cuh"
#include "launch.h"

namespace pplb200 {

namespace {

// Threads of a CTA: 1024 for long lists, one CTA per SM; for lists of up to kShortList positions, which come in large
// numbers, four times as many CTAs of a quarter of the threads.
constexpr int kSelectThreads = 1024;
constexpr int kShortThreads = 256;
constexpr int kShortList = 2048;
constexpr int kListCap = 12288;    // keys inside the bracket
constexpr int kSample = 4096;
constexpr int kMaskWords = 8192;   // 262144 positions
constexpr int kAhead = 8;          // weights per thread of a stage, of which two are on their way

// Unsigned key with the order of the weights: -0 counts as +0, NaN as the lowest.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (!(w == w)) {
        return 0u;
    }
    const uint32_t u = __float_as_uint(w + 0.0f);  // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The weight of a key (of a number, not of the NaN key 0)
__device__ __forceinline__ float key_weight(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

struct SelectArgs {
    const float* weight;  // [L, Hkv, MaxT], indexed by cache row
    const int64_t* cachestarts;
    const int64_t* kvlens;
    const int64_t* budgets;
    int64_t* kept;  // [batch, Hkv, max_budget]
    uint32_t* status;
    CacheGeom geom;
    int64_t sink, recent, max_budget, max_kvlen, max_tokens;
    int32_t num_kv_heads;
    int32_t mask_words;  // 32-bit words of a mask, and keys of the list: the shared memory the launch asked for
    int32_t list_cap;
};

struct SelectShared {
    uint32_t hist[256];
    uint32_t warp_sum[32];
    uint32_t digit, left, listed, above;
};

// The key of rank `rank` (1: the highest) among the keys that for_each(f) passes to f, and how many of that key belong
// to the `rank` highest.  Four rounds: a histogram of the next 8 bits of the keys that share the digits found so far.
template <typename ForEach>
__device__ __forceinline__ uint32_t radix_rank(SelectShared& sh, uint32_t rank, uint32_t& equal, ForEach for_each) {
    const int tid = threadIdx.x, lane = tid & 31;
    uint32_t prefix = 0, left = rank;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) {
            sh.hist[tid] = 0;
        }
        __syncthreads();
        for_each([&](uint32_t key) {
            if (shift == 24 || (key >> (shift + 8)) == prefix) {
                atomicAdd(&sh.hist[(key >> shift) & 255u], 1u);
            }
        });
        __syncthreads();
        if (tid < 32) {
            // lane l holds digits 255 - 8 l .. 248 - 8 l, from the highest down
            uint32_t c[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                c[i] = sh.hist[255 - 8 * lane - i];
                sum += c[i];
            }
            uint32_t before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
                before += lane >= o ? x : 0u;
            }
            before -= sum;  // keys with a higher digit than this lane's
            if (before < left && left <= before + sum) {
                uint32_t d = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (before < left) {
                        d = 255 - 8 * lane - i;
                        sh.left = left - before;
                    }
                    before += c[i];
                }
                sh.digit = d;
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | sh.digit;
        left = sh.left;
    }
    equal = left;
    return prefix;
}

// Exclusive sum over the CTA's warps of a warp-uniform value; `total` is the sum over all of them.
__device__ __forceinline__ uint32_t sum_before(SelectShared& sh, uint32_t v, uint32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) {
        sh.warp_sum[warp] = v;
    }
    __syncthreads();
    const uint32_t x = lane < static_cast<int>(blockDim.x >> 5) ? sh.warp_sum[lane] : 0u;
    uint32_t incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
        incl += lane >= o ? y : 0u;
    }
    total = __shfl_sync(0xffffffffu, incl, 31);
    return __shfl_sync(0xffffffffu, incl - x, warp);
}

__device__ __forceinline__ uint32_t warp_total(uint32_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

template <int NT>
__global__ void __launch_bounds__(NT) kv_evict_select_kernel(const SelectArgs a) {
    __shared__ SelectShared sh;
    extern __shared__ __align__(16) uint32_t dyn[];
    uint32_t* mask = dyn;                      // kept for sure
    uint32_t* tie = mask + a.mask_words;       // has the key of the last one taken
    uint32_t* list_key = tie + a.mask_words;
    int32_t* list_pos = reinterpret_cast<int32_t*>(list_key + a.list_cap);
    float* ring = reinterpret_cast<float*>(list_pos + a.list_cap);  // [2][kAhead][NT]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t b = blockIdx.y;
    const int head = blockIdx.x;
    int64_t n64 = a.kvlens[b], k64 = a.budgets[b];
    if (n64 > a.max_kvlen || n64 < 0) {
        if (tid == 0) {
            atomicOr(a.status, kDevLengthClamped);
        }
        n64 = n64 < 0 ? 0 : a.max_kvlen;
    }
    k64 = k64 > a.max_budget ? a.max_budget : k64;
    k64 = k64 > n64 ? n64 : (k64 < 0 ? 0 : k64);
    const int64_t r = a.recent < k64 ? a.recent : k64;
    const int64_t s = a.sink < k64 - r ? a.sink : k64 - r;
    const int32_t n = static_cast<int32_t>(n64), k = static_cast<int32_t>(k64);
    const int32_t lo = static_cast<int32_t>(s), hi = static_cast<int32_t>(n64 - r);  // candidates [lo, hi)
    const uint32_t want = static_cast<uint32_t>(k64 - r - s), have = static_cast<uint32_t>(hi - lo);
    const float* w = a.weight + (a.geom.layer_idx * a.num_kv_heads + head) * a.max_tokens;
    int64_t* out = a.kept + (b * a.num_kv_heads + head) * a.max_budget;

    const int64_t first_row = a.geom.cache_mode == 0 ? a.cachestarts[b] : 0;
    auto row_at = [&](int32_t pos) -> int64_t {
        if (a.geom.cache_mode != 0) {
            return cache_row(a.geom, a.cachestarts, b, pos);
        }
        return first_row < 0 ? -1 : first_row + pos;
    };
    auto key_at = [&](int32_t pos) -> uint32_t {
        const int64_t row = row_at(pos);
        if (!cache_row_ok(row, a.max_tokens)) {
            atomicOr(a.status, kDevRowOutOfRange);
            return 0u;
        }
        return order_key(__ldg(w + row));
    };
    auto all_keys = [&](auto f) {
        for (int32_t pos = lo + tid; pos < hi; pos += NT) {
            f(key_at(pos));
        }
    };

    // cut: the key of the last candidate taken; equal: how many candidates with that key are taken
    const bool choose = want > 0 && want < have;
    uint32_t cut = 0, equal = 0;
    const int32_t words = (n + 31) / 32;
    const bool fits = words <= a.mask_words;
    bool done = !choose;
    if (fits) {
        for (int32_t i = tid; i < words; i += NT) {
            // sinks and recent positions; all of them where there is no choice to make
            const int32_t p0 = i * 32;
            const uint32_t exist = n - p0 >= 32 ? ~0u : (1u << (n - p0)) - 1u;
            const int32_t c0 = lo - p0 < 0 ? 0 : (lo - p0 > 32 ? 32 : lo - p0), c1 = hi - p0 < c0 ? c0 : (hi - p0 > 32 ? 32 : hi - p0);
            const uint32_t from = c0 == 32 ? 0u : ~0u << c0, to = c1 == 32 ? ~0u : (1u << c1) - 1u;  // candidates: both
            const uint32_t m = !choose && want > 0 ? exist : exist & ~(from & to);
            mask[i] = m;
            tie[i] = 0;
        }
    }
    if (choose && fits) {
        uint32_t low = 0, high = 0xffffffffu;
        if (have > static_cast<uint32_t>(a.list_cap)) {
            const double step = static_cast<double>(have) / kSample;
            const float q = static_cast<float>(want) / static_cast<float>(have) * kSample;
            const float wide = 4.0f * sqrtf(q * (1.0f - q / kSample)) + 8.0f;
            uint32_t keys[kSample / NT];
#pragma unroll
            for (int i = 0; i < kSample / NT; ++i) {
                keys[i] = key_at(lo + static_cast<int32_t>((i * NT + tid) * step));
            }
            auto sample = [&](auto f) {
#pragma unroll
                for (int i = 0; i < kSample / NT; ++i) {
                    f(keys[i]);
                }
            };
            uint32_t unused;
            if (q - wide >= 1.0f) {
                high = radix_rank(sh, static_cast<uint32_t>(q - wide), unused, sample);
            }
            if (q + wide < kSample) {
                low = radix_rank(sh, static_cast<uint32_t>(q + wide) + 1u, unused, sample);
            }
        }
        if (tid == 0) {
            sh.listed = 0;
            sh.above = 0;
        }
        __syncthreads();
        // A warp takes 32 consecutive positions at a time; each thread copies its own weights, kAhead a stage, and no
        // one else reads them, so the stages need no barrier.
        const float high_w = high == 0xffffffffu ? INFINITY : key_weight(high);
        const float low_w = low == 0u ? -INFINITY : key_weight(low);
        const bool list_all = low == 0u;
        uint32_t above = 0;
        const int32_t first = (lo & ~31) + tid, step = NT * kAhead;
        const uint32_t mine = smem_u32(ring + tid);
        const bool plain = a.geom.cache_mode == 0 && first_row >= 0 && first_row + hi <= a.max_tokens;
        const float* src = w + first_row;  // used where plain
        auto fetch = [&](int stage, int32_t pos0) {
            if (plain && pos0 - lane >= lo && pos0 - lane + (kAhead - 1) * NT + 32 <= hi) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    cp_async4(mine + static_cast<uint32_t>(stage * kAhead + i) * (NT * 4), src + pos0 + i * NT);
                }
                cp_async_commit();
                return;
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int32_t pos = pos0 + i * NT;
                if (pos >= lo && pos < hi) {
                    const int64_t row = row_at(pos);
                    const uint32_t at = mine + static_cast<uint32_t>(stage * kAhead + i) * (NT * 4);
                    if (cache_row_ok(row, a.max_tokens)) {
                        cp_async4(at, w + row);
                    } else {
                        atomicOr(a.status, kDevRowOutOfRange);
                        ring[(stage * kAhead + i) * NT + tid] = __uint_as_float(0x7fffffffu);  // counts as a NaN
                    }
                }
            }
            cp_async_commit();
        };
        // The list's order does not matter: a lane with keys for it takes their places by itself.  ALL: every position
        // of the stage is a candidate.
        auto scan = [&](auto all, int stage, int32_t pos0) {
            constexpr bool ALL = decltype(all)::value;
            const float* mine_now = ring + stage * kAhead * NT + tid;
            uint32_t in_list = 0, my_up = 0;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int32_t pos = pos0 + i * NT;
                const bool in = ALL || (pos >= lo && pos < hi);
                const float x = in ? mine_now[i * NT] : 0.0f;
                const bool up_here = in && x > high_w;
                const uint32_t up = __ballot_sync(0xffffffffu, up_here);
                my_up = lane == i ? up : my_up;
                if (in && !up_here && (list_all || x >= low_w)) {
                    in_list |= 1u << i;
                }
            }
            if (my_up != 0u) {  // lanes 0 .. kAhead - 1 hold a word each; this warp alone owns them
                mask[(pos0 >> 5) + lane * (NT / 32)] |= my_up;
                above += __popc(my_up);
            }
            if (in_list != 0u) {
                uint32_t slot = atomicAdd(&sh.listed, __popc(in_list));
                for (; in_list != 0u && slot < static_cast<uint32_t>(a.list_cap); in_list &= in_list - 1u, ++slot) {
                    const int i = __ffs(in_list) - 1;
                    list_key[slot] = order_key(mine_now[i * NT]);
                    list_pos[slot] = pos0 + i * NT;
                }
            }
            __syncwarp();
        };
        fetch(0, first);
        int stage = 0;
        for (int32_t pos0 = first; pos0 - lane < hi; pos0 += step, stage ^= 1) {
            fetch(stage ^ 1, pos0 + step);
            cp_async_wait<1>();
            if (pos0 - lane >= lo && pos0 - lane + (kAhead - 1) * NT + 32 <= hi) {
                scan(std::true_type{}, stage, pos0);
            } else {
                scan(std::false_type{}, stage, pos0);
            }
        }
        cp_async_wait<0>();
        above = warp_total(above);
        if (lane == 0) {
            atomicAdd(&sh.above, above);
        }
        __syncthreads();
        above = sh.above;
        const uint32_t listed = sh.listed;
        done = listed <= static_cast<uint32_t>(a.list_cap) && above < want && want <= above + listed;
        if (done) {
            cut = radix_rank(sh, want - above, equal, [&](auto f) {
                for (uint32_t i = tid; i < listed; i += NT) {
                    f(list_key[i]);
                }
            });
            for (uint32_t i = tid; i < listed; i += NT) {
                if (list_key[i] >= cut) {
                    uint32_t* m = list_key[i] > cut ? mask : tie;
                    atomicOr(&m[list_pos[i] >> 5], 1u << (list_pos[i] & 31));
                }
            }
        }
    }
    if (!done) {
        cut = radix_rank(sh, want, equal, all_keys);
        if (fits) {
            __syncthreads();
            for (int32_t base = (lo & ~31) + warp * 32; base < hi; base += NT) {
                const int32_t pos = base + lane;
                const bool in = pos >= lo && pos < hi;
                const uint32_t key = in ? key_at(pos) : 0u;
                const uint32_t up = __ballot_sync(0xffffffffu, in && key > cut);
                const uint32_t mid = __ballot_sync(0xffffffffu, in && key == cut);
                const uint32_t forced = __ballot_sync(0xffffffffu, !in && pos < n);
                if (lane == 0) {
                    mask[pos >> 5] = forced | up;
                    tie[pos >> 5] = mid;
                }
            }
        }
    }
    __syncthreads();

    // kept positions in ascending order: a warp takes a run of words, after the counts of the runs before it
    const int32_t total_words = fits ? words : (n + 31) / 32;
    const int32_t run = (total_words + (NT / 32) - 1) / (NT / 32);
    const int32_t w0 = warp * run, w1 = w0 + run < total_words ? w0 + run : total_words;
    auto word_at = [&](int32_t i, uint32_t& ties) -> uint32_t {  // the words of 32 positions; all lanes call it
        if (fits) {
            ties = tie[i];
            return mask[i];
        }
        const int32_t pos = i * 32 + lane;
        const bool forced = pos < n && (pos < lo || pos >= hi || (!choose && want > 0));
        const uint32_t key = choose && pos >= lo && pos < hi ? key_at(pos) : 0u;
        ties = __ballot_sync(0xffffffffu, choose && pos >= lo && pos < hi && key == cut);
        return __ballot_sync(0xffffffffu, forced || (choose && pos >= lo && pos < hi && key > cut));
    };
    uint32_t sure = 0, ties = 0;
    if (fits) {
        for (int32_t i = w0 + lane; i < w1; i += 32) {
            sure += __popc(mask[i]);
            ties += __popc(tie[i]);
        }
        sure = warp_total(sure);
        ties = warp_total(ties);
    } else {
        for (int32_t i = w0; i < w1; ++i) {
            uint32_t t;
            sure += __popc(word_at(i, t));
            ties += __popc(t);
        }
    }
    uint32_t total;
    uint32_t ties_before = sum_before(sh, ties, total);
    const uint32_t ties_taken = ties_before >= equal ? 0u : (equal - ties_before < ties ? equal - ties_before : ties);
    uint32_t rank = sum_before(sh, sure + ties_taken, total);
    // the word of the positions kept among 32: the sure ones and the first of the ties, up to `equal` in the list
    auto with_ties = [&](uint32_t m, uint32_t t) -> uint32_t {
        while (t != 0u && ties_before < equal) {
            m |= t & (0u - t);
            t &= t - 1u;
            ++ties_before;
        }
        return m;
    };
    if (fits && k < n / 8) {
        // few bits a word: a lane takes a word and writes its positions one after the other
        for (int32_t i0 = w0; i0 < w1; i0 += 32) {
            const int32_t i = i0 + lane;
            uint32_t m = i < w1 ? mask[i] : 0u;
            const uint32_t t = i < w1 ? tie[i] : 0u;
            if (__any_sync(0xffffffffu, t != 0u)) {
                uint32_t incl = __popc(t);
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
                    incl += lane >= o ? y : 0u;
                }
                const uint32_t all = __shfl_sync(0xffffffffu, incl, 31), before = ties_before;
                ties_before = before + incl - __popc(t);
                m = with_ties(m, t);
                ties_before = before + all;
            }
            uint32_t incl = __popc(m);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
                incl += lane >= o ? y : 0u;
            }
            uint32_t at = rank + incl - __popc(m);
            rank += __shfl_sync(0xffffffffu, incl, 31);
            while (m != 0u) {
                if (at < static_cast<uint32_t>(k)) {
                    out[at] = i * 32 + __ffs(m) - 1;
                }
                m &= m - 1u;
                ++at;
            }
        }
    } else {
        for (int32_t i = w0; i < w1; ++i) {
            uint32_t t;
            uint32_t m = word_at(i, t);
            m = with_ties(m, t);
            const uint32_t at = rank + __popc(m & ((1u << lane) - 1u));
            if (((m >> lane) & 1u) != 0u && at < static_cast<uint32_t>(k)) {
                out[at] = i * 32 + lane;
            }
            rank += __popc(m);
        }
    }
    for (int64_t i = k + tid; i < a.max_budget; i += NT) {
        out[i] = -1;
    }
}

// ---- compaction ----------------------------------------------------------------------------------

// What the entries of a segment amount to
struct __align__(16) SegmentPlan {
    int32_t wait_from, wait_to;  // earlier segments whose sources may be among the destinations
    uint32_t moves[2];           // bit i: entry i counts
};

struct CompactArgs {
    const int64_t* kept;  // [batch, kept_heads, max_kept]
    const int64_t* base;
    const int64_t* kvlens;
    const int64_t* cachestarts;
    int8_t* cache;
    __half* scale;
    float* weight;  // [L, Hkv, MaxT] or null
    uint32_t* status;
    uint32_t* ticket;
    int2* ends;       // [batch, kept_heads]: the entries of a kept list, and whether all of them move (or stay)
    SegmentPlan* plans;  // [batch, kept_heads][segments]
    int32_t* tops;    // [batch, kept_heads][segments]: the highest of the positions that move before a segment, or -1
    uint32_t* flags;  // [segments][lists]
    CacheGeom geom;
    int64_t max_kept, max_kvlen, max_tokens;
    int64_t flag_words;
    uint32_t lists;       // batch * layers * head groups
    uint32_t move_tasks;  // segments * lists
    uint32_t tasks;       // and the clearing of weights
    int32_t kept_lists, kept_heads, num_kv_heads;
    uint32_t layers, head_groups;
    int32_t heads_shift, rows_per_seg, segments;  // 1 << heads_shift heads per CTA
};

constexpr int kScanThreads = 1024;
constexpr int kCompactThreads = 256;
constexpr int kCompactCtas = 8;       // per SM: 160 KB on their way
constexpr int kSegmentRows = 64;      // rows x heads of a segment
constexpr int kClearRows = 8192;      // weights zeroed by a CTA

// A flag orders a segment's reads before other CTAs' writes.  When it is raised the sources have arrived in shared memory
// (the asynchronous copies have completed and the CTA has met at a barrier); the release hands that on, and whoever
// acquires the flag meets at a barrier of its own before anyone there writes.  Measured against relaxed accesses, which
// leave the order to the machine: 55 against 58 us and 112 against 115 us (the calls of the header).
__device__ __forceinline__ void raise_flag(uint32_t* flag) {
    asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(flag), "r"(1u) : "memory");
}
__device__ __forceinline__ bool wait_flag(const uint32_t* flag) {
    long long t0 = 0;
    for (;;) {
        uint32_t v;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
        if (v != 0u) {
            return true;
        }
        const long long t = clock64();
        t0 = t0 == 0 ? t : t0;
        if (t - t0 > kWaitBudgetCycles) {
            return false;
        }
    }
}

// Entry i of a list; -1 where it leaves the sequence or would move up.  Of the entries in range those above all before them
// count, so the highest that counts before i is the highest in range before i.
__device__ __forceinline__ int32_t in_range(int64_t p, int64_t i, int64_t base, int64_t n) {
    return base >= 0 && p >= i && p < n - base ? static_cast<int32_t>(p) : -1;
}

__device__ __forceinline__ int32_t warp_max_scan(int32_t x, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t other = __shfl_up_sync(0xffffffffu, x, o);
        x = lane >= o && other > x ? other : x;
    }
    return x;
}

// How many of tops[0 .. count) are below `pos`; tops do not fall.
__device__ __forceinline__ int32_t count_below(const int32_t* tops, int32_t count, int64_t pos) {
    int32_t lo = 0, hi = count;
    while (lo < hi) {
        const int32_t mid = (lo + hi) >> 1;
        if (tops[mid] < pos) {
            lo = mid + 1;
        } else {
            hi = mid;
        }
    }
    return lo;
}

// A CTA per kept list: where it ends, and the plans of its segments.  Behind the first negative entry there may be
// anything, and a list may be out of order, so the entries up to there are looked at one and all: a bisection would have
// to trust them.  (What stands behind the end enters the maxima of segments that have nothing to move.)  Clears the status word,
// the ticket and the flags on the way, so that the call needs no other launch before the moving one.
__global__ void __launch_bounds__(kScanThreads) kv_compact_scan_kernel(const CompactArgs a) {
    __shared__ int32_t s_end, s_bad, warp_top[kScanThreads / 32], seg_top[kScanThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_launch_dependents();
    if (tid == 0) {
        s_end = static_cast<int32_t>(a.max_kept);
        s_bad = s_end;  // the first entry that does not count
    }
    __syncthreads();
    grid_dependency_wait();  // the workspace may still be in use, and the list still be written
    const int64_t id = blockIdx.x * static_cast<int64_t>(kScanThreads) + tid;
    if (id < 2) {
        a.status[id] = 0;  // and the ticket behind it
    }
    for (int64_t i = id; i < a.flag_words; i += gridDim.x * static_cast<int64_t>(kScanThreads)) {
        a.flags[i] = 0;
    }
    const int64_t* kept = a.kept + blockIdx.x * a.max_kept;
    int32_t* tops = a.segments <= kScanThreads ? seg_top : a.tops + blockIdx.x * static_cast<int64_t>(a.segments);
    const int64_t b = blockIdx.x / a.kept_heads, base = a.base[b];
    const int rows = a.rows_per_seg, shift = 31 - __clz(rows);  // 8, 16, 32 or 64
    int64_t n = a.kvlens[b];
    n = n > a.max_kvlen ? a.max_kvlen : n;
    constexpr int kUnroll = 8;  // entries of a thread whose loads go out together; a warp's 256 are neighbours
    bool ended = false;
    for (int64_t step = 0; step < a.max_kept && !ended; step += kUnroll * kScanThreads) {
        const int64_t i0 = step + warp * (32 * kUnroll) + lane;
        int64_t p[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            p[u] = i0 + u * 32 < a.max_kept ? kept[i0 + u * 32] : 0;
        }
        int32_t top[kUnroll];
        int32_t last = i0 > lane && lane == 0 ? in_range(kept[i0 - 1], i0 - 1, base, n) : -1;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int64_t i = i0 + u * 32;
            top[u] = i < a.max_kept ? in_range(p[u], i, base, n) : -1;
            const int32_t left = __shfl_up_sync(0xffffffffu, top[u], 1);
            if (i < a.max_kept) {
                if (p[u] < 0) {
                    ended = true;
                    atomicMin(&s_end, static_cast<int32_t>(i));
                } else if (top[u] <= (lane > 0 ? left : last)) {  // as long as all count, the one before is the highest
                    atomicMin(&s_bad, static_cast<int32_t>(i));
                }
            }
            last = __shfl_sync(0xffffffffu, top[u], 31);
        }
        if (rows >= 32) {  // one step of the warp, or two
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                top[u] = __reduce_max_sync(0xffffffffu, top[u]);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int64_t i = i0 + u * 32;
                if (lane == 0 && i < a.max_kept && (rows == 32 || (u & 1) == 0)) {
                    tops[i >> shift] = rows == 32 || top[u] > top[u | 1] ? top[u] : top[u | 1];
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) {
                    const int32_t other = __shfl_xor_sync(0xffffffffu, top[u], o);
                    top[u] = o < rows && other > top[u] ? other : top[u];
                }
                if ((lane & (rows - 1)) == 0 && i0 + u * 32 < a.max_kept) {
                    tops[(i0 + u * 32) >> shift] = top[u];
                }
            }
        }
        ended = __syncthreads_or(ended);
    }
    const int32_t end = s_end, used = (end + rows - 1) >> shift;  // segments with entries
    const bool orderly = s_bad >= end;
    if (tid == 0) {
        a.ends[blockIdx.x] = make_int2(end, orderly);
    }
    // each segment's own maximum -> the maximum of those before it
    int32_t carry = -1;
    for (int32_t e0 = 0; e0 < used; e0 += kScanThreads) {
        const int32_t e = e0 + tid;
        const int32_t top = warp_max_scan(e < used ? tops[e] : -1, lane);
        __syncthreads();
        if (lane == 31) {
            warp_top[warp] = top;
        }
        __syncthreads();
        const int32_t all = warp_max_scan(warp_top[lane], lane);
        int32_t before = __shfl_sync(0xffffffffu, all, warp > 0 ? warp - 1 : 0);  // of the warps before
        before = warp > 0 && before > carry ? before : carry;
        const int32_t mine = __shfl_up_sync(0xffffffffu, top, 1);
        if (e < used) {
            tops[e] = lane > 0 && mine > before ? mine : before;
        }
        const int32_t most = __shfl_sync(0xffffffffu, all, 31);
        carry = most > carry ? most : carry;
    }
    __syncthreads();
    // What counts in segment e lies above tops[e], up to tops[e + 1].  So of the segments before e it has to wait for those
    // from the first whose highest reaches its destinations to the last that begins below their end.
    SegmentPlan* plans = a.plans + blockIdx.x * static_cast<int64_t>(a.segments);
    for (int32_t e = tid; e < a.segments; e += kScanThreads) {
        const int64_t first = static_cast<int64_t>(e) * rows;
        SegmentPlan plan = {0, -1, {0u, 0u}};  // behind the end: nothing to move, nothing to wait for
        if (first < end) {
            plan.wait_from = count_below(tops + 1, e, first);
            plan.wait_to = count_below(tops, e, first + rows - 1) - 1;
            const int32_t count = end - first < rows ? static_cast<int32_t>(end - first) : rows;
            plan.moves[0] = count >= 32 ? ~0u : (1u << count) - 1u;
            plan.moves[1] = count <= 32 ? 0u : (count == 64 ? ~0u : (1u << (count - 32)) - 1u);
        }
        plans[e] = plan;
    }
    if (orderly) {
        return;
    }
    __syncthreads();
    for (int32_t e = warp; e < used; e += kScanThreads / 32) {  // a warp per segment
        const int64_t first = static_cast<int64_t>(e) * rows;
        int32_t before = tops[e];
        for (int32_t j = lane; j - lane < rows; j += 32) {
            const int64_t i = first + j;
            const int32_t p = j < rows && i < end ? in_range(kept[i], i, base, n) : -1;
            const int32_t incl = warp_max_scan(p, lane);
            const int32_t left = __shfl_up_sync(0xffffffffu, incl, 1);
            const uint32_t moves = __ballot_sync(0xffffffffu, p > (lane > 0 && left > before ? left : before));
            const int32_t most = __shfl_sync(0xffffffffu, incl, 31);
            before = most > before ? most : before;
            if (lane == 0) {
                plans[e].moves[j >> 5] = moves;
            }
        }
    }
}

// What a task works on
struct Task {
    int64_t b, base, n;   // sequence, its base, the positions it had
    int64_t kept_list;
    int32_t seg, head0;
    int64_t layer_idx;
    uint32_t list;
    bool clear;
};

// Rows of a segment, worked out while the segment before it is on its way
struct SegmentRows {
    int64_t src[kSegmentRows], dst[kSegmentRows];  // element offsets of K of the first head; src < 0: not to be moved
    int2 row[kSegmentRows];                        // cache rows
    int32_t wait_from, wait_to;                    // earlier segments whose sources may be among the destinations
    uint32_t ticket;
};

__device__ __forceinline__ Task task_of(const CompactArgs& a, uint32_t ticket) {
    Task t;
    t.clear = ticket >= a.move_tasks;
    const uint32_t task = t.clear ? ticket - a.move_tasks : ticket;
    t.list = task % a.lists;
    t.seg = task / a.lists;
    t.head0 = static_cast<int>(t.list % a.head_groups) << a.heads_shift;
    t.layer_idx = a.geom.layer_idx + t.list / a.head_groups % a.layers;
    t.b = t.list / a.head_groups / a.layers;
    t.kept_list = t.b * a.kept_heads + (a.kept_heads > 1 ? t.head0 : 0);
    t.base = a.base[t.b];
    t.n = a.kvlens[t.b];
    if (t.n > a.max_kvlen) {
        t.n = a.max_kvlen;
        atomicOr(a.status, kDevLengthClamped);
    }
    return t;
}

// Looks up the rows of the segment that `ticket` names, and its plan.
__device__ __forceinline__ void prepare_segment(const CompactArgs& a, uint32_t ticket, SegmentRows& rows) {
    const int tid = threadIdx.x;
    if (tid >= a.rows_per_seg || ticket >= a.move_tasks) {
        return;
    }
    const Task t = task_of(a, ticket);
    const int64_t i = static_cast<int64_t>(t.seg) * a.rows_per_seg + tid;
    const int4 plan = *reinterpret_cast<const int4*>(a.plans + t.kept_list * a.segments + t.seg);  // a SegmentPlan
    if (tid == 0) {
        rows.wait_from = plan.x;
        rows.wait_to = plan.y;
    }
    const bool counts = ((tid < 32 ? plan.z : plan.w) >> (tid & 31) & 1) != 0;
    const int64_t p = i < a.max_kept ? a.kept[t.kept_list * a.max_kept + i] : 0;  // loaded without waiting for the plan
    CacheGeom geom = a.geom;
    int64_t src = -1, dst = 0;
    if (counts && p != i) {
        src = cache_row(geom, a.cachestarts, t.b, t.base + p);
        dst = cache_row(geom, a.cachestarts, t.b, t.base + i);
        if (!cache_row_ok(src, a.max_tokens) || !cache_row_ok(dst, a.max_tokens)) {
            atomicOr(a.status, kDevRowOutOfRange);
            src = -1;
        }
    }
    const int64_t fixed = t.layer_idx * geom.stride_l + t.head0 * geom.stride_h;
    rows.src[tid] = src < 0 ? -1 : src * geom.stride_s + fixed;
    rows.dst[tid] = dst * geom.stride_s + fixed;
    rows.row[tid] = make_int2(static_cast<int>(src), static_cast<int>(dst));
}

// The positions behind the kept ones hold no token any more: the next ones start from zero weight.
__device__ __forceinline__ bool clear_weights(const CompactArgs& a, uint32_t ticket) {
    const Task t = task_of(a, ticket);
    if (t.base < 0) {
        return true;
    }
    const int64_t from = t.base + a.ends[t.kept_list].x + static_cast<int64_t>(t.seg) * kClearRows;
    const int64_t end = from + kClearRows < t.n ? from + kClearRows : t.n;
    if (from >= end) {
        return true;
    }
    bool ok = true;
    for (int32_t e = threadIdx.x; e < a.segments; e += kCompactThreads) {
        ok = wait_flag(a.flags + static_cast<int64_t>(e) * a.lists + t.list) && ok;
    }
    if (!__syncthreads_and(ok)) {
        return false;
    }
    float* weight = a.weight + (t.layer_idx * a.num_kv_heads + t.head0) * a.max_tokens;
    for (int64_t pos = from + threadIdx.x; pos < end; pos += kCompactThreads) {
        const int64_t row = cache_row(a.geom, a.cachestarts, t.b, pos);
        if (!cache_row_ok(row, a.max_tokens)) {
            atomicOr(a.status, kDevRowOutOfRange);
            continue;
        }
        for (int head = 0; head < 1 << a.heads_shift; ++head) {
            weight[head * a.max_tokens + row] = 0.0f;
        }
    }
    return true;
}

template <int DH>
__global__ void __launch_bounds__(kCompactThreads, kCompactCtas) kv_compact_kernel(const CompactArgs a) {
    constexpr int kCodePieces = DH / 16;   // 16-byte pieces of a row's codes
    constexpr int kScalePieces = DH / 64;  // and of its scales
    constexpr int kCodeStep = kCompactThreads / kCodePieces;  // rows (of K or V of a head) the CTA moves at once
    constexpr int kCodeSteps = 2 * kSegmentRows / kCodeStep;
    __shared__ SegmentRows s_rows[2];
    __shared__ uint4 stage[(kCodeSteps + 1) * kCompactThreads];
    __shared__ float stage_w[kSegmentRows];
    const int tid = threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    if (blockIdx.x == 0) {  // the status word has been cleared: now it can take what the scan found
        for (int32_t l = tid; l < a.kept_lists; l += kCompactThreads) {
            if (a.ends[l].y == 0) {
                atomicOr(a.status, kDevKeptInvalid);
            }
        }
    }
    if (tid == 0) {
        s_rows[0].ticket = atomicAdd(a.ticket, 1u);
    }
    __syncthreads();
    prepare_segment(a, s_rows[0].ticket, s_rows[0]);
    __syncthreads();
    for (int buf = 0;; buf ^= 1) {
        const SegmentRows& rows = s_rows[buf];
        SegmentRows& next = s_rows[buf ^ 1];
        const uint32_t ticket = rows.ticket;
        if (ticket >= a.tasks) {
            return;
        }
        const bool move = ticket < a.move_tasks;
        // x = (row * 2 + K | V) * heads + head, and pieces of it by neighbouring threads: neighbouring bytes.  A thread
        // stages its own pieces in shared memory, which keeps the bytes in flight out of the registers.
        const int shift = a.heads_shift, count = a.rows_per_seg * 2 << shift;
        auto offset = [&](const int64_t* of, int x) -> int64_t {  // of a row of K or V of a head, or negative
            const int y = x >> shift;
            const int64_t row = of[y >> 1];
            return row < 0 ? -1 : row + (y & 1) * a.geom.stride_kv + (x & ((1 << shift) - 1)) * a.geom.stride_h;
        };
        const int cx = tid / kCodePieces, cp = tid % kCodePieces * 16, sx = tid / kScalePieces, sp = tid % kScalePieces * 8;
        if (move) {
#pragma unroll
            for (int u = 0; u < kCodeSteps; ++u) {
                const int x = u * kCodeStep + cx;
                const int64_t off = x < count ? offset(rows.src, x) : -1;
                if (off >= 0) {
                    cp_async16(smem_u32(&stage[u * kCompactThreads + tid]), a.cache + off + cp);
                }
            }
            const int64_t off = sx < count ? offset(rows.src, sx) : -1;
            if (off >= 0) {
                cp_async16(smem_u32(&stage[kCodeSteps * kCompactThreads + tid]), a.scale + (off >> 3) + sp);
            }
        }
        const bool has_weight = move && a.weight != nullptr && tid < a.rows_per_seg << shift && rows.src[tid >> shift] >= 0;
        float* weight = nullptr;
        if (has_weight) {
            const uint32_t list = ticket % a.lists;
            const int64_t head = (static_cast<int64_t>(list % a.head_groups) << shift) + (tid & ((1 << shift) - 1));
            weight = a.weight + ((a.geom.layer_idx + list / a.head_groups % a.layers) * a.num_kv_heads + head) * a.max_tokens;
            cp_async4(smem_u32(&stage_w[tid]), weight + rows.row[tid >> shift].x);
        }
        cp_async_commit();
        // the next task's rows, while the copies are on their way
        if (tid == 0) {
            next.ticket = atomicAdd(a.ticket, 1u);
        }
        __syncthreads();
        prepare_segment(a, next.ticket, next);
        if (!move) {
            if (!clear_weights(a, ticket)) {
                if (tid == 0) {
                    atomicOr(a.status, kDevTmaTimeout);
                }
                return;
            }
            __syncthreads();
            continue;
        }
        cp_async_wait<0>();
        __syncthreads();  // every source of the segment has been read
        const uint32_t list = ticket % a.lists;
        const int32_t seg = ticket / a.lists;
        if (tid == 0) {
            raise_flag(a.flags + static_cast<int64_t>(seg) * a.lists + list);
        }
        bool ok = true;
        for (int32_t e = rows.wait_from + tid; e <= rows.wait_to; e += kCompactThreads) {
            ok = wait_flag(a.flags + static_cast<int64_t>(e) * a.lists + list) && ok;
        }
        if (!__syncthreads_and(ok)) {
            if (tid == 0) {
                atomicOr(a.status, kDevTmaTimeout);
            }
            return;
        }
#pragma unroll
        for (int u = 0; u < kCodeSteps; ++u) {
            const int x = u * kCodeStep + cx;
            if (x < count && rows.src[x >> shift >> 1] >= 0) {
                *reinterpret_cast<uint4*>(a.cache + offset(rows.dst, x) + cp) = stage[u * kCompactThreads + tid];
            }
        }
        if (sx < count && rows.src[sx >> shift >> 1] >= 0) {
            *reinterpret_cast<uint4*>(a.scale + (offset(rows.dst, sx) >> 3) + sp) = stage[kCodeSteps * kCompactThreads + tid];
        }
        if (has_weight) {
            weight[rows.row[tid >> shift].y] = stage_w[tid];
        }
    }
}

}  // namespace

int launch_kv_evict_select(const pplb200_attn_params& p, const CacheGeom& geom, const float* weight,
                           const int64_t* cachestarts, const int64_t* kvlens, const int64_t* budgets, int64_t sink,
                           int64_t recent, int64_t max_budget, uint32_t* status, int64_t* kept, cudaStream_t stream) {
    SelectArgs a = {};
    a.weight = weight;
    a.cachestarts = cachestarts;
    a.kvlens = kvlens;
    a.budgets = budgets;
    a.kept = kept;
    a.status = status;
    a.geom = geom;
    a.sink = sink;
    a.recent = recent;
    a.max_budget = max_budget;
    a.max_kvlen = p.max_kvlen;
    a.max_tokens = p.max_tokens;
    a.num_kv_heads = p.num_kv_heads;
    const int64_t words = (p.max_kvlen + 31) / 32;
    a.mask_words = static_cast<int32_t>(words > kMaskWords ? kMaskWords : words);
    a.list_cap = static_cast<int32_t>(p.max_kvlen > kListCap ? kListCap : p.max_kvlen);
    const dim3 grid(static_cast<unsigned>(p.num_kv_heads), static_cast<unsigned>(p.batch));
    const size_t fixed = 2 * (static_cast<size_t>(a.mask_words) + a.list_cap) * 4;
    const size_t bytes = fixed + 2 * kAhead * kSelectThreads * 4;
    if (p.max_kvlen <= kShortList) {
        // at most 48 KB of dynamic shared memory, what a kernel may have without asking
        static_assert(2 * (kShortList / 32 + kShortList) * 4 + 2 * kAhead * kShortThreads * 4 <= 47104, "short lists");
        kv_evict_select_kernel<kShortThreads><<<grid, kShortThreads, fixed + 2 * kAhead * kShortThreads * 4, stream>>>(a);
        return check_launch("kv_evict_select_kernel");
    }
    // the attribute belongs to the (kernel, device) pair
    static bool attr_set[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
        (void)cudaGetLastError();
        return PPLB200_DEVICE_RUNTIME_ERROR;
    }
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(kv_evict_select_kernel<kSelectThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 2 * (kMaskWords + kListCap) * 4 + 2 * kAhead * kSelectThreads * 4) != cudaSuccess) {
            (void)cudaGetLastError();
            return PPLB200_DEVICE_RUNTIME_ERROR;
        }
        attr_set[dev] = true;
    }
    kv_evict_select_kernel<kSelectThreads><<<grid, kSelectThreads, bytes, stream>>>(a);
    return check_launch("kv_evict_select_kernel");
}

int make_compact_plan(const pplb200_attn_params& p, int64_t kept_heads, int64_t max_kept, int64_t layers,
                      CompactPlan* plan) {
    // One list per kv head: a CTA takes 64 rows of it.  One list for all heads: as many rows times up to 8 heads, whose
    // rows lie next to one another in the token-major layout, and short lists fill a CTA.
    plan->heads_per_cta = 1;
    if (kept_heads == 1) {
        for (int h = 8; h > 1; h >>= 1) {
            if (p.num_kv_heads % h == 0) {
                plan->heads_per_cta = h;
                break;
            }
        }
    }
    plan->rows_per_seg = kSegmentRows / plan->heads_per_cta;
    plan->lists = p.batch * layers * (p.num_kv_heads / plan->heads_per_cta);
    plan->segments = (max_kept + plan->rows_per_seg - 1) / plan->rows_per_seg;
    plan->bytes = 0;
    if (plan->lists > 0x7fffffff) {
        return PPLB200_UNSUPPORTED;
    }
    plan->off_ends = 256;  // behind the status word and the ticket counter
    const uint64_t kept_lists = static_cast<uint64_t>(p.batch) * kept_heads;
    plan->off_tops = plan->off_ends + (kept_lists * 8 + 255) / 256 * 256;
    const bool spills = plan->segments > kScanThreads;  // else the scan has them in shared memory
    plan->off_plans = plan->off_tops + (spills ? (kept_lists * plan->segments * 4 + 255) / 256 * 256 : 0);
    plan->off_flags = plan->off_plans + (kept_lists * plan->segments * sizeof(SegmentPlan) + 255) / 256 * 256;
    plan->bytes = plan->off_flags + (static_cast<uint64_t>(plan->segments) * plan->lists * 4 + 255) / 256 * 256;
    const int64_t clears = (p.max_kvlen + kClearRows - 1) / kClearRows;
    return (plan->segments + clears) * plan->lists > 0x7fffffff ? PPLB200_UNSUPPORTED : PPLB200_SUCCESS;
}

int launch_kv_compact(const pplb200_attn_params& p, const CacheGeom& geom, const CompactPlan& plan, const int64_t* kept,
                      int64_t kept_heads, int64_t max_kept, const int64_t* base, const int64_t* kvlens,
                      const int64_t* cachestarts, int64_t layers, void* cache, void* scale, float* weight,
                      void* workspace, int sm_count, cudaStream_t stream) {
    CompactArgs a = {};
    a.kept = kept;
    a.base = base;
    a.kvlens = kvlens;
    a.cachestarts = cachestarts;
    a.cache = static_cast<int8_t*>(cache);
    a.scale = static_cast<__half*>(scale);
    a.weight = weight;
    a.status = static_cast<uint32_t*>(workspace);
    a.ticket = a.status + 1;
    a.ends = reinterpret_cast<int2*>(static_cast<uint8_t*>(workspace) + plan.off_ends);
    a.tops = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + plan.off_tops);
    a.plans = reinterpret_cast<SegmentPlan*>(static_cast<uint8_t*>(workspace) + plan.off_plans);
    a.flags = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + plan.off_flags);
    a.flag_words = plan.segments * plan.lists;
    a.geom = geom;
    a.max_kept = max_kept;
    a.max_kvlen = p.max_kvlen;
    a.max_tokens = p.max_tokens;
    a.lists = static_cast<uint32_t>(plan.lists);
    a.move_tasks = static_cast<uint32_t>(plan.segments * plan.lists);
    a.kept_lists = static_cast<int32_t>(p.batch * kept_heads);
    a.kept_heads = static_cast<int32_t>(kept_heads);
    a.num_kv_heads = p.num_kv_heads;
    a.layers = static_cast<uint32_t>(layers);
    while (1 << a.heads_shift < plan.heads_per_cta) {
        ++a.heads_shift;
    }
    a.head_groups = p.num_kv_heads / plan.heads_per_cta;
    a.rows_per_seg = plan.rows_per_seg;
    a.segments = static_cast<int32_t>(plan.segments);
    // each kernel starts while the one before it drains, and waits for it before it reads or writes anything
    launch_dependent(kv_compact_scan_kernel, dim3(static_cast<unsigned>(a.kept_lists)), dim3(kScanThreads), 0, stream, a);
    const int rc = check_launch("kv_compact_scan_kernel");
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    const int64_t clears = weight == nullptr ? 0 : (p.max_kvlen + kClearRows - 1) / kClearRows;
    const int64_t tasks = (plan.segments + clears) * plan.lists;
    if (tasks <= 0) {
        return PPLB200_SUCCESS;
    }
    a.tasks = static_cast<uint32_t>(tasks);
    const int64_t resident = static_cast<int64_t>(sm_count) * kCompactCtas;
    const int64_t ctas = tasks < resident ? tasks : resident;
    auto kernel = p.head_dim == 128 ? kv_compact_kernel<128> : kv_compact_kernel<64>;
    launch_dependent(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kCompactThreads), 0, stream, a);
    return check_launch("kv_compact_kernel");
}

}  // namespace pplb200
