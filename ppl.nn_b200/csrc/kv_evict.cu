// Eviction from the KV cache: the choice of the positions to keep, and the in-place compaction of their rows.
//
// Select.  For one (sequence, kv head) with n cached positions and a budget of k, the last r = min(recent, k)
// positions stay, then the first s = min(sink, k - r), and of the positions [s, n - r) the k - r - s of highest
// accumulated weight, ties going to the lowest position.  The order of fp32 weights is the order of a 32-bit
// key (order_key below), so the weight of the last one taken is found exactly by a radix descent: four rounds
// of 8 bits, each a histogram of the keys that share the digits found so far.  A last pass over the positions
// writes the kept ones in ascending order.
//
// Compact.  Row base + kept[i] moves to row base + i.  kept is strictly ascending, so kept[i] >= i, and a list
// can be worked through in place in ascending blocks: a later block's sources lie at or behind its own
// destinations, hence behind every destination of the earlier blocks; only the writes of a block have to wait
// until the sources of that block (and of those before it) have been read.
#include "common.cuh"
#include "launch.h"

namespace pplb200 {

namespace {

constexpr int kSelectThreads = 1024;

// Unsigned key with the order of the weights: -0 counts as +0, NaN as the lowest.
__device__ __forceinline__ uint32_t order_key(float w) {
    if (!(w == w)) {
        return 0u;
    }
    const uint32_t u = __float_as_uint(w + 0.0f);  // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
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
};

__global__ void __launch_bounds__(kSelectThreads) kv_evict_select_kernel(const SelectArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t warp_sum[2][32];
    __shared__ uint32_t s_digit, s_below;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t b = blockIdx.y;
    const int head = blockIdx.x;
    int64_t n = a.kvlens[b], k = a.budgets[b];
    if (n > a.max_kvlen || k > a.max_budget) {
        if (tid == 0) {
            atomicOr(a.status, kDevLengthClamped);
        }
        n = n > a.max_kvlen ? a.max_kvlen : n;
    }
    n = n < 0 ? 0 : n;
    k = k > a.max_budget ? a.max_budget : k;
    k = k > n ? n : (k < 0 ? 0 : k);
    const int64_t r = a.recent < k ? a.recent : k;
    const int64_t s = a.sink < k - r ? a.sink : k - r;
    const int32_t lo = static_cast<int32_t>(s), hi = static_cast<int32_t>(n - r);  // candidates [lo, hi)
    const uint32_t want = static_cast<uint32_t>(k - r - s);
    const float* w = a.weight + (a.geom.layer_idx * a.num_kv_heads + head) * a.max_tokens;
    int64_t* out = a.kept + (b * a.num_kv_heads + head) * a.max_budget;

    auto key_at = [&](int32_t pos) -> uint32_t {
        const int64_t row = cache_row(a.geom, a.cachestarts, b, pos);
        if (!cache_row_ok(row, a.max_tokens)) {
            atomicOr(a.status, kDevRowOutOfRange);
            return 0u;
        }
        return order_key(w[row]);
    };

    // the key of the last candidate taken, and how many candidates with exactly that key are taken
    uint32_t cut = 0, equal_left = want;
    if (want > 0 && static_cast<int64_t>(want) < hi - lo) {
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kSelectThreads) {
                hist[i] = 0;
            }
            __syncthreads();
            for (int32_t pos = lo + tid; pos < hi; pos += kSelectThreads) {
                const uint32_t key = key_at(pos);
                if (shift == 24 || (key >> (shift + 8)) == prefix) {
                    atomicAdd(&hist[(key >> shift) & 255u], 1u);
                }
            }
            __syncthreads();
            if (tid == 0) {  // from the highest digit down
                uint32_t above = 0;
                int d = 255;
                while (d > 0 && above + hist[d] < equal_left) {
                    above += hist[d];
                    --d;
                }
                s_digit = static_cast<uint32_t>(d);
                s_below = equal_left - above;
            }
            __syncthreads();
            prefix = (prefix << 8) | s_digit;
            equal_left = s_below;
        }
        cut = prefix;
    }
    const bool all = static_cast<int64_t>(want) >= hi - lo;

    // kept positions in ascending order
    uint32_t taken = 0, equal_seen = 0;
    for (int32_t base = 0; base < n; base += kSelectThreads) {
        const int32_t pos = base + tid;
        bool forced = false, above = false, equal = false;
        if (pos < n) {
            forced = pos < lo || pos >= hi;
            if (!forced && want > 0) {
                const uint32_t key = all ? 1u : key_at(pos);
                above = key > cut;
                equal = key == cut;
            }
        }
        const uint32_t eq_mask = __ballot_sync(0xffffffffu, equal);
        if (lane == 0) {
            warp_sum[0][warp] = __popc(eq_mask);
        }
        __syncthreads();
        uint32_t v = warp_sum[0][lane], before = 0, total = 0;
        for (int o = 0; o < 32; ++o) {
            const uint32_t x = __shfl_sync(0xffffffffu, v, o);
            before += o < warp ? x : 0u;
            total += x;
        }
        const uint32_t eq_rank = equal_seen + before + __popc(eq_mask & ((1u << lane) - 1u));
        equal_seen += total;
        const bool keep = forced || above || (equal && eq_rank < equal_left);
        const uint32_t mask = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) {
            warp_sum[1][warp] = __popc(mask);
        }
        __syncthreads();
        v = warp_sum[1][lane];
        before = total = 0;
        for (int o = 0; o < 32; ++o) {
            const uint32_t x = __shfl_sync(0xffffffffu, v, o);
            before += o < warp ? x : 0u;
            total += x;
        }
        const uint32_t rank = taken + before + __popc(mask & ((1u << lane) - 1u));
        taken += total;
        if (keep && rank < k) {
            out[rank] = pos;
        }
    }
    for (int64_t i = k + tid; i < a.max_budget; i += kSelectThreads) {
        out[i] = -1;
    }
}

// ---- compaction ----------------------------------------------------------------------------------

struct CompactArgs {
    const int64_t* kept;  // [batch, kept_heads, max_kept]
    const int64_t* base;
    const int64_t* kvlens;
    const int64_t* cachestarts;
    int8_t* cache;
    __half* scale;
    float* weight;  // [L, Hkv, MaxT] or null
    uint32_t* status;
    CacheGeom geom;
    int64_t max_kept, max_kvlen, max_tokens;
    int32_t kept_heads, num_kv_heads, layers;
};

constexpr int kCompactThreads = 256;
constexpr int kUnits = 4;  // 16-byte pieces a thread has in flight

// One CTA per (sequence, layer, kv head, K | V | weight).
template <int DH>
__global__ void __launch_bounds__(kCompactThreads) kv_compact_kernel(const CompactArgs a) {
    constexpr int kCodeUnits = DH / 16;            // 16-byte pieces of a row's codes
    constexpr int kRowUnits = kCodeUnits + DH / 64;  // and of its scales
    constexpr int kRows = kCompactThreads * kUnits / kRowUnits;  // rows of a block
    const int tid = threadIdx.x;
    const int parts = a.weight != nullptr ? 3 : 2;
    int64_t id = blockIdx.x;
    const int part = static_cast<int>(id % parts);
    id /= parts;
    const int head = static_cast<int>(id % a.num_kv_heads);
    id /= a.num_kv_heads;
    const int layer = static_cast<int>(id % a.layers);
    const int64_t b = id / a.layers;
    const int64_t* kept = a.kept + (b * a.kept_heads + (a.kept_heads > 1 ? head : 0)) * a.max_kept;
    const int64_t base = a.base[b];
    int64_t n = a.kvlens[b];
    if (n > a.max_kvlen) {
        n = a.max_kvlen;
        if (tid == 0) {
            atomicOr(a.status, kDevLengthClamped);
        }
    }
    CacheGeom geom = a.geom;
    geom.layer_idx += layer;

    // cache rows of entry i: destination, and source (or -1: not to be moved)
    auto rows_of = [&](int64_t i, int64_t& dst) -> int64_t {
        const int64_t p = kept[i];
        const int64_t before = i > 0 ? kept[i - 1] : -1;
        if (p < 0) {
            return -1;
        }
        if (base < 0 || p < i || (i > 0 && (before < 0 || p <= before)) || base + p >= n) {
            atomicOr(a.status, kDevKeptInvalid);
            return -1;
        }
        if (p == i) {
            return -1;
        }
        const int64_t src = cache_row(geom, a.cachestarts, b, base + p);
        dst = cache_row(geom, a.cachestarts, b, base + i);
        if (!cache_row_ok(src, a.max_tokens) || !cache_row_ok(dst, a.max_tokens)) {
            atomicOr(a.status, kDevRowOutOfRange);
            return -1;
        }
        return src;
    };

    if (part < 2) {
        const int64_t fixed = cache_offset(geom, 0, part, head);
        for (int64_t first = 0; first < a.max_kept; first += kRows) {
            uint4 v[kUnits];
            uint8_t* to[kUnits];
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int unit = u * kCompactThreads + tid;
                const int rr = unit / kRowUnits, piece = unit - rr * kRowUnits;
                to[u] = nullptr;
                if (rr < kRows && first + rr < a.max_kept) {
                    int64_t dst = 0;
                    const int64_t src = rows_of(first + rr, dst);
                    if (src >= 0) {
                        const int64_t so = fixed + src * geom.stride_s, d_o = fixed + dst * geom.stride_s;
                        const uint8_t* from;
                        if (piece < kCodeUnits) {
                            from = reinterpret_cast<const uint8_t*>(a.cache + so) + piece * 16;
                            to[u] = reinterpret_cast<uint8_t*>(a.cache + d_o) + piece * 16;
                        } else {
                            from = reinterpret_cast<const uint8_t*>(a.scale + (so >> 3)) + (piece - kCodeUnits) * 16;
                            to[u] = reinterpret_cast<uint8_t*>(a.scale + (d_o >> 3)) + (piece - kCodeUnits) * 16;
                        }
                        v[u] = *reinterpret_cast<const uint4*>(from);
                    }
                }
            }
            const bool end = kept[first] < 0;
            __syncthreads();  // every source of the block has been read
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                if (to[u] != nullptr) {
                    *reinterpret_cast<uint4*>(to[u]) = v[u];
                }
            }
            if (end) {
                break;
            }
        }
        return;
    }

    float* w = a.weight + ((a.geom.layer_idx + layer) * a.num_kv_heads + head) * a.max_tokens;
    for (int64_t first = 0; first < a.max_kept; first += kCompactThreads * kUnits) {
        float v[kUnits];
        int64_t to[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int64_t i = first + u * kCompactThreads + tid;
            to[u] = -1;
            v[u] = 0.0f;
            if (i < a.max_kept) {
                int64_t dst = 0;
                const int64_t src = rows_of(i, dst);
                if (src >= 0) {
                    v[u] = w[src];
                    to[u] = dst;
                }
            }
        }
        const bool end = kept[first] < 0;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            if (to[u] >= 0) {
                w[to[u]] = v[u];
            }
        }
        if (end) {
            break;
        }
    }
    __syncthreads();
    // the positions behind the kept ones hold no token any more: the next ones start from zero
    int64_t count = 0, top = a.max_kept;  // first negative entry
    while (count < top) {
        const int64_t mid = (count + top) >> 1;
        if (kept[mid] >= 0) {
            count = mid + 1;
        } else {
            top = mid;
        }
    }
    if (base < 0) {
        return;
    }
    for (int64_t pos = base + count + tid; pos < n; pos += kCompactThreads) {
        const int64_t row = cache_row(geom, a.cachestarts, b, pos);
        if (cache_row_ok(row, a.max_tokens)) {
            w[row] = 0.0f;
        } else {
            atomicOr(a.status, kDevRowOutOfRange);
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
    const dim3 grid(static_cast<unsigned>(p.num_kv_heads), static_cast<unsigned>(p.batch));
    kv_evict_select_kernel<<<grid, kSelectThreads, 0, stream>>>(a);
    return check_launch("kv_evict_select_kernel");
}

int launch_kv_compact(const pplb200_attn_params& p, const CacheGeom& geom, const int64_t* kept, int64_t kept_heads,
                      int64_t max_kept, const int64_t* base, const int64_t* kvlens, const int64_t* cachestarts,
                      int64_t layers, void* cache, void* scale, float* weight, uint32_t* status, cudaStream_t stream) {
    CompactArgs a = {};
    a.kept = kept;
    a.base = base;
    a.kvlens = kvlens;
    a.cachestarts = cachestarts;
    a.cache = static_cast<int8_t*>(cache);
    a.scale = static_cast<__half*>(scale);
    a.weight = weight;
    a.status = status;
    a.geom = geom;
    a.max_kept = max_kept;
    a.max_kvlen = p.max_kvlen;
    a.max_tokens = p.max_tokens;
    a.kept_heads = static_cast<int32_t>(kept_heads);
    a.num_kv_heads = p.num_kv_heads;
    a.layers = static_cast<int32_t>(layers);
    const int64_t ctas = p.batch * layers * p.num_kv_heads * (weight != nullptr ? 3 : 2);
    if (ctas > 0x7fffffff) {
        return PPLB200_UNSUPPORTED;
    }
    auto kernel = p.head_dim == 128 ? kv_compact_kernel<128> : kv_compact_kernel<64>;
    kernel<<<static_cast<unsigned>(ctas), kCompactThreads, 0, stream>>>(a);
    return check_launch("kv_compact_kernel");
}

}  // namespace pplb200
