// Accumulated attention weight of many query rows per kv head (the observation window at the end of a prompt), on the
// tensor cores.  128 query rows (token x head of the group) are the M dimension of tcgen05.mma, 64 positions the N
// dimension.  The same kernel runs twice: once for the maximum and the sum of exponentials of each row and chunk of
// positions (attn_window_merge_kernel joins the chunks), once for the weights.  Forming the scores twice costs
// 2 x 2 Dh flops a pair; keeping them would cost 8 bytes of traffic a pair, four times the K row itself at 128 rows.
//
// As in attn_weight.cu the keys are split into fp16(k) and the exact remainder, which makes two tiles of a block; the
// scores accumulate the remainders' products first, the large ones on top.
//
// Roles of a CTA (two per SM): four softmax warps, one thread per query row; they also bring Q, which is the A operand
// in TMEM (64 columns), so that the MMAs read only K from shared memory.  Four converter warps turn raw codes and scales
// into the two swizzled tiles (two stages); one warp issues the MMAs, one fetches raw blocks by TMA.  TMEM: Q 64 | S 2 x
// 64 columns.  The column sums of the weights: scores are read in the fragment layout, four rows and sixteen positions a
// thread; 14 exchanges within the warp leave every lane with the sums of two positions over the warp's 32 rows, shared
// memory adds the four warps up.
// The order of every sum is fixed.
//
// Measured: 4 sequences of 8192 to 32768 positions, 8 kv heads of 128, 116 to 128 rows: statistics 68 us, join 4, weights
// 84 (each kernel by itself), 159 to 164 a call; with warp-level products (mma.sync, 32 rows at a time) 408 us.  For up to
// 32 rows attn_weight.cu is the faster one (figures there).  Bound by no pipe: tensor 39 % and 31 %, DRAM 22 % and 18 %, 2.3
// and 2.1 instructions a cycle; 760 CTAs on 296 places leave the third wave partly empty, but chunks of 512 or 2048
// positions took longer (tried on an earlier form, whose two passes together took 196 and 208 us against 180).
#include "attn_weight.cuh"
#include "kv_tiles.cuh"
#include "ragged.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace pplb200 {

namespace {

constexpr int kRows = 128;      // query rows of a tile
constexpr int kBlockN = kTileRows;
constexpr int kThreads = 320;   // softmax 0..3, converters 4..7, MMA 8, TMA 9
constexpr int kRawStages = 2;
constexpr int kTileStages = 2;
// Warps 0 and 1 add the warps' column sums of a block up.  The scores of block n + 3 imply that every thread is done with
// the scores of n + 1, hence with its part in the sums of n, so four buffers need no barrier for their reuse.
constexpr int kSumStages = 4;

template <int DH>
struct WTraits {
    static constexpr int kColBlocks = DH / 64;
    static constexpr int kKBlockBytes = kBlockN * 128;
    static constexpr int kTileBytes = kColBlocks * kKBlockBytes;  // keys, or their remainders
    static constexpr int kCodeBytes = kBlockN * DH;
    static constexpr int kRawBytes = kCodeBytes + kBlockN * (DH / 8) * 2;
    // the same for every head size: never more than two CTAs share an SM, as its TMEM has room for
    static constexpr int kSmemBytes = kTileStages * 2 * (kBlockN * 256) + kRawStages * (kBlockN * 160) + kSumStages * 4 * kBlockN * 4 +
                                      kWindowChunk * 4 + 512;
    static constexpr uint32_t kColQ = 0, kColS = 64, kTmemCols = 256;
};

struct Barriers {
    uint64_t q_full, q_empty;
    uint64_t raw_full[kRawStages], raw_empty[kRawStages];
    uint64_t k_full[kTileStages], k_empty[kTileStages];
    uint64_t s_full[2], s_free[2];
    uint64_t sum_full[kSumStages];
    uint32_t tmem_slot;
    int abort_word;
};
static_assert(sizeof(Barriers) <= 512, "barrier block");

struct WindowMaps {
    int32_t box_rows;
    CacheMapOrder order;
};

// v[2j + c] = this lane's value for position 8j + 2t + c (t = lane % 4).  Afterwards v[0] and v[1] are the sums over the
// lanes of the same t for j = lane / 4, i.e. for the positions 2 * lane and 2 * lane + 1: halves of the positions are
// exchanged with the lane 16, 8 and 4 away.
__device__ __forceinline__ void sum_positions(float (&v)[16], int lane) {
#pragma unroll
    for (int half = 8; half >= 2; half >>= 1) {
        const bool upper = (lane & (2 * half)) != 0;
#pragma unroll
        for (int e = 0; e < half; ++e) {
            const float give = upper ? v[e] : v[e + half], keep = upper ? v[e + half] : v[e];
            v[e] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * half);
        }
    }
}

template <int DH, bool APPLY>
__global__ void __launch_bounds__(kThreads, 2)
attn_window_kernel(const __grid_constant__ CUtensorMap tm_code, const __grid_constant__ CUtensorMap tm_scale,
                   const WindowMaps maps, const WeightArgs a) {
    using T = WTraits<DH>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sK = smem;  // [stage][keys | remainders]
    uint8_t* sRaw = sK + kTileStages * 2 * T::kTileBytes;
    float* sSum = reinterpret_cast<float*>(sRaw + kRawStages * T::kRawBytes);  // [stage][4 warps][64 positions]
    float* sChunk = sSum + kSumStages * 4 * kBlockN;  // [chunk]: sums of the row tiles so far
    Barriers& bars = *reinterpret_cast<Barriers*>(sChunk + kWindowChunk);
    volatile int* abort_flag = &bars.abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_launch_dependents();
    grid_dependency_wait();
    if ((smem_u32(smem) & 1023u) != 0u) {  // no static shared memory: the window starts on a 1 KB boundary
        if (threadIdx.x == 0) {
            atomicOr(a.status, kDevMmaTimeout);
        }
        return;
    }
    const int64_t b = blockIdx.z;
    const int head = blockIdx.x, chunk = blockIdx.y;  // neighbouring CTAs read neighbouring heads of the same rows
    const Span s = span_of(a, b);
    const int32_t first = chunk * kWindowChunk;
    if (first >= s.len) {
        return;  // uniform for the CTA, before any barrier or TMEM allocation
    }
    const int32_t end = first + kWindowChunk < s.len ? first + kWindowChunk : s.len;
    const int32_t blocks = (end - first + kBlockN - 1) / kBlockN;
    const int32_t row_tiles = (s.rows + kRows - 1) / kRows;
    const int32_t steps = row_tiles * blocks;  // row tiles one after the other, each over all blocks
    if (threadIdx.x == 0) {
        bars.abort_word = 0;
        mbar_init(&bars.q_full, 128);
        mbar_init(&bars.q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.raw_full[i], 1);
            mbar_init(&bars.raw_empty[i], 128);
            mbar_init(&bars.k_full[i], 128);
            mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.s_free[i], 128);
        }
        for (int i = 0; i < kSumStages; ++i) {
            mbar_init(&bars.sum_full[i], 128);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tm_code);
        tma_prefetch_desc(&tm_scale);
    }
    if (warp == 8) {
        tmem_alloc(&bars.tmem_slot, T::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = bars.tmem_slot;

    if (warp == 9) {
        // =========================== TMA producer ===========================
        bool ok = true;
        const int boxes = kBlockN / maps.box_rows;
        int32_t n = 0;
        for (; ok && n < steps; ++n) {
            const int st = n % kRawStages;
            const int32_t blk = n % blocks;
            // lane i < boxes: cache row of the i-th copy; rows outside the cache are flagged and read as zeros
            int row = static_cast<int>(a.max_tokens);
            if (lane < boxes) {
                const int32_t pos = first + blk * kBlockN + lane * maps.box_rows;
                const int32_t rows = s.len - pos < maps.box_rows ? s.len - pos : maps.box_rows;
                if (rows > 0) {
                    const int64_t at = cache_row(a.geom, a.cachestarts, b, pos);
                    if (at < 0 || at + rows > a.max_tokens) {
                        atomicOr(a.status, kDevRowOutOfRange);
                    }
                    if (at >= 0 && at < a.max_tokens) {
                        row = static_cast<int>(at);
                    }
                }
            }
            if (n >= kRawStages) {
                ok = wait_or_abort_parked(&bars.raw_empty[st], ((n / kRawStages) - 1) & 1, abort_flag, a.status, kDevMmaTimeout);
                if (!ok) {
                    break;
                }
            }
            uint8_t* dst = sRaw + st * T::kRawBytes;
            if (lane == 0) {
                mbar_arrive_expect_tx(&bars.raw_full[st], T::kRawBytes);
            }
            __syncwarp();
            if (lane < boxes) {
                load_rows(dst + lane * maps.box_rows * DH, &tm_code, &bars.raw_full[st], maps.order, row, head, 0, a.geom.layer_idx);
                load_rows(dst + T::kCodeBytes + lane * maps.box_rows * (DH / 4), &tm_scale, &bars.raw_full[st], maps.order, row,
                          head, 0, a.geom.layer_idx);
            }
            __syncwarp();
        }
        if (*abort_flag) {
            // every copy this warp issued must have landed before the CTA may exit
            for (int32_t j = n > kRawStages ? n - kRawStages : 0; j < n; ++j) {
                mbar_wait_bounded(&bars.raw_full[j % kRawStages], (j / kRawStages) & 1);
            }
        }
    } else if (warp == 8) {
        // =========================== MMA issuer ===========================
        constexpr uint32_t idesc = instr_desc_f16(kBlockN, false);
        constexpr uint32_t hi_sw128 = desc_hi(1024, 2);
        const uint32_t k_lo = desc_lo(smem_u32(sK), 16);
        bool ok = true;
        for (int32_t n = 0; ok && n < steps; ++n) {
            const int st = n % kTileStages, sb = n & 1;
            if (n % blocks == 0) {
                ok = wait_or_abort(&bars.q_full, (n / blocks) & 1, abort_flag, a.status, kDevMmaTimeout);
            }
            ok = ok && wait_or_abort(&bars.k_full[st], (n / kTileStages) & 1, abort_flag, a.status, kDevMmaTimeout) &&
                 (n < 2 || wait_or_abort(&bars.s_free[sb], ((n >> 1) - 1) & 1, abort_flag, a.status, kDevMmaTimeout));
            if (!ok) {
                break;
            }
            tc_fence_after();
            if (elect_one()) {
                const uint32_t d = tmem_base + T::kColS + sb * kBlockN, q = tmem_base + T::kColQ;
#pragma unroll
                for (int part = 1; part >= 0; --part) {  // remainders first
                    const uint32_t k = k_lo + (st * 2 + part) * (T::kTileBytes >> 4);
#pragma unroll
                    for (int cb = 0; cb < T::kColBlocks; ++cb) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            tc_mma_f16_ts(d, q + 8 * (cb * 4 + i), desc_join(k + cb * (T::kKBlockBytes >> 4) + 2 * i, hi_sw128),
                                          idesc, (part == 0 || (cb | i)) ? 1u : 0u);
                        }
                    }
                }
                tc_commit(&bars.s_full[sb]);
                tc_commit(&bars.k_empty[st]);
                if (n % blocks == blocks - 1) {
                    tc_commit(&bars.q_empty);
                }
            }
            __syncwarp();
        }
    } else if (warp >= 4) {
        // =========================== converters ===========================
        constexpr int kPieces = Raw<DH>::kPieces;
        const int piece = lane % kPieces, row = (warp - 4) * 16 + lane / kPieces;
        const uint32_t tiles = smem_u32(sK), raw0 = smem_u32(sRaw);
        for (int32_t n = 0; n < steps; ++n) {
            const int rs = n % kRawStages, st = n % kTileStages;
            if (!wait_or_abort(&bars.raw_full[rs], (n / kRawStages) & 1, abort_flag, a.status, kDevTmaTimeout)) {
                break;
            }
            Raw<DH> raw;
            raw.load(raw0 + rs * T::kRawBytes, row, piece, s.len - (first + n % blocks * kBlockN));
            if (n >= kTileStages && !wait_or_abort(&bars.k_empty[st], ((n / kTileStages) - 1) & 1, abort_flag, a.status, kDevMmaTimeout)) {
                break;
            }
            const uint32_t tile = tiles + st * 2 * T::kTileBytes;
            raw.store_split(tile, tile + T::kTileBytes, row, piece);
            hand_over(&bars.k_full[st], &bars.raw_empty[rs]);
        }
    } else {
        // =========================== softmax ===========================
        const int r = warp * 32 + lane;  // row of the tile = TMEM lane
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
        const float sc = a.scale_log2;
        float* w = a.weight + (a.geom.layer_idx * a.num_kv_heads + head) * a.max_tokens;
        const int64_t first_row = a.geom.cache_mode == 0 ? a.cachestarts[b] : 0;
        bool ok = true;
        for (int32_t rt = 0; ok && rt < row_tiles; ++rt) {
            const int32_t row = rt * kRows + r;
            const bool live = row < s.rows;
            const int32_t i = live ? row / a.group : 0;
            const int64_t at = (s.tok0 + i) * a.num_heads + head * a.group + (live ? row - i * a.group : 0);
            // Q -> TMEM, two halves per column; rows behind the last are zeros
            if (rt > 0) {
                ok = wait_or_abort(&bars.q_empty, (rt - 1) & 1, abort_flag, a.status, kDevMmaTimeout);
                if (!ok) {
                    break;
                }
                tc_fence_after();
            }
#pragma unroll
            for (int c = 0; c < DH / 32; ++c) {
                uint32_t v[16];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint4 x = live ? *reinterpret_cast<const uint4*>(a.q + at * DH + c * 32 + e * 8) : make_uint4(0u, 0u, 0u, 0u);
                    v[4 * e] = x.x;
                    v[4 * e + 1] = x.y;
                    v[4 * e + 2] = x.z;
                    v[4 * e + 3] = x.w;
                }
                __syncwarp();
                tmem_st16(t_lane + T::kColQ + 16 * c, v);
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars.q_full);

            // Statistics: one thread per row.  Weights: a thread has the rows g + 8k (k = 0..3) of its warp's 32, two of
            // eight positions each, so that most of the sum over the rows stays within it.
            constexpr int kMine = APPLY ? 4 : 1;
            int64_t last[kMine];  // the last position a row sees
            float m[kMine], l[kMine];
#pragma unroll
            for (int k = 0; k < kMine; ++k) {
                const int32_t x = APPLY ? rt * kRows + warp * 32 + (lane >> 2) + 8 * k : row;
                const int32_t tok = x < s.rows ? x / a.group : 0;
                last[k] = a.causal ? s.start + tok : s.len - 1;
                last[k] = last[k] < s.len - 1 ? last[k] : s.len - 1;
                m[k] = APPLY ? INFINITY : kWeightNegBig;  // INFINITY: rows behind the last have no weight
                l[k] = 0.0f;
                if (APPLY && x < s.rows) {
                    const float2 v = a.norm[(s.tok0 + tok) * a.num_heads + head * a.group + (x - tok * a.group)];
                    m[k] = v.x;
                    l[k] = v.y;  // the reciprocal sum
                }
            }
            for (int32_t blk = 0; blk < blocks; ++blk) {
                const int32_t n = rt * blocks + blk;
                const int sb = n & 1;
                ok = wait_or_abort(&bars.s_full[sb], (n >> 1) & 1, abort_flag, a.status, kDevMmaTimeout);
                if (!ok) {
                    break;
                }
                tc_fence_after();
                uint32_t u[2][32];
                __syncwarp();
                if constexpr (APPLY) {
                    tmem_ld_16x64(t_lane + T::kColS + sb * kBlockN, u[0]);
                    tmem_ld_16x64(t_lane + (16u << 16) + T::kColS + sb * kBlockN, u[1]);
                } else {
                    tmem_ld32(t_lane + T::kColS + sb * kBlockN, u[0]);
                    tmem_ld32(t_lane + T::kColS + sb * kBlockN + 32, u[1]);
                }
                tmem_wait_ld();
                tc_fence_before();
                mbar_arrive(&bars.s_free[sb]);
                const int32_t pos0 = first + blk * kBlockN;
                const bool edge = pos0 + kBlockN - 1 > s.start || pos0 + kBlockN > s.len;  // the first row sees up to s.start
                if constexpr (!APPLY) {
                    float v[kBlockN];
#pragma unroll
                    for (int e = 0; e < kBlockN; ++e) {
                        v[e] = __uint_as_float(u[e >> 5][e & 31]);
                    }
                    if (edge) {
                        const int32_t limit = last[0] - pos0 > kBlockN ? kBlockN : static_cast<int32_t>(last[0] - pos0);
#pragma unroll
                        for (int e = 0; e < kBlockN; ++e) {
                            v[e] = e <= limit ? v[e] : -INFINITY;
                        }
                    }
                    float x = fmax3(v[0], v[1], v[2]), y = fmax3(v[3], v[4], v[5]);
#pragma unroll
                    for (int e = 6; e + 3 < kBlockN; e += 4) {
                        x = fmax3(x, v[e], v[e + 1]);
                        y = fmax3(y, v[e + 2], v[e + 3]);
                    }
                    const float top = fmaxf(m[0], fmax3(x, y, fmaxf(v[kBlockN - 2], v[kBlockN - 1])) * sc);
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < kBlockN; e += 2) {
                        const float2 z = __ffma2_rn(make_float2(v[e], v[e + 1]), make_float2(sc, sc), make_float2(-top, -top));
                        sum[e & 2] += ex2_approx(z.x);
                        sum[(e & 2) + 1] += ex2_approx(z.y);
                    }
                    l[0] = l[0] * ex2_approx(m[0] - top) + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                    m[0] = top;
                } else {
                    if (edge) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int64_t rest = last[k] - pos0 - 2 * (lane & 3);
                            const int32_t limit = rest > kBlockN ? kBlockN : static_cast<int32_t>(rest);
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                uint32_t& x = u[k >> 1][4 * (e >> 1) + 2 * (k & 1) + (e & 1)];
                                x = 8 * (e >> 1) + (e & 1) <= limit ? x : 0xff800000u;  // -inf
                            }
                        }
                    }
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {  // row g + 8k
                            const float2 x = make_float2(__uint_as_float(u[k >> 1][4 * j + 2 * (k & 1)]),
                                                         __uint_as_float(u[k >> 1][4 * j + 2 * (k & 1) + 1]));
                            const float2 y = __ffma2_rn(x, make_float2(sc, sc), make_float2(-m[k], -m[k]));
                            sum = __ffma2_rn(make_float2(ex2_approx(y.x), ex2_approx(y.y)), make_float2(l[k], l[k]), sum);
                        }
                        v[2 * j] = sum.x;
                        v[2 * j + 1] = sum.y;
                    }
                    sum_positions(v, lane);
                    float* buf = sSum + (n % kSumStages) * (4 * kBlockN);
                    *reinterpret_cast<float2*>(buf + warp * kBlockN + 2 * lane) = make_float2(v[0], v[1]);
                    mbar_arrive(&bars.sum_full[n % kSumStages]);
                    if (warp >= 2) {
                        continue;
                    }
                    ok = wait_or_abort(&bars.sum_full[n % kSumStages], (n / kSumStages) & 1, abort_flag, a.status, kDevMmaTimeout);
                    if (!ok) {
                        break;
                    }
                    const int32_t e = threadIdx.x;
                    float* sum = &sChunk[blk * kBlockN + e];
                    const float x = (buf[e] + buf[kBlockN + e]) + (buf[2 * kBlockN + e] + buf[3 * kBlockN + e]);
                    *sum = rt > 0 ? *sum + x : x;
                    __syncwarp();
                }
            }
            if constexpr (!APPLY) {
                if (ok && live) {
                    a.part[chunk * a.total_tokens * a.num_heads + at] = make_float2(m[0], l[0]);
                }
            }
        }
        if constexpr (APPLY) {
            // behind the last row tile, not block by block: a row of the cache gets one addition per call
            for (int32_t pos = first + static_cast<int32_t>(threadIdx.x); ok && warp < 2 && pos < end; pos += kBlockN) {
                const int64_t at_row = a.geom.cache_mode == 0 ? (first_row < 0 ? -1 : first_row + pos)
                                                              : cache_row(a.geom, a.cachestarts, b, pos);
                if (cache_row_ok(at_row, a.max_tokens)) {
                    add_weight(w + at_row, sChunk[pos - first]);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem_base, T::kTmemCols);
    }
}

// One warp per (query token, head): joins the chunks of its sequence.
__global__ void __launch_bounds__(256) attn_window_merge_kernel(const WeightArgs a, int32_t batch) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int64_t id = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
    const int64_t tok = id / a.num_heads;
    if (tok >= a.total_tokens) {
        return;
    }
    int32_t lo = 0, hi = batch;  // sequence of the token
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) >> 1;
        if (a.seqstarts[mid] <= tok) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    const int64_t i = tok - a.seqstarts[lo], start = a.start_pos[lo];
    int64_t n = a.seqstarts[lo + 1] - a.seqstarts[lo];
    n = n > a.max_seqlen ? a.max_seqlen : n;
    int64_t len = start < 0 ? 0 : start + n;
    len = len > a.max_kvlen ? a.max_kvlen : len;
    if (i < 0 || i >= n) {
        return;
    }
    const float2 v = join_chunks(a, id, static_cast<int32_t>((len + a.chunk - 1) / a.chunk), lane);
    if (lane == 0) {
        a.norm[id] = v;
    }
}

template <int DH, bool APPLY>
int launch_pass(const pplb200_attn_params& p, const CUtensorMap& tm_code, const CUtensorMap& tm_scale, const WindowMaps& maps,
                const WeightArgs& a, cudaStream_t stream) {
    using T = WTraits<DH>;
    auto kernel = attn_window_kernel<DH, APPLY>;
    // the attribute belongs to the (kernel, device) pair
    static bool attr_set[kMaxDevices] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
        (void)cudaGetLastError();
        return PPLB200_DEVICE_RUNTIME_ERROR;
    }
    if (!attr_set[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmemBytes) != cudaSuccess) {
            (void)cudaGetLastError();
            return PPLB200_DEVICE_RUNTIME_ERROR;
        }
        attr_set[dev] = true;
    }
    const dim3 grid(static_cast<unsigned>(p.num_kv_heads), static_cast<unsigned>(a.chunks), static_cast<unsigned>(p.batch));
    launch_dependent(kernel, grid, dim3(kThreads), T::kSmemBytes, stream, tm_code, tm_scale, maps, a);
    return check_launch("attn_window_kernel");
}

template <int DH>
int launch_dh(const pplb200_attn_params& p, const WeightArgs& a, cudaStream_t stream) {
    WindowMaps maps;
    maps.box_rows = a.geom.cache_mode == 0 || a.geom.page_size % kBlockN == 0 ? kBlockN : 16;
    CUtensorMap tm_code, tm_scale;
    int rc = make_cache_tensor_map(p, a.cache, maps.box_rows, &tm_code, &maps.order);
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    rc = make_scale_tensor_map(p, a.scale, maps.box_rows, &tm_scale);
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    // each kernel starts while the one before it drains, and waits for it before it reads anything
    rc = launch_pass<DH, false>(p, tm_code, tm_scale, maps, a, stream);
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    const int64_t warps = p.total_tokens * p.num_heads;
    launch_dependent(attn_window_merge_kernel, dim3(static_cast<unsigned>((warps * 32 + 255) / 256)), dim3(256), 0, stream, a,
                     static_cast<int32_t>(p.batch));
    rc = check_launch("attn_window_merge_kernel");
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    return launch_pass<DH, true>(p, tm_code, tm_scale, maps, a, stream);
}

}  // namespace

int launch_weight_window(const pplb200_attn_params& p, WeightArgs a, cudaStream_t stream) {
    return p.head_dim == 128 ? launch_dh<128>(p, a, stream) : launch_dh<64>(p, a, stream);
}

}  // namespace pplb200
