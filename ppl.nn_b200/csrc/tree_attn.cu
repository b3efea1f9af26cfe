// Attention of a tree of drafted tokens over the INT8 KV cache (speculative decoding's verification step).
//
// Sequence b has start_pos[b] tokens of history and n_b drafted tokens behind them, all in the cache.  Drafted token i
// sees the history, itself and its ancestors.  The query rows that share a kv head -- n_b tokens x the heads of the
// group -- are the M dimension of tcgen05.mma, so that each cached byte is read once per 128 rows:
//   bytes per (position, kv head)  2 (Dh + Dh/4) = 320 at Dh 128; flops 4 Dh per query row, so with the measured
//   rates 160 rows per kv head balance HBM and the tensor cores; below that the cache's bytes are the bound.
//
// Shape of the computation
//   * The unit of work is a BLOCK of 64 positions of one segment = (sequence, kv head, tile of 128 MT query rows).  The
//     kv heads are dealt round-robin into `lanes` classes; neighbouring CTAs take the same range of different classes,
//     i.e. neighbouring heads of the same rows at the same time.  All blocks of a class form one sequence, cut into
//     equal ranges, one per resident CTA.  A range that holds part of a segment leaves an fp32 partial (at most two
//     per range), which tree_merge_kernel joins.
//   * tree_plan_kernel turns the device-side lengths into the prefix sum of blocks, and the parents into one bit mask
//     of ancestors per token.  Only blocks that reach behind the history look at the masks, 64 bits a row and block.
//   * Roles of a CTA: 4 MT softmax warps, one thread per query row; four converter warps, which turn the raw codes and
//     scales of a block into the swizzled fp16 tiles of K, its remainders and V; MT warps that issue the MMAs of a 128-row
//     tile each; one warp that fetches the raw blocks by TMA into a ring of three (MT = 1) or four, in the converters'
//     order.  S = Q K^T goes to a 64-column TMEM
//     buffer, P returns to TMEM as the A operand of O += P V (two buffers), as in the prefill kernel.
//   * MT = 1: two CTAs per SM.  MT = 2, for more than 128 rows per kv head: one CTA per SM, whose two tiles share the
//     fetched and converted K and V.
//
// Roundings: a key rounded to fp16 costs 1e-3 of the output's magnitude where keys have outlying channels, and 3e-3 where
// several positions compete for a row (against 2e-4 for the fp16 output itself), so K is split into fp16(k) and the exact
// remainder, two tiles whose products with Q meet in one accumulator.  Weights and values are rounded to fp16, by up to
// 2^-11 of each and independently, which averages out (weights below 2^-21 of the row's largest by up to 2^-32 of that);
// scores, maxima, sums and outputs are held in fp32.
//
// Measured (8 kv heads of 128): 32 sequences of 256 to 8192 positions, 4 to 64 rows per kv head, 392 MB of cache: 167 us
// for the main kernel by itself, 3 for the plan, 13 for the merge, 193 to 199 a call; 64 such sequences, 200 to 264 rows:
// 493, 3 and 23, 601 to 615 a call; 4 of up to 131072, paged, 228 to 256 rows: 617, 3 and 20, 706 to 719 a call.  The
// kernels by themselves run at 1965 MHz; calls one behind the other draw the card's 1000 W and run at about 1690, which is
// what the calls take beyond the sum.  (Keys rounded to fp16: 163, 515 and 549 a call.)
// What bounds it: tensor pipe 39 % with one tile and 50 % with two, DRAM 30 % and 22 %, 1.9 and 2.1 instructions a cycle:
// the converters, the MMAs' reads of shared memory and the softmax are about as long as one another.  With one tile the 96
// registers that two CTAs an SM leave a thread are just short (56 bytes spilled); with two there are 128.  More converter
// warps were tried with one tile and with rounded keys only, where they did not pay: converters apart for K and V and
// double-buffered scores took 177, 565 and 574 us.  MT = 2 against MT = 1 for 256 rows: K and V are fetched and converted
// once for both tiles; what lies between 129 and 199 rows, and batches of which only some sequences have that many, were
// not measured apart.
//
// Waits on mbarriers are bounded and give up together (see warp_wait.cuh).
#include <cub/block/block_scan.cuh>

#include "common.cuh"
#include "kv_tiles.cuh"
#include "launch.h"
#include "ragged.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace pplb200 {

namespace {

constexpr int kTileM = 128;  // rows of an MMA
constexpr int kBlockN = kTileRows;  // positions of a block
constexpr int kMinRange = 4;  // blocks: no range is cut finer
constexpr float kNegBig = -1.0e30f;
constexpr float kRescaleSlack = 8.0f;  // how far, in powers of two, a maximum may run ahead of a row's reference
// A weight is held in fp16 as 2^kLift times its ratio to the reference: at most 2^(7 + 8), and nothing above 2^-32 of the
// largest vanishes.  (Without the lift 2^-25: behind one token that takes 98 % of a row, the other 131071 would lose a
// quarter of their part.)  The factor is in numerator and sum alike.
constexpr float kLift = 7.0f;

template <int DH, int MT>
struct TTraits {
    static constexpr int kBlockM = kTileM * MT;
    static constexpr int kThreads = 32 * (4 * MT + 4 + MT + 1);
    static constexpr int kCtasPerSm = MT == 1 ? 2 : 1;
    static constexpr int kConvWarp = 4 * MT, kMmaWarp = kConvWarp + 4, kLoadWarp = kMmaWarp + MT;
    static constexpr int kColBlocks = DH / 64;
    static constexpr int kQBlockBytes = kTileM * 128;
    static constexpr int kKVBlockBytes = kBlockN * 128;
    static constexpr int kQBytes = kColBlocks * kQBlockBytes;  // one 128-row tile
    static constexpr int kKVBytes = kColBlocks * kKVBlockBytes;
    static constexpr int kCodeBytes = kBlockN * DH;
    static constexpr int kRawBytes = kCodeBytes + kBlockN * (DH / 8) * 2;  // codes and scales of K or V of a block
    static constexpr int kRawSlots = MT == 1 ? 3 : 4;    // what fits beside a second CTA, or more
    static constexpr int kTileStages = MT == 1 ? 1 : 2;  // converted tiles of K (with remainders) and of V
    // The same for every head size, so that never more CTAs share an SM than its TMEM holds; MT = 2 asks for more
    // than half of the SM's.
    static constexpr int kSmemBytes = MT * 32768 + 3 * kTileStages * (kBlockN * 256) + kRawSlots * (kBlockN * 160) + 512;
    static constexpr uint32_t kPCols = kBlockN / 2;
    static constexpr uint32_t kColS = 0, kColP = kBlockN, kColO = kColP + 2 * kPCols;
    static constexpr uint32_t kTileCols = 256;  // TMEM columns of a tile: S 64 | P 2 x 32 | O 128
};

struct TreeHeader {
    uint32_t status;  // first word of the workspace
    uint32_t reserved;
    int64_t total;  // blocks
    int64_t range;  // blocks per range
};

struct TreeArgs {
    const __half* q;
    const int64_t* parents;
    const int64_t* seqstarts;
    const int64_t* cachestarts;
    const int64_t* start_pos;
    const int8_t* cache;
    const __half* scale;
    __half* out;
    TreeHeader* hdr;
    int64_t* prefix;     // [batch + 1] blocks before each sequence
    uint32_t* flags;     // [batch] what the planning of each sequence has to report
    uint64_t* ancestor;  // [total_tokens][words]
    float* part_o;       // [slots][128][Dh]
    float2* part_ml;     // [slots][128]
    CacheGeom geom;
    int64_t max_kvlen, max_tokens, total_tokens;
    int32_t max_seqlen;
    int32_t words;
    int32_t batch;
    int32_t num_heads, num_kv_heads, group;
    int32_t ranges;   // of a class
    int32_t lanes;    // classes of kv heads
    int32_t tile_rows;  // query rows of a segment: 128 MT
    int32_t box_rows;  // rows of a copy: 64, or 16 where pages may end inside a block
    CacheMapOrder order;
    float scale_log2;
};

// What a sequence is made of; every kernel goes by this
struct Seq {
    int64_t tok0;
    int32_t n, len, start, blocks, row_tiles;
};

__device__ __forceinline__ Seq seq_of(const TreeArgs& a, int64_t b) {
    Seq s;
    s.tok0 = a.seqstarts[b];
    int64_t n = a.seqstarts[b + 1] - s.tok0;
    if (s.tok0 < 0 || s.tok0 + n > a.total_tokens || n < 0) {
        n = 0;
    }
    n = n > a.max_seqlen ? a.max_seqlen : n;
    int64_t start = a.start_pos[b];
    start = start < 0 ? 0 : start;
    start = start > a.max_kvlen ? a.max_kvlen : start;
    const int64_t len = start + n > a.max_kvlen ? a.max_kvlen : start + n;
    s.n = static_cast<int32_t>(n);
    s.start = static_cast<int32_t>(start);
    s.len = static_cast<int32_t>(len);
    s.blocks = n > 0 ? (s.len + kBlockN - 1) / kBlockN : 0;
    s.row_tiles = (s.n * a.group + a.tile_rows - 1) / a.tile_rows;
    return s;
}

// ---- planning: prefix sum of blocks (CTA 0), ancestor masks (a CTA per sequence) --------------------
constexpr int kPlanThreads = 256;

__global__ void __launch_bounds__(kPlanThreads) tree_plan_kernel(const TreeArgs a) {
    using Scan = cub::BlockScan<int64_t, kPlanThreads>;
    __shared__ typename Scan::TempStorage tmp;
    __shared__ int64_t carry;
    __shared__ int32_t up[kTreeMaxTokens];
    const int tid = threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();  // the workspace may still be read by the previous call's kernels
    if (blockIdx.x == 0) {
        if (tid == 0) {
            carry = 0;
            a.hdr->status = 0;
        }
        __syncthreads();
        for (int32_t base = 0; base < a.batch; base += kPlanThreads) {
            const int32_t b = base + tid;
            int64_t units = 0;
            if (b < a.batch) {
                const Seq s = seq_of(a, b);
                units = static_cast<int64_t>(s.blocks) * s.row_tiles * (a.num_kv_heads / a.lanes);
            }
            int64_t excl, total;
            Scan(tmp).ExclusiveSum(units, excl, total);
            const int64_t c = carry;
            if (b < a.batch) {
                a.prefix[b] = c + excl;
            }
            __syncthreads();
            if (tid == 0) {
                carry = c + total;
            }
            __syncthreads();
        }
        if (tid == 0) {
            a.prefix[a.batch] = carry;
            int64_t r = (carry + a.ranges - 1) / a.ranges;
            a.hdr->total = carry;
            a.hdr->range = r < kMinRange ? kMinRange : r;
        }
        return;
    }
    const int32_t b = blockIdx.x - 1;
    const Seq s = seq_of(a, b);
    const int64_t n = a.seqstarts[b + 1] - s.tok0;
    bool bad = false;
    for (int32_t i = tid; i < s.n; i += kPlanThreads) {
        int64_t p = a.parents != nullptr ? a.parents[s.tok0 + i] : i - 1;
        if (p < -1 || p >= i) {
            bad = true;
            p = -1;
        }
        up[i] = static_cast<int32_t>(p);
    }
    bad = __syncthreads_or(bad);
    if (tid == 0) {
        // (a sequence without tokens, as in a padded batch, has nothing to cut, wherever it starts)
        const bool cut = n != 0 && (n != s.n || a.start_pos[b] != s.start || s.start + n > a.max_kvlen);
        a.flags[b] = (cut ? kDevLengthClamped : 0u) | (bad ? kDevParentInvalid : 0u);
    }
    for (int32_t i = tid; i < s.n; i += kPlanThreads) {
        uint64_t* row = a.ancestor + (s.tok0 + i) * a.words;
        int32_t at = i;  // ancestors have strictly smaller indices: the words fill from the highest down
        for (int32_t w = a.words - 1; w >= 0; --w) {
            uint64_t bits = 0;
            while (at >= w * 64) {
                bits |= 1ull << (at & 63);
                at = up[at];
            }
            row[w] = bits;
        }
    }
}

// ---- main kernel -----------------------------------------------------------------------------------

// Part of a segment that lies in the CTA's range
struct Piece {
    Seq seq;
    int32_t b, kvh, rows_valid, row0;  // row0: first query row (token x head of the group) of the segment
    int32_t blk0, blk1;                // blocks [blk0, blk1) of the segment's seq.blocks
};

// The piece that starts at unit u of [.., end) of class `lane_class`; all lanes of a warp call it together.
__device__ __forceinline__ void piece_at(const TreeArgs& a, int64_t u, int64_t end, int lane_class, int lane, Piece& p) {
    p.b = warp_find_segment(a.prefix, a.batch, u, lane);
    p.seq = seq_of(a, p.b);
    const int32_t per_head = p.seq.blocks * p.seq.row_tiles;
    const int64_t q = u - a.prefix[p.b];
    const int32_t vc = static_cast<int32_t>(q / per_head);
    p.kvh = vc * a.lanes + lane_class;
    const int32_t rem = static_cast<int32_t>(q - static_cast<int64_t>(vc) * per_head);
    const int32_t rt = rem / p.seq.blocks;
    p.blk0 = rem - rt * p.seq.blocks;
    const int64_t stop = p.blk0 + (end - u);
    p.blk1 = stop < p.seq.blocks ? static_cast<int32_t>(stop) : p.seq.blocks;
    p.row0 = rt * a.tile_rows;
    const int32_t rows = p.seq.n * a.group - p.row0;
    p.rows_valid = rows < a.tile_rows ? rows : a.tile_rows;
}

template <int MT>
struct Barriers {
    uint64_t q_full, q_empty;
    uint64_t raw_full[4], raw_empty[4];
    uint64_t k_full[MT], k_empty[MT], v_full[MT], v_empty[MT];  // MT stages
    uint64_t o_free[MT], s_full[MT], s_free[MT];
    uint64_t p_full[MT][2], pv_done[MT][2];
    uint32_t tmem_slot;
    int abort_word;
};
static_assert(sizeof(Barriers<2>) <= 512, "barrier block");

template <int DH, int MT>
__global__ void __launch_bounds__(TTraits<DH, MT>::kThreads, TTraits<DH, MT>::kCtasPerSm)
tree_attn_kernel(const __grid_constant__ CUtensorMap tm_code, const __grid_constant__ CUtensorMap tm_scale, const TreeArgs a) {
    using T = TTraits<DH, MT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + MT * T::kQBytes;
    uint8_t* sV = sK + T::kTileStages * 2 * T::kKVBytes;  // K: keys, then their remainders
    uint8_t* sRaw = sV + T::kTileStages * T::kKVBytes;    // a ring of raw K and V blocks
    Barriers<MT>& bars = *reinterpret_cast<Barriers<MT>*>(sRaw + T::kRawSlots * T::kRawBytes);
    volatile int* abort_flag = &bars.abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t* status = &a.hdr->status;

    grid_launch_dependents();
    grid_dependency_wait();
    if ((smem_u32(smem) & 1023u) != 0u) {  // no static shared memory: the window starts on a 1 KB boundary
        if (threadIdx.x == 0) {
            atomicOr(status, kDevMmaTimeout);
        }
        return;
    }
    if (blockIdx.x == 0) {  // the status word has been cleared: now it can take what the planning found
        for (int32_t b = threadIdx.x; b < a.batch; b += T::kThreads) {
            if (a.flags[b] != 0u) {
                atomicOr(status, a.flags[b]);
            }
        }
    }
    const int lane_class = blockIdx.x % a.lanes;
    const int64_t begin = blockIdx.x / a.lanes * a.hdr->range;
    const int64_t total = a.hdr->total;
    const int64_t end = begin + a.hdr->range < total ? begin + a.hdr->range : total;
    if (begin >= end) {
        return;  // uniform for the CTA, before any barrier or TMEM allocation
    }
    if (threadIdx.x == 0) {
        bars.abort_word = 0;
        mbar_init(&bars.q_full, 128);
        mbar_init(&bars.q_empty, MT);
        for (int s = 0; s < T::kRawSlots; ++s) {
            mbar_init(&bars.raw_full[s], 1);
            mbar_init(&bars.raw_empty[s], 128);
        }
        for (int s = 0; s < T::kTileStages; ++s) {
            mbar_init(&bars.k_full[s], 128);
            mbar_init(&bars.v_full[s], 128);
            mbar_init(&bars.k_empty[s], MT);
            mbar_init(&bars.v_empty[s], MT);
        }
        for (int t = 0; t < MT; ++t) {
            mbar_init(&bars.o_free[t], 128);
            mbar_init(&bars.s_full[t], 1);
            mbar_init(&bars.s_free[t], 128);
            for (int i = 0; i < 2; ++i) {
                mbar_init(&bars.p_full[t][i], 128);
                mbar_init(&bars.pv_done[t][i], 1);
            }
        }
        mbar_fence_init();
        tma_prefetch_desc(&tm_code);
        tma_prefetch_desc(&tm_scale);
    }
    if (warp == T::kMmaWarp) {
        tmem_alloc(&bars.tmem_slot, MT * T::kTileCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = bars.tmem_slot;

    if (warp == T::kLoadWarp) {
        // =========================== TMA producer ===========================
        bool ok = true;
        int n = 0;  // raw blocks requested so far
        for (int64_t u = begin; ok && u < end;) {
            Piece p;
            piece_at(a, u, end, lane_class, lane, p);
            const int boxes = kBlockN / a.box_rows, blocks = p.blk1 - p.blk0;
            u += blocks;
            for (int i = 0; ok && i < 2 * blocks; ++i, ++n) {
                // the converters' order: K(0) K(1) V(0) K(2) V(1) ..
                const int kv = i == 2 * blocks - 1 || (i > 0 && (i & 1) == 0) ? 1 : 0;
                const int32_t blk = p.blk0 + (kv == 0 ? (i + 1) / 2 : (i & 1) ? blocks - 1 : i / 2 - 1);
                const int s = n % T::kRawSlots;
                // lane i < boxes: cache row of the i-th copy; rows outside the cache are flagged and read as zeros
                int row = static_cast<int>(a.max_tokens);
                if (lane < boxes) {
                    const int32_t pos = blk * kBlockN + lane * a.box_rows;
                    const int32_t rows = p.seq.len - pos < a.box_rows ? p.seq.len - pos : a.box_rows;
                    if (rows > 0) {
                        const int64_t first = cache_row(a.geom, a.cachestarts, p.b, pos);
                        if (first < 0 || first + rows > a.max_tokens) {
                            atomicOr(status, kDevRowOutOfRange);
                        }
                        if (first >= 0 && first < a.max_tokens) {
                            row = static_cast<int>(first);
                        }
                    }
                }
                if (n >= T::kRawSlots) {
                    ok = wait_or_abort_parked(&bars.raw_empty[s], ((n / T::kRawSlots) - 1) & 1, abort_flag, status, kDevMmaTimeout);
                    if (!ok) {
                        break;
                    }
                }
                uint8_t* dst = sRaw + s * T::kRawBytes;
                uint64_t* bar = &bars.raw_full[s];
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar, T::kRawBytes);
                }
                __syncwarp();
                if (lane < boxes) {
                    load_rows(dst + lane * a.box_rows * DH, &tm_code, bar, a.order, row, p.kvh, kv, a.geom.layer_idx);
                    load_rows(dst + T::kCodeBytes + lane * a.box_rows * (DH / 4), &tm_scale, bar, a.order, row, p.kvh, kv, a.geom.layer_idx);
                }
                __syncwarp();
            }
        }
        if (*abort_flag) {
            // every copy this warp issued must have landed before the CTA may exit; a slot whose copies were issued
            // is complete at the latest parity it was armed with (a slot that was never armed is left alone)
            for (int j = n > T::kRawSlots ? n - T::kRawSlots : 0; j < n; ++j) {
                mbar_wait_bounded(&bars.raw_full[j % T::kRawSlots], (j / T::kRawSlots) & 1);
            }
        }
    } else if (warp >= T::kMmaWarp) {
        // =========================== MMA issuer of one 128-row tile ===========================
        constexpr uint32_t idesc_qk = instr_desc_f16(kBlockN, false);
        constexpr uint32_t idesc_pv = instr_desc_f16(DH, true);
        constexpr uint32_t hi_sw128 = desc_hi(1024, 2);
        const int t = warp - T::kMmaWarp;
        const uint32_t q_lo = desc_lo(smem_u32(sQ) + t * T::kQBytes, 16);
        const uint32_t k_lo = desc_lo(smem_u32(sK), 16);
        const uint32_t v_lo = desc_lo(smem_u32(sV), T::kKVBlockBytes);
        const uint32_t tm = tmem_base + t * T::kTileCols;
        const uint32_t d_s = tm + T::kColS, d_o = tm + T::kColO, a_p = tm + T::kColP;
        bool ok = true;
        int pieces = 0, blocks_done = 0;    // of the CTA
        int mine = 0, kc = 0, vc = 0;       // pieces, Q K^T and P V of this tile
        for (int64_t u = begin; ok && u < end; ++pieces) {
            Piece p;
            piece_at(a, u, end, lane_class, lane, p);
            const int32_t blocks = p.blk1 - p.blk0;
            u += blocks;
            ok = wait_or_abort(&bars.q_full, pieces & 1, abort_flag, status, kDevMmaTimeout);
            if (t * kTileM >= p.rows_valid) {
                // no rows for this tile: only hand the operands back
                for (int32_t j = 0; ok && j < blocks; ++j, ++blocks_done) {
                    const int st = blocks_done % T::kTileStages, parity = (blocks_done / T::kTileStages) & 1;
                    ok = wait_or_abort_parked(&bars.k_full[st], parity, abort_flag, status, kDevMmaTimeout);
                    if (ok && lane == 0) {
                        mbar_arrive(&bars.k_empty[st]);
                        if (j == blocks - 1) {
                            mbar_arrive(&bars.q_empty);
                        }
                    }
                    ok = ok && wait_or_abort_parked(&bars.v_full[st], parity, abort_flag, status, kDevMmaTimeout);
                    if (ok && lane == 0) {
                        mbar_arrive(&bars.v_empty[st]);
                    }
                    __syncwarp();
                }
                continue;
            }
            for (int32_t j = 0; ok && j <= blocks; ++j) {
                if (j < blocks) {
                    const int st = (blocks_done + j) % T::kTileStages;
                    ok = wait_or_abort(&bars.k_full[st], ((blocks_done + j) / T::kTileStages) & 1, abort_flag, status, kDevMmaTimeout) &&
                         (kc == 0 || wait_or_abort(&bars.s_free[t], (kc - 1) & 1, abort_flag, status, kDevMmaTimeout));
                    if (!ok) {
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int part = 1; part >= 0; --part) {  // the remainders' products first, the large ones on top
#pragma unroll
                            for (int cb = 0; cb < T::kColBlocks; ++cb) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    tc_mma_f16(d_s, desc_join(q_lo + cb * (T::kQBlockBytes >> 4) + 2 * k, hi_sw128),
                                               desc_join(k_lo + ((2 * st + part) * T::kKVBytes + cb * T::kKVBlockBytes) / 16 + 2 * k, hi_sw128),
                                               idesc_qk, (part == 0 || (cb | k)) ? 1u : 0u);
                                }
                            }
                        }
                        tc_commit(&bars.s_full[t]);
                        tc_commit(&bars.k_empty[st]);
                        if (j == blocks - 1) {
                            tc_commit(&bars.q_empty);
                        }
                    }
                    __syncwarp();
                    ++kc;
                }
                if (j > 0) {
                    const int st = (blocks_done + j - 1) % T::kTileStages;
                    ok = wait_or_abort(&bars.v_full[st], ((blocks_done + j - 1) / T::kTileStages) & 1, abort_flag, status, kDevMmaTimeout) &&
                         wait_or_abort(&bars.p_full[t][vc & 1], (vc >> 1) & 1, abort_flag, status, kDevMmaTimeout);
                    if (ok && j == 1 && mine > 0) {
                        ok = wait_or_abort(&bars.o_free[t], (mine - 1) & 1, abort_flag, status, kDevMmaTimeout);
                    }
                    if (!ok) {
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t pa = a_p + (vc & 1) * T::kPCols;
#pragma unroll
                        for (int ks = 0; ks < kBlockN / 16; ++ks) {
                            tc_mma_f16_ts(d_o, pa + 8 * ks, desc_join(v_lo + st * (T::kKVBytes >> 4) + ks * (2048 >> 4), hi_sw128), idesc_pv,
                                          ((j - 1) | ks) ? 1u : 0u);
                        }
                        tc_commit(&bars.v_empty[st]);
                        tc_commit(&bars.pv_done[t][vc & 1]);
                    }
                    __syncwarp();
                    ++vc;
                }
            }
            blocks_done += blocks;
            ++mine;
        }
    } else if (warp >= T::kConvWarp) {
        // =========================== converters ===========================
        const int ct = threadIdx.x - 32 * T::kConvWarp;
        constexpr int kPieces = Raw<DH>::kPieces;
        const int piece = lane % kPieces;
        const int row = (warp - T::kConvWarp) * 16 + lane / kPieces;  // first of the thread's rows of a block
        const uint32_t k_tile = smem_u32(sK), v_tile = smem_u32(sV), raw0 = smem_u32(sRaw), q_tile = smem_u32(sQ);
        bool ok = true;
        int pieces = 0, n = 0, taken = 0;  // pieces, blocks and raw blocks so far
        // K (0) or V (1) of the CTA's block number `blk_no`, of which `rows` rows exist: the next one of the ring
        auto convert = [&](int kv, int blk_no, int32_t rows) -> bool {
            const int s = taken % T::kRawSlots;
            if (!wait_or_abort(&bars.raw_full[s], (taken / T::kRawSlots) & 1, abort_flag, status, kDevTmaTimeout)) {
                return false;
            }
            ++taken;
            Raw<DH> raw;
            raw.load(raw0 + s * T::kRawBytes, row, piece, rows);
            const int st = blk_no % T::kTileStages;
            if (blk_no >= T::kTileStages && !wait_or_abort(kv ? &bars.v_empty[st] : &bars.k_empty[st],
                                                           ((blk_no / T::kTileStages) - 1) & 1, abort_flag, status, kDevMmaTimeout)) {
                return false;
            }
            if (kv) {
                raw.store(v_tile + st * T::kKVBytes, row, piece);
            } else {
                raw.store_split(k_tile + 2 * st * T::kKVBytes, k_tile + (2 * st + 1) * T::kKVBytes, row, piece);
            }
            hand_over(kv ? &bars.v_full[st] : &bars.k_full[st], &bars.raw_empty[s]);
            return true;
        };
        for (int64_t u = begin; ok && u < end; ++pieces) {
            Piece p;
            piece_at(a, u, end, lane_class, lane, p);
            u += p.blk1 - p.blk0;
            // Q: row r of the tile is query row row0 + r = token x head of the group
            if (pieces > 0) {
                ok = wait_or_abort(&bars.q_empty, (pieces - 1) & 1, abort_flag, status, kDevMmaTimeout);
                if (!ok) {
                    break;
                }
            }
            constexpr int kQPieces = DH / 8;  // 16-byte pieces of a query row
            for (int i = ct; i < p.rows_valid * kQPieces; i += 128) {
                const int r = i / kQPieces, c = i - r * kQPieces;
                const int32_t qrow = p.row0 + r;
                const int32_t tok = qrow / a.group;
                const uint4 v = *reinterpret_cast<const uint4*>(
                    a.q + ((p.seq.tok0 + tok) * a.num_heads + p.kvh * a.group + (qrow - tok * a.group)) * DH + c * 8);
                sts128(q_tile + (r / kTileM) * T::kQBytes + (c >> 3) * T::kQBlockBytes + (r % kTileM) * 128 +
                           (((c & 7) ^ (r & 7)) << 4), v);
            }
            fence_proxy_async_smem();
            mbar_arrive(&bars.q_full);
            // K runs one block ahead of V: V(j) has to wait for P V(j - 1), i.e. for a softmax, and the scores of block
            // j + 1 should not wait with it
            ok = convert(0, n, p.seq.len - p.blk0 * kBlockN);
            for (int32_t blk = p.blk0; ok && blk < p.blk1; ++blk, ++n) {
                if (blk + 1 < p.blk1) {
                    ok = convert(0, n + 1, p.seq.len - (blk + 1) * kBlockN);
                }
                ok = ok && convert(1, n, p.seq.len - blk * kBlockN);
            }
        }
    } else {
        // =========================== softmax / epilogue ===========================
        const int t = warp >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane;  // row of the tile = TMEM lane
        const uint32_t t_lane = (static_cast<uint32_t>(quarter * 32) << 16) + t * T::kTileCols;
        const uint32_t t_s = tmem_base + t_lane + T::kColS;
        const uint32_t t_o = tmem_base + t_lane + T::kColO;
        const uint32_t t_p = tmem_base + t_lane + T::kColP;
        const float sc = a.scale_log2;
        bool ok = true;
        int pc = 0;
        for (int64_t u = begin; ok && u < end;) {
            Piece p;
            piece_at(a, u, end, lane_class, lane, p);
            u += p.blk1 - p.blk0;
            const int32_t rows_valid = p.rows_valid - t * kTileM;  // of this tile
            if (rows_valid <= 0) {
                continue;
            }
            if (quarter * 32 >= rows_valid) {
                // the rows of this warp are behind the last one: its lanes only keep the barriers going
                for (int32_t blk = p.blk0; ok && blk < p.blk1; ++blk, ++pc) {
                    ok = wait_or_abort_parked(&bars.s_full[t], pc & 1, abort_flag, status, kDevMmaTimeout);
                    if (ok) {
                        mbar_arrive(&bars.s_free[t]);
                        mbar_arrive(&bars.p_full[t][pc & 1]);
                    }
                }
                ok = ok && wait_or_abort_parked(&bars.pv_done[t][(pc - 1) & 1], ((pc - 1) >> 1) & 1, abort_flag, status,
                                                kDevMmaTimeout);
                if (ok) {
                    mbar_arrive(&bars.o_free[t]);
                }
                continue;
            }
            const bool live = r < rows_valid;
            const int32_t row = p.row0 + t * kTileM + r;
            const int32_t tok = live ? row / a.group : 0;
            const uint64_t* anc = a.ancestor + (p.seq.tok0 + tok) * a.words;
            float m_ref = kNegBig, l_sum = 0.0f;
            for (int32_t blk = p.blk0; ok && blk < p.blk1; ++blk, ++pc) {
                if (pc >= 2) {
                    ok = wait_or_abort(&bars.pv_done[t][pc & 1], ((pc - 2) >> 1) & 1, abort_flag, status, kDevMmaTimeout);
                    if (!ok) {
                        break;
                    }
                }
                ok = wait_or_abort(&bars.s_full[t], pc & 1, abort_flag, status, kDevMmaTimeout);
                if (!ok) {
                    break;
                }
                tc_fence_after();
                float sv[kBlockN];
                {
                    uint32_t v[kBlockN / 32][32];
#pragma unroll
                    for (int c = 0; c < kBlockN / 32; ++c) {
                        tmem_ld32(t_s + 32 * c, v[c]);
                    }
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < kBlockN / 32; ++c) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            sv[32 * c + e] = __uint_as_float(v[c][e]);
                        }
                    }
                }
                tc_fence_before();
                mbar_arrive(&bars.s_free[t]);
                const int32_t a0 = blk * kBlockN - p.seq.start;  // index of the block's first position among the drafts
                if (a0 + kBlockN > 0) {
                    // 64 positions of this row: bit e = position blk * 64 + e is visible
                    uint64_t seen = ~0ull;
                    if (live) {
                        if (a0 <= 0) {
                            seen = (a0 == 0 ? 0ull : ~0ull >> (64 + a0)) | (anc[0] << -a0);
                        } else {
                            const int32_t w = a0 >> 6, sh = a0 & 63;
                            seen = w < a.words ? anc[w] >> sh : 0ull;
                            if (sh > 0 && w + 1 < a.words) {
                                seen |= anc[w + 1] << (64 - sh);
                            }
                        }
                        const int32_t room = p.seq.len - blk * kBlockN;  // positions that exist
                        if (room < kBlockN) {
                            seen &= ~0ull >> (64 - room);
                        }
                    }
                    const uint32_t lo = static_cast<uint32_t>(seen), hi = static_cast<uint32_t>(seen >> 32);
#pragma unroll
                    for (int e = 0; e < kBlockN; ++e) {
                        sv[e] = ((e < 32 ? lo : hi) >> (e & 31)) & 1u ? sv[e] : -INFINITY;
                    }
                }
                float mx0 = fmax3(sv[0], sv[1], sv[2]), mx1 = fmax3(sv[3], sv[4], sv[5]);
#pragma unroll
                for (int e = 6; e + 3 < kBlockN; e += 4) {
                    mx0 = fmax3(mx0, sv[e], sv[e + 1]);
                    mx1 = fmax3(mx1, sv[e + 2], sv[e + 3]);
                }
                float mx = fmax3(mx0, mx1, fmaxf(sv[kBlockN - 2], sv[kBlockN - 1]));
                mx *= sc;
                const bool grow = mx > m_ref + kRescaleSlack;
                if (__any_sync(0xffffffffu, grow)) {
                    const float m_new = grow ? mx : m_ref;
                    const float f = ex2_approx(m_ref - m_new);
                    m_ref = m_new;
                    l_sum *= f;
                    if (blk > p.blk0) {
                        ok = wait_or_abort(&bars.pv_done[t][(pc - 1) & 1], ((pc - 1) >> 1) & 1, abort_flag, status, kDevMmaTimeout);
                        if (!ok) {
                            break;
                        }
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < DH / 8; ++c) {  // eight columns at a time: the scores stay in registers
                            uint32_t v[8];
                            tmem_ld8(t_o + c * 8, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                            }
                            tmem_st8(t_o + c * 8, v);
                        }
                        tmem_wait_st();
                    }
                }
                // P = exp2(s * scale - m_ref + kLift) as packed fp16; the row sum adds the rounded values that P V uses, in
                // four chains (one chain of 64 dependent additions would be as long as the exponentials)
                const uint32_t t_pb = t_p + (pc & 1) * T::kPCols;
                const float lift = kLift - m_ref;
                float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int q = 0; q < kBlockN / 32; ++q) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 x = __ffma2_rn(make_float2(sv[32 * q + 2 * e], sv[32 * q + 2 * e + 1]),
                                                    make_float2(sc, sc), make_float2(lift, lift));
                        pk[e] = h2_as_u32(__floats2half2_rn(ex2_approx(x.x), ex2_approx(x.y)));
                        add_half2_to_float(l4[e & 3], pk[e]);
                    }
                    tmem_st16(t_pb + 16 * q, pk);
                }
                l_sum += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&bars.p_full[t][pc & 1]);
            }
            // ---- epilogue: the whole segment -> fp16 rows; a part of one -> fp32 partial ----
            if (ok) {
                ok = wait_or_abort(&bars.pv_done[t][(pc - 1) & 1], ((pc - 1) >> 1) & 1, abort_flag, status, kDevMmaTimeout);
            }
            if (ok) {
                tc_fence_after();
                const bool whole = p.blk0 == 0 && p.blk1 == p.seq.blocks;
                const float inv = l_sum > 0.0f ? 1.0f / l_sum : 0.0f;
                __half* dst = a.out + ((p.seq.tok0 + tok) * a.num_heads + p.kvh * a.group + (row - tok * a.group)) * DH;
                const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (p.blk0 == 0 ? 1 : 0)) * T::kBlockM + t * kTileM + r;
                float* part = a.part_o + slot * DH;
                if (!whole && live) {
                    a.part_ml[slot] = make_float2(m_ref, l_sum);
                }
#pragma unroll
                for (int c = 0; c < DH / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld32(t_o + c * 32, v);
                    tmem_wait_ld();
                    if (c == DH / 32 - 1) {
                        tc_fence_before();
                        mbar_arrive(&bars.o_free[t]);
                    }
                    if (live && whole) {
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            uint32_t o[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                o[e] = h2_as_u32(__floats2half2_rn(__uint_as_float(v[16 * q + 2 * e]) * inv,
                                                                   __uint_as_float(v[16 * q + 2 * e + 1]) * inv));
                            }
                            st_global_v8(dst + c * 32 + q * 16, o);
                        }
                    } else if (live) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint32_t o[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                o[e] = v[8 * q + e];
                            }
                            st_global_v8(part + c * 32 + q * 8, o);
                        }
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == T::kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, MT * T::kTileCols);
    }
}

// ---- joining the parts of a segment that several ranges hold -----------------------------------------

// A CTA per range and 32 query rows: the segment that begins in the range and goes on behind it, if there is one.  A
// warp per row.
constexpr int kMergeThreads = 512;
constexpr int kMergeRows = 32;

template <int DH>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const TreeArgs a) {
    constexpr int kPer = DH / 32;  // channels of a lane
    const int lane = threadIdx.x & 31;
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t range = a.hdr->range, first = blockIdx.x / a.lanes, lane_class = blockIdx.x % a.lanes;
    const int64_t last_unit = (first + 1) * range - 1;
    if (last_unit + 1 >= a.hdr->total) {
        return;
    }
    Piece p;  // of the range's last block: its segment
    piece_at(a, last_unit, last_unit + 1, static_cast<int>(lane_class), lane, p);
    const int64_t u0 = last_unit - p.blk0, u1 = u0 + p.seq.blocks;  // units of the segment
    if (u0 < first * range || u1 <= last_unit + 1) {
        return;  // it began before the range, or ends with it
    }
    const int64_t last = (u1 - 1) / range;
    const int32_t r0 = blockIdx.y * kMergeRows, r1 = r0 + kMergeRows < p.rows_valid ? r0 + kMergeRows : p.rows_valid;
    for (int32_t r = r0 + (threadIdx.x >> 5); r < r1; r += kMergeThreads / 32) {
        // the segment's first part is the second of its range's two, the others are first ones
        auto slot_of = [&](int64_t w) -> int64_t {
            return (2 * (w * a.lanes + lane_class) + (w == first ? 1 : 0)) * a.tile_rows + r;
        };
        float m = kNegBig;
        for (int64_t w = first; w <= last; ++w) {
            m = fmaxf(m, a.part_ml[slot_of(w)].x);
        }
        float l = 0.0f, o[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            o[e] = 0.0f;
        }
        for (int64_t w = first; w <= last; ++w) {
            const int64_t slot = slot_of(w);
            const float2 ml = a.part_ml[slot];
            const float f = ex2_approx(ml.x - m);
            const float* part = a.part_o + slot * DH + lane * kPer;
            l += ml.y * f;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                o[e] += part[e] * f;
            }
        }
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        const int32_t row = p.row0 + r, tok = row / a.group;
        __half2* dst = reinterpret_cast<__half2*>(
            a.out + ((p.seq.tok0 + tok) * a.num_heads + p.kvh * a.group + (row - tok * a.group)) * DH + lane * kPer);
#pragma unroll
        for (int e = 0; e < kPer; e += 2) {
            dst[e / 2] = __floats2half2_rn(o[e] * inv, o[e + 1] * inv);
        }
    }
}

uint64_t align256(uint64_t x) {
    return (x + 255) / 256 * 256;
}

template <int DH, int MT>
int launch_dh(const pplb200_attn_params& p, TreeArgs a, cudaStream_t stream) {
    using T = TTraits<DH, MT>;
    auto kernel = tree_attn_kernel<DH, MT>;
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
    a.tile_rows = T::kBlockM;
    a.box_rows = a.geom.cache_mode == 0 || a.geom.page_size % kBlockN == 0 ? kBlockN : 16;
    CUtensorMap tm_code, tm_scale;
    int rc = make_cache_tensor_map(p, a.cache, a.box_rows, &tm_code, &a.order);
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    rc = make_scale_tensor_map(p, a.scale, a.box_rows, &tm_scale);
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    // each kernel starts while the one before it drains, and waits for it before it touches anything
    launch_dependent(tree_plan_kernel, dim3(static_cast<unsigned>(a.batch + 1)), dim3(kPlanThreads), 0, stream, a);
    rc = check_launch("tree_plan_kernel");
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    launch_dependent(kernel, dim3(static_cast<unsigned>(a.ranges * a.lanes)), dim3(T::kThreads), T::kSmemBytes, stream, tm_code,
                     tm_scale, a);
    rc = check_launch("tree_attn_kernel");
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    launch_dependent(tree_merge_kernel<DH>, dim3(static_cast<unsigned>(a.ranges * a.lanes), T::kBlockM / kMergeRows), dim3(kMergeThreads), 0, stream, a);
    return check_launch("tree_merge_kernel");
}

}  // namespace

int make_tree_plan(const pplb200_attn_params& p, int sm_count, TreePlan* plan) {
    // query rows per kv head beyond one MMA tile: two tiles of a CTA share K and V
    plan->tiles = p.max_seqlen * (p.num_heads / p.num_kv_heads) > kTileM ? 2 : 1;
    const int64_t tile_rows = plan->tiles * kTileM;
    const int64_t resident = plan->tiles == 1 ? 2 * static_cast<int64_t>(sm_count) : sm_count;
    plan->lanes = 8;
    while (p.num_kv_heads % plan->lanes != 0 || resident % plan->lanes != 0) {
        plan->lanes >>= 1;
    }
    // no more ranges than there can be work for
    const int64_t row_tiles = (p.max_seqlen * (p.num_heads / p.num_kv_heads) + tile_rows - 1) / tile_rows;
    const int64_t blocks = (p.max_kvlen + kBlockN - 1) / kBlockN;
    // (in floating point: the product of the largest sizes does not fit 64 bits)
    const double units = static_cast<double>(p.batch) * (p.num_kv_heads / plan->lanes) * row_tiles * blocks;
    const int64_t places = resident / plan->lanes;
    plan->ranges = units > static_cast<double>(places) * kMinRange ? places : (static_cast<int64_t>(units) + kMinRange - 1) / kMinRange;
    plan->ranges = plan->ranges < 1 ? 1 : plan->ranges;  // lengths that the bounds cut to nothing are still reported
    plan->words = (p.max_seqlen + 63) / 64;
    const uint64_t slot_rows = static_cast<uint64_t>(plan->ranges) * plan->lanes * 2 * tile_rows;
    plan->off_prefix = 256;
    plan->off_flags = plan->off_prefix + align256(static_cast<uint64_t>(p.batch + 1) * 8);
    plan->off_ancestor = plan->off_flags + align256(static_cast<uint64_t>(p.batch) * 4);
    plan->off_part_ml = plan->off_ancestor + align256(static_cast<uint64_t>(p.total_tokens) * plan->words * 8);
    plan->off_part_o = plan->off_part_ml + slot_rows * 8;
    plan->bytes = plan->off_part_o + slot_rows * p.head_dim * 4;
    return PPLB200_SUCCESS;
}

int launch_tree_attn(const pplb200_attn_params& p, const CacheGeom& geom, const TreePlan& plan, const void* query,
                     const int64_t* parents, const int64_t* seqstarts, const int64_t* cachestarts,
                     const int64_t* start_pos, const void* cache, const void* scale, void* workspace,
                     void* attn_output, cudaStream_t stream) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    TreeArgs a = {};
    a.q = static_cast<const __half*>(query);
    a.parents = parents;
    a.seqstarts = seqstarts;
    a.cachestarts = cachestarts;
    a.start_pos = start_pos;
    a.cache = static_cast<const int8_t*>(cache);
    a.scale = static_cast<const __half*>(scale);
    a.out = static_cast<__half*>(attn_output);
    a.hdr = reinterpret_cast<TreeHeader*>(ws);
    a.prefix = reinterpret_cast<int64_t*>(ws + plan.off_prefix);
    a.flags = reinterpret_cast<uint32_t*>(ws + plan.off_flags);
    a.ancestor = reinterpret_cast<uint64_t*>(ws + plan.off_ancestor);
    a.part_ml = reinterpret_cast<float2*>(ws + plan.off_part_ml);
    a.part_o = reinterpret_cast<float*>(ws + plan.off_part_o);
    a.geom = geom;
    a.max_kvlen = p.max_kvlen;
    a.max_tokens = p.max_tokens;
    a.total_tokens = p.total_tokens;
    a.max_seqlen = static_cast<int32_t>(p.max_seqlen);
    a.words = static_cast<int32_t>(plan.words);
    a.batch = static_cast<int32_t>(p.batch);
    a.num_heads = p.num_heads;
    a.num_kv_heads = p.num_kv_heads;
    a.group = p.num_heads / p.num_kv_heads;
    a.ranges = static_cast<int32_t>(plan.ranges);
    a.lanes = static_cast<int32_t>(plan.lanes);
    a.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(p.head_dim));
    if (plan.tiles == 2) {
        return p.head_dim == 128 ? launch_dh<128, 2>(p, a, stream) : launch_dh<64, 2>(p, a, stream);
    }
    return p.head_dim == 128 ? launch_dh<128, 1>(p, a, stream) : launch_dh<64, 1>(p, a, stream);
}

}  // namespace pplb200
