// Accumulated attention weight: w[row(j)] += sum over the query heads of a kv group and over the query tokens of
// softmax_j(q . k_j / sqrt(Dh)), for every cached position j of every sequence.  Only K is read.
//
// The normaliser of a row needs all its scores before any weight is known.  This file has the form for up to 32 query
// rows (token x head of the group) per kv head, i.e. for decode steps and short windows; attn_window.cu the one for more.
// attn_weight_stats_kernel leaves, per query row and chunk of positions, the maximum and the sum of exponentials, and
// writes the raw scores to the workspace (4 bytes a row against the 160 of a K row at Dh 128), so that K is read once;
// attn_weight_spread_kernel joins the chunks and turns the scores into weights.
//
// The score kernel: a CTA takes a chunk of the positions of one (sequence, kv head), a warp 16 positions at a time.
// Positions are the M dimension of mma.m16n8k16.  A thread needs the channels 2t, 2t+1, 2t+8, 2t+9 of each block of 16 for
// rows g and g+8 of the A operand; as the order of the channels does not matter as long as Q has the same, thread t takes
// 16 consecutive code bytes per 64 channels.
//
// The weights are fp32 and proportional to exp(score), so a key rounded to fp16 would cost 1e-4 of their value.  With up
// to 4 query rows the codes themselves (exact in fp16) are the A operand and the columns of B are (scale group, query
// row) pairs, each zero outside its group: the accumulators hold a row's products of one group, which are scaled in
// fp32.  With more rows there are too few columns for that, and k = code * scale is split into fp16(k) and the exact
// remainder, which have accumulators of their own.
//
// Measured: 64 sequences of 128 to 4096 positions, 32 kv heads of 128 (771 MB of keys), one row: scores 127 us (6.1 TB/s,
// 92 % of a copy's rate), 155 us with the spread kernel, whose traffic is 4 + 4 + 8 bytes a position against 160.  With
// split keys, bound by their instructions, it was 190.  64 sequences of up to 16384 positions, 8 kv heads (739 MB): 4 rows
// 160, 8 rows 185, 16 rows 255, 32 rows 480 us; attn_window.cu takes 785 us for up to 32 rows and 839 for 128, the kept
// scores of more than 32 rows would be twice the bytes of K and more.  The score kernel of 4
// and 8 rows is bound by its instructions (2.7 a cycle, DRAM 54 %), that of 16 and 32 rows by latency (113 and 168 registers
// leave 23 and 18 % of an SM's warps; tensor pipe 33 and 40 %), and 32 rows have 256 bytes of scores written and read
// against 160 of K.  At Dh 128 the forms for 4 and for 32 rows spill a little (24 and 68 bytes).  Chunks of 512 positions waste a CTA's start, so
// they grow to 4096 while the chip stays full.
#include "attn_weight.cuh"

namespace pplb200 {

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 512;     // positions of a CTA, at least
constexpr int kSpread = 2048;   // positions of a CTA of attn_weight_spread_kernel, where a grid holds that many CTAs
constexpr int64_t kMaxChunks = 65535;  // a grid dimension
// Scores that would take more than this are formed twice instead: the bounds ask for batch x max_kvlen of them, whatever
// the lengths are.  (64 sequences of up to 16384 positions, 8 kv heads: 32 rows keep 1 GB and take 480 us, twice formed 785;
// 4 rows 128 MB and 160 us.  So the limit is high, a fortieth of the memory.)
constexpr uint64_t kScoreBytes = 4ull << 30;
constexpr int kStages = 3;      // tiles of a warp's ring
constexpr float kNegBig = kWeightNegBig;

// D = A B, without an accumulator to start from
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// Four codes with their group's scale -> the two half2 of fp16(code * scale) and of the exact remainders
__device__ __forceinline__ void split_key_word(uint32_t w, __half2 s2, uint32_t& k0, uint32_t& k1, uint32_t& e0,
                                               uint32_t& e1) {
    const uint32_t x = w ^ 0x80808080u;
    const __half2 c0 = biased_bytes_to_half2<0x5140u>(x), c1 = biased_bytes_to_half2<0x5342u>(x);
    const __half2 p0 = __hmul2(c0, s2), p1 = __hmul2(c1, s2);
    k0 = h2_as_u32(p0);
    k1 = h2_as_u32(p1);
    e0 = h2_as_u32(__hfma2(c0, s2, __hneg2(p0)));
    e1 = h2_as_u32(__hfma2(c1, s2, __hneg2(p1)));
}

// A warp's ring of tiles in shared memory: 16 K rows of one (sequence, kv head), codes and scales, copied
// asynchronously, so that kStages - 1 tiles are on their way while one is worked on.
template <int DH>
struct Ring {
    static constexpr int kCodeBytes = 16 * DH;
    static constexpr int kTileBytes = kCodeBytes + 2 * DH * 2;
    static constexpr int kWarpBytes = kStages * kTileBytes;
    static constexpr int kPieces = DH / 16;           // 16-byte pieces of a row's codes
    static constexpr int kRowStep = 32 / kPieces;     // rows the warp copies at once
    static constexpr int kScalePieces = DH / 64;
    const int8_t* code;    // this lane's piece of cache row 0
    const __half* scale;
    int64_t first;         // cache row of position 0 (contiguous cache)
    int32_t safe;          // contiguous cache: tiles below this position are whole and inside the cache
    uint32_t base;         // the ring, in shared memory
    uint32_t code_at, scale_at;  // where in a tile this lane's first copies go

    __device__ __forceinline__ Ring(const WeightArgs& a, const Span& s, int64_t b, int head, int warp, int lane, void* smem) {
        const int64_t off = a.geom.layer_idx * a.geom.stride_l + head * a.geom.stride_h;
        const int i = lane / kPieces, c = lane % kPieces;
        code = a.cache + off + i * a.geom.stride_s + c * 16;
        scale = a.scale + ((off + lane / kScalePieces * a.geom.stride_s) >> 3) + lane % kScalePieces * 8;
        // Dh 128: neighbouring rows swap halves, so that the eight lanes of a read fill all banks
        code_at = i * DH + (DH == 128 ? c ^ ((i & 1) << 2) : c) * 16;
        scale_at = kCodeBytes + lane * 16;
        first = a.geom.cache_mode == 0 ? a.cachestarts[b] : 0;
        safe = s.len & ~15;
        if (a.geom.cache_mode != 0 || first < 0 || first + s.len > a.max_tokens) {
            safe = 0;
        }
        base = smem_u32(smem) + warp * kWarpBytes;
    }

    __device__ __forceinline__ int64_t row_of(const WeightArgs& a, int64_t b, int32_t tile0) const {
        return tile0 < safe ? first + tile0 : cache_row(a.geom, a.cachestarts, b, tile0);
    }

    // The copies of the tile at position tile0 into stage `stage`; every call is one group
    __device__ __forceinline__ void issue(const WeightArgs& a, int64_t b, int32_t tile0, int32_t end, int32_t len, int stage,
                                          int lane) const {
        const uint32_t dst = base + stage * kTileBytes;
        const int64_t row_step = kRowStep * a.geom.stride_s;
        if (tile0 < end && tile0 < safe) {
            const int64_t off = (first + tile0) * a.geom.stride_s;
            const int8_t* src = code + off;
#pragma unroll
            for (int k = 0; k < 16 / kRowStep; ++k) {
                cp_async16(dst + code_at + k * kRowStep * DH, src);
                src += row_step;
            }
            if (lane < 16 * kScalePieces) {
                cp_async16(dst + scale_at, scale + (off >> 3));
            }
        } else if (tile0 < end) {
            // a page, or the last tile: rows that do not exist read as zeros
            const int64_t row0 = cache_row(a.geom, a.cachestarts, b, tile0);
            auto there = [&](int i) -> bool {
                const bool ok = row0 >= 0 && cache_row_ok(row0 + i, a.max_tokens);
                if (tile0 + i < len && !ok) {
                    atomicOr(a.status, kDevRowOutOfRange);
                }
                return tile0 + i < len && ok;
            };
            const int64_t off = row0 * a.geom.stride_s;
#pragma unroll
            for (int k = 0; k < 16 / kRowStep; ++k) {
                const bool ok = there(k * kRowStep + lane / kPieces);
                cp_async16(dst + code_at + k * kRowStep * DH, ok ? code + off + k * row_step : a.cache, ok ? 16u : 0u);
            }
            if (lane < 16 * kScalePieces) {
                const bool ok = there(lane / kScalePieces);
                cp_async16(dst + scale_at, ok ? scale + (off >> 3) : a.scale, ok ? 16u : 0u);
            }
        }
        cp_async_commit();
    }
};

// Where the scores of a thread belong: RB is the number of query rows that the columns of B have room for.
// RB 8, 16, 32: positions g and g + 8, rows 2t and 2t + 1 of each octet.  Below, the four threads of a g share the
// positions out.
template <int RB>
struct Place {
    static constexpr int kOctets = RB < 8 ? 1 : RB / 8;
    static constexpr int kPos = RB >= 8 ? 2 : 1;                         // positions of a thread, 8 apart
    static constexpr int kCols = (RB >= 4 ? 2 : 1) * kOctets;            // rows of a thread
    static __device__ __forceinline__ int position(int lane) {
        return (lane >> 2) + (RB >= 8 ? 0 : 8 * (RB == 4 ? (lane >> 1) & 1 : lane & 1));
    }
    static __device__ __forceinline__ int row(int lane, int c) {
        return RB >= 8 ? 8 * (c >> 1) + 2 * (lane & 3) + (c & 1)
                       : (RB == 4 ? 2 * (lane & 1) + c : (RB == 2 ? (lane >> 1) & 1 : 0));
    }
    // lanes (by their differences) that hold other positions of the same rows; RB 1 has each score twice
    static constexpr uint32_t kPeers = RB >= 8 ? 4 + 8 + 16 : (RB == 4 ? 2 + 4 + 8 + 16 : 1 + 4 + 8 + 16);
    static __device__ __forceinline__ bool first(int lane) { return (lane & kPeers) == 0 && (RB > 1 || lane == 0); }
    static __device__ __forceinline__ bool stores(int lane) { return RB > 1 || (lane & 2) == 0; }
};

// Scores (unscaled) of 16 positions against the query rows whose fragments are in qf.
template <int DH, int RB>
struct Tile {
    static constexpr int kWords = DH / 16;
    static constexpr int kHalves = RB == 4 ? 2 : 1;  // RB 4: two of the four groups of a k-step at a time
    static constexpr int kFrags = kHalves * Place<RB>::kOctets;
    static constexpr int kPos = Place<RB>::kPos, kCols = Place<RB>::kCols;
    using Query = uint2[kFrags][kWords];
    uint4 code[2][DH / 64];
    uint32_t sc[kHalves][2][DH / 64];

    // Where in a tile a lane reads its 16 code bytes of row g (Dh 128: of the first 64 channels; the others are 64
    // bytes up or down, as the copy left them) and its scales
    static __device__ __forceinline__ uint32_t code_offset(int lane) {
        const int g = lane >> 2, t = lane & 3;
        return g * DH + (DH == 128 ? t ^ ((g & 1) << 2) : t) * 16;
    }
    static __device__ __forceinline__ uint32_t scale_offset(int lane) {
        return Ring<DH>::kCodeBytes + (lane >> 2) * (DH / 4) + (RB == 4 ? (lane & 3) >> 1 : lane & 3) * 4;
    }

    __device__ __forceinline__ void read(uint32_t code_addr, uint32_t scale_addr) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int h = 0; h < DH / 64; ++h) {
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(code[r][h].x), "=r"(code[r][h].y), "=r"(code[r][h].z), "=r"(code[r][h].w)
                             : "r"((h == 0 ? code_addr : code_addr ^ 64u) + r * 8 * DH)
                             : "memory");
#pragma unroll
                for (int x = 0; x < kHalves; ++x) {
                    asm volatile("ld.shared.u32 %0, [%1];"
                                 : "=r"(sc[x][r][h])
                                 : "r"(scale_addr + r * 8 * (DH / 4) + h * 16 + x * 8)
                                 : "memory");
                }
            }
        }
    }

    __device__ __forceinline__ uint32_t word(int r, int w) const {
        const uint4 c = code[r][w / 4];
        return (w & 3) == 0 ? c.x : ((w & 3) == 1 ? c.y : ((w & 3) == 2 ? c.z : c.w));
    }

    // Query fragments: row g of an octet, or of column g's (group, row) pair; zeros elsewhere.  Thread t holds the
    // channels of the groups 2t (words 0 and 1 of a block of 64) and 2t + 1.
    static __device__ __forceinline__ void load_queries(const WeightArgs& a, const Span& s, int head, int lane, Query& qf) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int x = 0; x < kFrags; ++x) {
            const int row = RB >= 8 ? 8 * x + g : (RB == 1 ? 0 : g % RB);
            const int32_t i = row / a.group;
            const __half* src = a.q + ((s.tok0 + i) * a.num_heads + head * a.group + (row - i * a.group)) * DH;
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                const bool mine = RB >= 8 || (RB == 4 ? t == 2 * x + (g >> 2) : (RB == 2 ? t == g >> 1 : g == 2 * t + ((w & 3) >> 1)));
                qf[x][w] = make_uint2(0u, 0u);
                if (row < s.rows && mine) {
                    qf[x][w] = *reinterpret_cast<const uint2*>(src + (w / 4) * 64 + t * 16 + (w & 3) * 4);
                }
            }
        }
    }

    __device__ __forceinline__ void scores(const Query& qf, int lane, float (&out)[kPos][kCols]) const {
        if constexpr (RB >= 8) {
            // with one octet two accumulators each for the keys and their remainders: short chains of dependent
            // instructions, and of roundings
            constexpr int kOctets = RB / 8, kChains = RB == 8 ? 2 : 1;
            float key[kChains * kOctets][4], rest[kChains * kOctets][4];
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                uint32_t k[2][2], e[2][2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t s = prmt(sc[0][r][w / 4], 0u, (w & 2) ? 0x3232u : 0x1010u);
                    split_key_word(word(r, w), u32_as_h2(s), k[r][0], k[r][1], e[r][0], e[r][1]);
                }
#pragma unroll
                for (int o = 0; o < kOctets; ++o) {
                    const uint2 q = qf[o][w];
                    const int x = o * kChains + w % kChains;
                    if (w < kChains) {
                        mma_first(key[x], k[0][0], k[1][0], k[0][1], k[1][1], q.x, q.y);
                        mma_first(rest[x], e[0][0], e[1][0], e[0][1], e[1][1], q.x, q.y);
                    } else {
                        mma_m16n8k16_f16f32(key[x], k[0][0], k[1][0], k[0][1], k[1][1], q.x, q.y);
                        mma_m16n8k16_f16f32(rest[x], e[0][0], e[1][0], e[0][1], e[1][1], q.x, q.y);
                    }
                }
            }
#pragma unroll
            for (int o = 0; o < kOctets; ++o) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = o * kChains, y = x + kChains - 1;
                    out[e >> 1][2 * o + (e & 1)] =
                        kChains == 2 ? (key[x][e] + key[y][e]) + (rest[x][e] + rest[y][e]) : key[x][e] + rest[x][e];
                }
            }
        } else {
            constexpr int kSteps = RB == 1 ? 4 : 2;  // k-steps of the same groups
            float sum[2][2] = {};                    // positions g and g + 8; RB 1: [.][0] alone
#pragma unroll
            for (int w0 = 0; w0 < kWords; w0 += kSteps) {
                uint32_t k[kSteps][2][2];
#pragma unroll
                for (int w = 0; w < kSteps; ++w) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint32_t x = word(r, w0 + w) ^ 0x80808080u;
                        k[w][r][0] = h2_as_u32(biased_bytes_to_half2<0x5140u>(x));
                        k[w][r][1] = h2_as_u32(biased_bytes_to_half2<0x5342u>(x));
                    }
                }
#pragma unroll
                for (int x = 0; x < kHalves; ++x) {
                    float acc[4];
                    mma_first(acc, k[0][0][0], k[0][1][0], k[0][0][1], k[0][1][1], qf[x][w0].x, qf[x][w0].y);
#pragma unroll
                    for (int w = 1; w < kSteps; ++w) {
                        mma_m16n8k16_f16f32(acc, k[w][0][0], k[w][1][0], k[w][0][1], k[w][1][1], qf[x][w0 + w].x,
                                            qf[x][w0 + w].y);
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float2 g2 = __half22float2(u32_as_h2(sc[x][r][w0 / 4]));
                        if constexpr (RB == 1) {  // columns 2t, 2t + 1: this thread's own two groups
                            sum[r][0] = fmaf(acc[2 * r], g2.x, fmaf(acc[2 * r + 1], g2.y, sum[r][0]));
                        } else {  // two rows of one group
                            const float f = (w0 & 2) ? g2.y : g2.x;
                            sum[r][0] = fmaf(acc[2 * r], f, sum[r][0]);
                            sum[r][1] = fmaf(acc[2 * r + 1], f, sum[r][1]);
                        }
                    }
                }
            }
            // over the threads of a g: each keeps one of the two positions, RB 2 one of the two rows as well
            constexpr int kFirst = RB == 4 ? 2 : 1;
            const bool upper = (lane & kFirst) != 0;
            float x[2];
#pragma unroll
            for (int c = 0; c < (RB == 1 ? 1 : 2); ++c) {
                x[c] = (upper ? sum[1][c] : sum[0][c]) + __shfl_xor_sync(0xffffffffu, upper ? sum[0][c] : sum[1][c], kFirst);
            }
            if constexpr (RB == 1) {
                out[0][0] = x[0] + __shfl_xor_sync(0xffffffffu, x[0], 2);
            } else if constexpr (RB == 2) {
                const bool second = (lane & 2) != 0;
                out[0][0] = (second ? x[1] : x[0]) + __shfl_xor_sync(0xffffffffu, second ? x[0] : x[1], 2);
            } else {
                out[0][0] = x[0];
                out[0][1] = x[1];
            }
        }
    }
};

template <int DH, int RB>
__global__ void __launch_bounds__(kThreads, RB == 32 ? 3 : RB == 16 ? 4 : RB >= 4 ? 5 : 6) attn_weight_stats_kernel(const WeightArgs a) {
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float2 red[kWarps][RB];
    __shared__ __align__(128) uint8_t smem[kWarps * Ring<DH>::kWarpBytes];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t b = blockIdx.z;
    const int head = blockIdx.x, chunk = blockIdx.y;  // neighbouring CTAs read neighbouring heads of the same rows
    const Span s = span_of(a, b);
    const int32_t first = chunk * a.chunk;
    if (first >= s.len) {
        return;
    }
    const int32_t end = first + a.chunk < s.len ? first + a.chunk : s.len;
    const Ring<DH> ring(a, s, b, head, warp, lane, smem);
    float* score = a.score + (b * a.num_kv_heads + head) * a.max_kvlen * a.score_rows;
    using T = Tile<DH, RB>;
    using At = Place<RB>;
    typename T::Query qf;
    T::load_queries(a, s, head, lane, qf);
    const int my_pos = At::position(lane);
    // the last position that this thread's rows see
    int64_t last[At::kCols];
    float m[At::kCols], l[At::kCols];
#pragma unroll
    for (int c = 0; c < At::kCols; ++c) {
        last[c] = a.causal ? s.start + At::row(lane, c) / a.group : s.len - 1;
        last[c] = last[c] < s.len - 1 ? last[c] : s.len - 1;
        m[c] = kNegBig;
        l[c] = 0.0f;
    }
    constexpr int kStep = kWarps * 16;
    int32_t tile0 = first + warp * 16;
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) {
        ring.issue(a, b, tile0 + k * kStep, end, s.len, k, lane);
    }
    const uint32_t code_addr = ring.base + T::code_offset(lane);
    const uint32_t scale_addr = ring.base + T::scale_offset(lane);
    int stage = 0, ahead = kStages - 1;
    for (; tile0 < end; tile0 += kStep) {
        ring.issue(a, b, tile0 + (kStages - 1) * kStep, end, s.len, ahead, lane);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        T tile;
        tile.read(code_addr + stage * Ring<DH>::kTileBytes, scale_addr + stage * Ring<DH>::kTileBytes);
        __syncwarp();  // everyone has read: the next round may overwrite the stage
        ahead = stage;
        stage = stage + 1 == kStages ? 0 : stage + 1;
        float x[At::kPos][At::kCols];
        tile.scores(qf, lane, x);
        const int32_t pos = tile0 + my_pos;
        if (tile0 + 15 > s.start || tile0 + 15 >= s.len) {
#pragma unroll
            for (int p = 0; p < At::kPos; ++p) {
#pragma unroll
                for (int c = 0; c < At::kCols; ++c) {
                    if (pos + 8 * p > last[c]) {
                        x[p][c] = -INFINITY;
                    }
                }
            }
        }
        if (At::stores(lane)) {
            float* dst = score + static_cast<int64_t>(pos) * a.score_rows;
#pragma unroll
            for (int p = 0; p < At::kPos; ++p) {
                if (pos + 8 * p < s.len) {
#pragma unroll
                    for (int c = 0; c < At::kCols; c += 2) {
                        const int row = At::row(lane, c);
                        if (At::kCols > 1 && row + 1 < a.score_rows) {  // score_rows is even here
                            *reinterpret_cast<float2*>(dst + p * 8 * a.score_rows + row) = make_float2(x[p][c], x[p][(c + 1) % At::kCols]);
                        } else if (row < a.score_rows) {
                            dst[p * 8 * a.score_rows + row] = x[p][c];
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < At::kCols; ++c) {
            float top = m[c], sum = 0.0f;
#pragma unroll
            for (int p = 0; p < At::kPos; ++p) {
                x[p][c] *= a.scale_log2;
                top = fmaxf(top, x[p][c]);
            }
#pragma unroll
            for (int p = 0; p < At::kPos; ++p) {
                sum += ex2_approx(x[p][c] - top);
            }
            l[c] = fmaf(l[c], ex2_approx(m[c] - top), sum);
            m[c] = top;
        }
    }
    cp_async_wait<0>();
    // over the positions a row's values are spread over, then over the warps
#pragma unroll
    for (int c = 0; c < At::kCols; ++c) {
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            if (At::kPeers & x) {
                const float om = __shfl_xor_sync(0xffffffffu, m[c], x);
                const float ol = __shfl_xor_sync(0xffffffffu, l[c], x);
                const float top = fmaxf(m[c], om);
                l[c] = l[c] * ex2_approx(m[c] - top) + ol * ex2_approx(om - top);
                m[c] = top;
            }
        }
        if (At::first(lane)) {
            red[warp][At::row(lane, c)] = make_float2(m[c], l[c]);
        }
    }
    __syncthreads();
    if (static_cast<int32_t>(threadIdx.x) < s.rows) {
        float2 v = red[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) {
            const float2 u = red[k][threadIdx.x];
            const float top = fmaxf(v.x, u.x);
            v.y = v.y * ex2_approx(v.x - top) + u.y * ex2_approx(u.x - top);
            v.x = top;
        }
        const int32_t i = threadIdx.x / a.group;
        const int64_t at = (s.tok0 + i) * a.num_heads + head * a.group + (threadIdx.x - i * a.group);
        a.part[chunk * a.total_tokens * a.num_heads + at] = v;
    }
}

// A thread per position at a time: the weights of the kept scores.  V: how many float4 the rows of a position take; 0: one
// or two rows.
template <int V>
__global__ void __launch_bounds__(256) attn_weight_spread_kernel(const WeightArgs a, int32_t spread) {
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float2 norm[kScoreRows];
    const int64_t b = blockIdx.z;
    const int head = blockIdx.x;
    const Span s = span_of(a, b);
    const int32_t first = blockIdx.y * spread;
    if (first >= s.len) {
        return;
    }
    // a warp per query row joins its chunks
    for (int32_t row = threadIdx.x >> 5; row < s.rows; row += 8) {
        const int32_t i = row / a.group;
        const int64_t at = (s.tok0 + i) * a.num_heads + head * a.group + (row - i * a.group);
        const float2 v = join_chunks(a, at, (s.len + a.chunk - 1) / a.chunk, threadIdx.x & 31);
        if ((threadIdx.x & 31) == 0) {
            norm[row] = v;
        }
    }
    __syncthreads();
    float* w = a.weight + (a.geom.layer_idx * a.num_kv_heads + head) * a.max_tokens;
    const float* score = a.score + (b * a.num_kv_heads + head) * a.max_kvlen * a.score_rows;
    const int64_t start_row = a.geom.cache_mode == 0 ? a.cachestarts[b] : 0;
    auto add = [&](int32_t pos, float x) {
        const int64_t row = a.geom.cache_mode == 0 ? (start_row < 0 ? -1 : start_row + pos)
                                                   : cache_row(a.geom, a.cachestarts, b, pos);
        if (cache_row_ok(row, a.max_tokens)) {
            add_weight(w + row, x);  // one addition per position and call
        }
    };
    auto weight_of = [&](float x, int32_t r) -> float {
        const float2 v = norm[r];
        return ex2_approx(fmaf(x, a.scale_log2, -v.x)) * v.y;
    };
    constexpr int kPer = V == 0 ? 8 : (V >= 8 ? 1 : 8 / V);  // positions of a thread whose loads go out together
    for (int32_t pos0 = first + threadIdx.x; pos0 < first + spread && pos0 < s.len; pos0 += kPer * 256) {
        float sum[kPer];
        if constexpr (V == 0) {
            float x[kPer][2];
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const float* src = score + static_cast<int64_t>(pos0 + k * 256) * a.score_rows;
                const bool there = pos0 + k * 256 < s.len;
                x[k][0] = there ? src[0] : -INFINITY;
                x[k][1] = there && s.rows > 1 ? src[1] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                sum[k] = weight_of(x[k][0], 0) + (s.rows > 1 ? weight_of(x[k][1], 1) : 0.0f);
            }
        } else {
            float4 x[kPer][V];
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const float* src = score + static_cast<int64_t>(pos0 + k * 256) * a.score_rows;
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    x[k][c] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (pos0 + k * 256 < s.len && 4 * c < s.rows) {
                        x[k][c] = *reinterpret_cast<const float4*>(src + 4 * c);
                    }
                }
                sum[k] = 0.0f;
            }
#pragma unroll
            for (int c = 0; c < 4 * V; ++c) {
                if (c < s.rows) {  // rows behind the last were not written, or are another call's
#pragma unroll
                    for (int k = 0; k < kPer; ++k) {
                        const float4 y = x[k][c / 4];
                        sum[k] += weight_of(c % 4 == 0 ? y.x : (c % 4 == 1 ? y.y : (c % 4 == 2 ? y.z : y.w)), c);
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (pos0 + k * 256 < s.len) {
                add(pos0 + k * 256, sum[k]);
            }
        }
    }
}

template <int DH>
int launch_dh(const pplb200_attn_params& p, const WeightArgs& a, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.num_kv_heads), static_cast<unsigned>(a.chunks), static_cast<unsigned>(p.batch));
    // each kernel starts while the one before it drains, and waits for it before it reads anything
    const int64_t rows = p.max_seqlen * a.group;
    launch_dependent(rows <= 1    ? attn_weight_stats_kernel<DH, 1>
                     : rows <= 2  ? attn_weight_stats_kernel<DH, 2>
                     : rows <= 4  ? attn_weight_stats_kernel<DH, 4>
                     : rows <= 8  ? attn_weight_stats_kernel<DH, 8>
                     : rows <= 16 ? attn_weight_stats_kernel<DH, 16>
                                  : attn_weight_stats_kernel<DH, 32>,
                     grid, dim3(kThreads), 0, stream, a);
    const int rc = check_launch("attn_weight_stats_kernel");
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    int64_t share = kSpread;
    while (share * kMaxChunks < p.max_kvlen) {
        share *= 2;
    }
    const dim3 spread(grid.x, static_cast<unsigned>(p.max_kvlen > 0 ? (p.max_kvlen + share - 1) / share : 1), grid.z);
    launch_dependent(rows <= 2    ? attn_weight_spread_kernel<0>
                     : rows <= 4  ? attn_weight_spread_kernel<1>
                     : rows <= 8  ? attn_weight_spread_kernel<2>
                     : rows <= 16 ? attn_weight_spread_kernel<4>
                                  : attn_weight_spread_kernel<8>,
                     spread, dim3(256), 0, stream, a, static_cast<int32_t>(share));
    return check_launch("attn_weight_spread_kernel");
}

}  // namespace

int make_weight_plan(const pplb200_attn_params& p, WeightPlan* plan) {
    // With kept scores a CTA's start (lengths, rows and queries, each waiting for the one before) is worth longer chunks
    // as long as there are some 8 CTAs for each place on the chip.
    const int64_t rows = p.max_seqlen * (p.num_heads / p.num_kv_heads);
    plan->score_rows = rows > kScoreRows ? 0 : static_cast<int32_t>(rows <= 2 ? rows : (rows + 3) / 4 * 4);
    const uint64_t all_rows = static_cast<uint64_t>(p.total_tokens) * p.num_heads;
    const uint64_t positions = static_cast<uint64_t>(p.batch) * p.num_kv_heads * p.max_kvlen;
    if (positions > 1ull << 50 || all_rows > 1ull << 40) {  // keeps the sizes below from wrapping around
        return PPLB200_UNSUPPORTED;
    }
    plan->kept = rows <= kScoreRows &&
                 (positions * plan->score_rows * 4 <= kScoreBytes || p.max_kvlen > kWindowChunk * kMaxChunks);
    plan->chunk = plan->kept ? kChunk : kWindowChunk;
    while (plan->kept && plan->chunk < 8 * kChunk &&
           p.batch * p.num_kv_heads * ((p.max_kvlen + 2 * plan->chunk - 1) / (2 * plan->chunk)) >= 148 * 4 * 8) {
        plan->chunk *= 2;
    }
    // at least one: lengths that the bounds cut to nothing are still looked at, and reported
    plan->chunks = p.max_kvlen > 0 ? (p.max_kvlen + plan->chunk - 1) / plan->chunk : 1;
    plan->off_norm = 256;  // behind the status word
    plan->off_part = plan->off_norm + (all_rows * 8 + 255) / 256 * 256;
    plan->off_score = plan->off_part + (all_rows * plan->chunks * 8 + 255) / 256 * 256;
    plan->bytes = plan->off_score + (plan->kept ? (positions * plan->score_rows * 4 + 255) / 256 * 256 : 0);
    return plan->chunks > kMaxChunks ? PPLB200_UNSUPPORTED : PPLB200_SUCCESS;
}

int launch_attn_weight(const pplb200_attn_params& p, const CacheGeom& geom, const WeightPlan& plan, const void* query,
                       const int64_t* seqstarts, const int64_t* cachestarts, const int64_t* start_pos,
                       const void* cache, const void* scale, float* weight, void* workspace, cudaStream_t stream) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    WeightArgs a = {};
    a.q = static_cast<const __half*>(query);
    a.seqstarts = seqstarts;
    a.cachestarts = cachestarts;
    a.start_pos = start_pos;
    a.cache = static_cast<const int8_t*>(cache);
    a.scale = static_cast<const __half*>(scale);
    a.weight = weight;
    a.norm = reinterpret_cast<float2*>(ws + plan.off_norm);
    a.part = reinterpret_cast<float2*>(ws + plan.off_part);
    a.score = reinterpret_cast<float*>(ws + plan.off_score);
    a.score_rows = plan.score_rows;
    a.status = reinterpret_cast<uint32_t*>(ws);
    a.geom = geom;
    a.max_seqlen = p.max_seqlen;
    a.max_kvlen = p.max_kvlen;
    a.max_tokens = p.max_tokens;
    a.total_tokens = p.total_tokens;
    a.num_heads = p.num_heads;
    a.num_kv_heads = p.num_kv_heads;
    a.group = p.num_heads / p.num_kv_heads;
    a.causal = p.is_causal ? 1 : 0;
    a.chunks = static_cast<int32_t>(plan.chunks);
    a.chunk = plan.chunk;
    a.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(p.head_dim));
    if (!plan.kept) {
        return launch_weight_window(p, a, stream);
    }
    return p.head_dim == 128 ? launch_dh<128>(p, a, stream) : launch_dh<64>(p, a, stream);
}

}  // namespace pplb200
