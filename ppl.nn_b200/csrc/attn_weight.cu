// Accumulated attention weight: w[row(j)] += sum over the query heads of a kv group and over the query tokens of
// softmax_j(q . k_j / sqrt(Dh)), for every cached position j of every sequence.  Only K is read.
//
// The normaliser of a row needs all its scores before any weight is known.  attn_weight_stats_kernel leaves, per query
// row and chunk of positions, the maximum and the sum of exponentials, and attn_weight_merge_kernel joins the chunks.
// With up to 8 query rows per kv head (decode steps) the scores themselves go to the workspace as well (4 bytes a row
// against the 160 of a K row at Dh 128), and attn_weight_spread_kernel joins the chunks and reads the scores; with more
// rows attn_weight_apply_kernel forms them again and adds each position's normalised weights up.
//
// Both score kernels: a CTA takes a chunk of the positions of one (sequence, kv head), a warp 16 positions at a
// time.  Positions are the M dimension of mma.m16n8k16, the query rows (token x head of the group) come in octets as
// its N dimension.  A thread needs the channels 2t, 2t+1, 2t+8, 2t+9 of each block of 16 for rows g and g+8 of the
// A operand; as the order of the channels does not matter as long as Q has the same, thread t takes 16 consecutive
// code bytes per 64 channels straight from global memory.
//
// The weights are fp32 and proportional to exp(score), so a key rounded to fp16 would cost 1e-4 of their value;
// k = code * scale is therefore split into fp16(k) and the exact remainder, and both enter the accumulator.
#include "common.cuh"
#include "launch.h"

namespace pplb200 {

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 512;     // positions of a CTA where the scores are formed twice
constexpr int kSpread = 2048;   // positions of a CTA of attn_weight_spread_kernel
constexpr int kRowBlock = 32;   // query rows whose fragments are held in registers at a time
constexpr int kScoreRows = 8;   // up to so many query rows per kv head the scores are kept
constexpr int kStages = 3;      // tiles of a warp's ring
constexpr float kNegBig = -1.0e30f;

struct WeightArgs {
    const __half* q;
    const int64_t* seqstarts;
    const int64_t* cachestarts;
    const int64_t* start_pos;
    const int8_t* cache;
    const __half* scale;
    float* weight;   // [L, Hkv, MaxT]
    float2* part;    // [chunks][T][Hq]: maximum (exp2 domain) and sum
    float2* norm;    // [T][Hq]: maximum and reciprocal sum
    float* score;    // [batch][Hkv][max_kvlen][kScoreRows or fewer]: raw scores, -inf where hidden, or null
    int32_t score_rows;
    uint32_t* status;
    CacheGeom geom;
    int64_t max_seqlen, max_kvlen, max_tokens, total_tokens;
    int32_t num_heads, num_kv_heads, group, causal, chunks;
    int32_t chunk;   // positions of a chunk
    float scale_log2;
};

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

// What a CTA works on
struct Span {
    int64_t tok0;   // first query row of the sequence
    int64_t start;  // positions before its first query token
    int32_t rows;   // query rows: tokens * group
    int32_t len;    // positions
};

__device__ __forceinline__ Span span_of(const WeightArgs& a, int64_t b) {
    Span s;
    s.tok0 = a.seqstarts[b];
    int64_t n = a.seqstarts[b + 1] - s.tok0;
    if (s.tok0 < 0 || s.tok0 + n > a.total_tokens) {
        n = 0;
    }
    bool cut = n > a.max_seqlen;
    n = cut ? a.max_seqlen : (n < 0 ? 0 : n);
    s.start = a.start_pos[b];
    int64_t len = s.start < 0 ? 0 : s.start + n;
    if (len > a.max_kvlen) {
        len = a.max_kvlen;
        cut = true;
    }
    if (cut && threadIdx.x == 0) {
        atomicOr(a.status, kDevLengthClamped);
    }
    s.rows = static_cast<int32_t>(n) * a.group;
    s.len = n > 0 ? static_cast<int32_t>(len) : 0;
    return s;
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

// Scores (unscaled) of 16 positions against NOCT octets of query rows whose fragments are in qf.
// acc[o][0..1]: position g, rows 2t and 2t+1 of octet o; acc[o][2..3]: position g + 8.
template <int DH, int NOCT>
struct Tile {
    static constexpr int kWords = DH / 16;
    uint4 code[2][DH / 64];
    uint32_t sc[2][DH / 64];

    // Where in a tile a lane reads its 16 code bytes of row g (Dh 128: of the first 64 channels; the others are 64
    // bytes up or down, as the copy left them) and its scales
    static __device__ __forceinline__ uint32_t code_offset(int lane) {
        const int g = lane >> 2, t = lane & 3;
        return g * DH + (DH == 128 ? t ^ ((g & 1) << 2) : t) * 16;
    }
    static __device__ __forceinline__ uint32_t scale_offset(int lane) {
        return Ring<DH>::kCodeBytes + (lane >> 2) * (DH / 4) + (lane & 3) * 4;
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
                asm volatile("ld.shared.u32 %0, [%1];"
                             : "=r"(sc[r][h])
                             : "r"(scale_addr + r * 8 * (DH / 4) + h * 16)
                             : "memory");
            }
        }
    }

    // The keys and their remainders have accumulators of their own, and with one octet there are two of each: shorter
    // chains of dependent instructions, and of roundings.
    __device__ __forceinline__ void scores(const uint2 (&qf)[NOCT][kWords], float (&acc)[NOCT][4]) const {
        constexpr int kChains = NOCT == 1 ? 2 : 1;
        float key[kChains][NOCT][4], rest[kChains][NOCT][4];
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            uint32_t k[2][2], e[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint4 c = code[r][w / 4];
                const uint32_t word = (w & 3) == 0 ? c.x : ((w & 3) == 1 ? c.y : ((w & 3) == 2 ? c.z : c.w));
                const uint32_t s = prmt(sc[r][w / 4], 0u, (w & 2) ? 0x3232u : 0x1010u);
                split_key_word(word, u32_as_h2(s), k[r][0], k[r][1], e[r][0], e[r][1]);
            }
#pragma unroll
            for (int o = 0; o < NOCT; ++o) {
                if (w < kChains) {
                    mma_first(key[w % kChains][o], k[0][0], k[1][0], k[0][1], k[1][1], qf[o][w].x, qf[o][w].y);
                } else {
                    mma_m16n8k16_f16f32(key[w % kChains][o], k[0][0], k[1][0], k[0][1], k[1][1], qf[o][w].x, qf[o][w].y);
                }
            }
#pragma unroll
            for (int o = 0; o < NOCT; ++o) {
                if (w < kChains) {
                    mma_first(rest[w % kChains][o], e[0][0], e[1][0], e[0][1], e[1][1], qf[o][w].x, qf[o][w].y);
                } else {
                    mma_m16n8k16_f16f32(rest[w % kChains][o], e[0][0], e[1][0], e[0][1], e[1][1], qf[o][w].x, qf[o][w].y);
                }
            }
        }
#pragma unroll
        for (int o = 0; o < NOCT; ++o) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[o][e] = key[0][o][e] + rest[0][o][e];
                if constexpr (kChains == 2) {
                    acc[o][e] = (key[0][o][e] + key[1][o][e]) + (rest[0][o][e] + rest[1][o][e]);
                }
            }
        }
    }
};

// Query fragments of the rows [row0, row0 + 8 NOCT): rows behind the last read as zeros
template <int DH, int NOCT>
__device__ __forceinline__ void load_queries(const WeightArgs& a, const Span& s, int head, int32_t row0, int lane,
                                             uint2 (&qf)[NOCT][DH / 16]) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int o = 0; o < NOCT; ++o) {
        const int32_t r = row0 + o * 8 + g;
        const int32_t i = r / a.group;
        const __half* src = a.q + ((s.tok0 + i) * a.num_heads + head * a.group + (r - i * a.group)) * DH;
#pragma unroll
        for (int w = 0; w < DH / 16; ++w) {
            qf[o][w] = make_uint2(0u, 0u);
            if (r < s.rows) {
                qf[o][w] = *reinterpret_cast<const uint2*>(src + (w / 4) * 64 + t * 16 + (w & 3) * 4);
            }
        }
    }
}

// -inf in the places of `acc` that a query row may not see
template <int NOCT>
__device__ __forceinline__ void hide(const WeightArgs& a, const Span& s, int32_t row0, int32_t tile0, int lane,
                                     float (&acc)[NOCT][4]) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int o = 0; o < NOCT; ++o) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int32_t r = row0 + o * 8 + 2 * t + c;
            const int64_t last = a.causal ? s.start + r / a.group : s.len - 1;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int32_t j = tile0 + g + 8 * p;
                if (j > last || j >= s.len) {
                    acc[o][2 * p + c] = -INFINITY;
                }
            }
        }
    }
}

// work(tile, position) for this warp's tiles of [tile0, end)
template <int DH, int NOCT, typename Work>
__device__ __forceinline__ void for_tiles(const WeightArgs& a, const Ring<DH>& ring, int64_t b, int32_t tile0, int32_t end,
                                          int32_t len, int lane, Work work) {
    constexpr int kStep = kWarps * 16;
    __syncwarp();  // the ring may still be read for the rows before
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) {
        ring.issue(a, b, tile0 + k * kStep, end, len, k, lane);
    }
    const uint32_t code_addr = ring.base + Tile<DH, NOCT>::code_offset(lane);
    const uint32_t scale_addr = ring.base + Tile<DH, NOCT>::scale_offset(lane);
    int stage = 0, ahead = kStages - 1;
    for (; tile0 < end; tile0 += kStep) {
        ring.issue(a, b, tile0 + (kStages - 1) * kStep, end, len, ahead, lane);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        Tile<DH, NOCT> tile;
        tile.read(code_addr + stage * Ring<DH>::kTileBytes, scale_addr + stage * Ring<DH>::kTileBytes);
        __syncwarp();  // everyone has read: the next round may overwrite the stage
        work(tile, tile0);
        ahead = stage;
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    cp_async_wait<0>();
}

template <int DH, int NOCT>
__global__ void __launch_bounds__(kThreads, NOCT == 1 ? 6 : 3) attn_weight_stats_kernel(const WeightArgs a) {
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float2 red[kWarps][NOCT * 8];
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
    float* score = a.score + (b * a.num_kv_heads + head) * a.max_kvlen * a.score_rows;  // NOCT == 1
    for (int32_t row0 = 0; row0 < s.rows; row0 += NOCT * 8) {
        uint2 qf[NOCT][DH / 16];
        load_queries<DH, NOCT>(a, s, head, row0, lane, qf);
        float m[NOCT][2], l[NOCT][2];
#pragma unroll
        for (int o = 0; o < NOCT; ++o) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[o][c] = kNegBig;
                l[o][c] = 0.0f;
            }
        }
        auto work = [&](const Tile<DH, NOCT>& tile, int32_t tile0) {
            float acc[NOCT][4];
            tile.scores(qf, acc);
            if (tile0 + 15 > s.start || tile0 + 15 >= s.len) {
                hide<NOCT>(a, s, row0, tile0, lane, acc);
            }
            if constexpr (NOCT == 1) {
                const int g = lane >> 2, t = lane & 3;
                if (2 * t < s.rows) {
                    float* dst = score + (tile0 + g) * a.score_rows + 2 * t;
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        if (tile0 + g + 8 * p < s.len) {
                            dst[p * 8 * a.score_rows] = acc[0][2 * p];
                            if (2 * t + 1 < s.rows) {
                                dst[p * 8 * a.score_rows + 1] = acc[0][2 * p + 1];
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int o = 0; o < NOCT; ++o) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float x = acc[o][c] * a.scale_log2, y = acc[o][2 + c] * a.scale_log2;
                    const float top = fmaxf(m[o][c], fmaxf(x, y));
                    l[o][c] = l[o][c] * ex2_approx(m[o][c] - top) + ex2_approx(x - top) + ex2_approx(y - top);
                    m[o][c] = top;
                }
            }
        };
        for_tiles<DH, NOCT>(a, ring, b, first + warp * 16, end, s.len, lane, work);
        // over the eight positions a column's values are spread over, then over the warps
#pragma unroll
        for (int o = 0; o < NOCT; ++o) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    const float om = __shfl_xor_sync(0xffffffffu, m[o][c], x);
                    const float ol = __shfl_xor_sync(0xffffffffu, l[o][c], x);
                    const float top = fmaxf(m[o][c], om);
                    l[o][c] = l[o][c] * ex2_approx(m[o][c] - top) + ol * ex2_approx(om - top);
                    m[o][c] = top;
                }
                if (lane < 4) {
                    red[warp][o * 8 + 2 * lane + c] = make_float2(m[o][c], l[o][c]);
                }
            }
        }
        __syncthreads();
        const int32_t r = row0 + threadIdx.x;
        if (threadIdx.x < NOCT * 8 && r < s.rows) {
            float2 v = red[0][threadIdx.x];
#pragma unroll
            for (int k = 1; k < kWarps; ++k) {
                const float2 u = red[k][threadIdx.x];
                const float top = fmaxf(v.x, u.x);
                v.y = v.y * ex2_approx(v.x - top) + u.y * ex2_approx(u.x - top);
                v.x = top;
            }
            const int32_t i = r / a.group;
            const int64_t at = (s.tok0 + i) * a.num_heads + head * a.group + (r - i * a.group);
            a.part[chunk * a.total_tokens * a.num_heads + at] = v;
        }
        __syncthreads();
    }
}

// Maximum and reciprocal sum of row `at` over its chunks; all lanes of a warp call it.
__device__ __forceinline__ float2 join_chunks(const WeightArgs& a, int64_t at, int32_t chunks, int lane) {
    float m = kNegBig, l = 0.0f;
    for (int32_t c = lane; c < chunks; c += 32) {
        const float2 v = a.part[c * a.total_tokens * a.num_heads + at];
        const float top = fmaxf(m, v.x);
        l = l * ex2_approx(m - top) + v.y * ex2_approx(v.x - top);
        m = top;
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, x), ol = __shfl_xor_sync(0xffffffffu, l, x);
        const float top = fmaxf(m, om);
        l = l * ex2_approx(m - top) + ol * ex2_approx(om - top);
        m = top;
    }
    return make_float2(m, l > 0.0f ? 1.0f / l : 0.0f);
}

// One warp per (query token, head): joins the chunks of its sequence.
__global__ void __launch_bounds__(256) attn_weight_merge_kernel(const WeightArgs a, int32_t batch) {
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

template <int DH, int NOCT>
__global__ void __launch_bounds__(kThreads, 3) attn_weight_apply_kernel(const WeightArgs a) {
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float sum[kChunk];
    __shared__ __align__(128) uint8_t smem[kWarps * Ring<DH>::kWarpBytes];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int64_t b = blockIdx.z;
    const int head = blockIdx.x, chunk = blockIdx.y;  // neighbouring CTAs read neighbouring heads of the same rows
    const Span s = span_of(a, b);
    const int32_t first = chunk * kChunk;
    if (first >= s.len) {
        return;
    }
    const int32_t end = first + kChunk < s.len ? first + kChunk : s.len;
    const Ring<DH> ring(a, s, b, head, warp, lane, smem);
    float* w = a.weight + (a.geom.layer_idx * a.num_kv_heads + head) * a.max_tokens;
    for (int32_t row0 = 0; row0 < s.rows; row0 += NOCT * 8) {
        uint2 qf[NOCT][DH / 16];
        load_queries<DH, NOCT>(a, s, head, row0, lane, qf);
        float neg_m[NOCT][2], inv[NOCT][2];
#pragma unroll
        for (int o = 0; o < NOCT; ++o) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int32_t r = row0 + o * 8 + 2 * t + c;
                neg_m[o][c] = -INFINITY;  // rows behind the last: no weight
                inv[o][c] = 0.0f;
                if (r < s.rows) {
                    const int32_t i = r / a.group;
                    const float2 v = a.norm[(s.tok0 + i) * a.num_heads + head * a.group + (r - i * a.group)];
                    neg_m[o][c] = -v.x;
                    inv[o][c] = v.y;
                }
            }
        }
        const bool last_rows = row0 + NOCT * 8 >= s.rows;
        auto work = [&](const Tile<DH, NOCT>& tile, int32_t tile0) {
            float acc[NOCT][4];
            tile.scores(qf, acc);
            if (tile0 + 15 > s.start || tile0 + 15 >= s.len) {
                hide<NOCT>(a, s, row0, tile0, lane, acc);
            }
            float part[2] = {0.0f, 0.0f};
#pragma unroll
            for (int o = 0; o < NOCT; ++o) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        part[p] = fmaf(ex2_approx(fmaf(acc[o][2 * p + c], a.scale_log2, neg_m[o][c])), inv[o][c], part[p]);
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                part[p] += __shfl_xor_sync(0xffffffffu, part[p], 1);
                part[p] += __shfl_xor_sync(0xffffffffu, part[p], 2);
            }
            // lane t = 0 of a quad owns position g, t = 1 position g + 8: one addition per position and call
            if (t < 2) {
                const int i = g + 8 * t;
                float x = t == 0 ? part[0] : part[1];
                float* acc_row = &sum[tile0 - first + i];
                if (row0 > 0) {
                    x += *acc_row;
                }
                if (!last_rows) {
                    *acc_row = x;
                } else if (tile0 + i < s.len) {
                    const int64_t row = ring.row_of(a, b, tile0);
                    if (row >= 0 && cache_row_ok(row + i, a.max_tokens)) {
                        atomicAdd(w + row + i, x);
                    }
                }
            }
        };
        for_tiles<DH, NOCT>(a, ring, b, first + warp * 16, end, s.len, lane, work);
    }
}

// One thread per position: the weights of the kept scores.
__global__ void __launch_bounds__(256) attn_weight_spread_kernel(const WeightArgs a) {
    grid_launch_dependents();
    grid_dependency_wait();
    __shared__ float2 norm[kScoreRows];
    const int64_t b = blockIdx.z;
    const int head = blockIdx.x;
    const Span s = span_of(a, b);
    const int32_t first = blockIdx.y * kSpread;
    if (first >= s.len) {
        return;
    }
    // a warp per query row joins its chunks
    const int32_t my_row = threadIdx.x >> 5;
    if (my_row < s.rows) {
        const int32_t i = my_row / a.group;
        const int64_t at = (s.tok0 + i) * a.num_heads + head * a.group + (my_row - i * a.group);
        const float2 v = join_chunks(a, at, (s.len + a.chunk - 1) / a.chunk, threadIdx.x & 31);
        if ((threadIdx.x & 31) == 0) {
            norm[my_row] = v;
        }
    }
    __syncthreads();
    float* w = a.weight + (a.geom.layer_idx * a.num_kv_heads + head) * a.max_tokens;
    const float* score = a.score + (b * a.num_kv_heads + head) * a.max_kvlen * a.score_rows;
    const int64_t start_row = a.geom.cache_mode == 0 ? a.cachestarts[b] : 0;
    constexpr int kPer = kSpread / 256;  // positions of a thread: their loads go out together
    const int32_t pos0 = first + threadIdx.x;
    float sum[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        sum[k] = 0.0f;
    }
    for (int32_t r = 0; r < s.rows; ++r) {
        const float2 v = norm[r];
        float x[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            x[k] = pos0 + k * 256 < s.len ? score[static_cast<int64_t>(pos0 + k * 256) * a.score_rows + r] : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            sum[k] = fmaf(ex2_approx(fmaf(x[k], a.scale_log2, -v.x)), v.y, sum[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int32_t pos = pos0 + k * 256;
        if (pos < s.len) {
            const int64_t row = a.geom.cache_mode == 0 ? (start_row < 0 ? -1 : start_row + pos)
                                                       : cache_row(a.geom, a.cachestarts, b, pos);
            if (cache_row_ok(row, a.max_tokens)) {
                atomicAdd(w + row, sum[k]);  // one addition per position and call
            }
        }
    }
}

template <int DH>
int launch_dh(const pplb200_attn_params& p, const WeightArgs& a, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(p.num_kv_heads), static_cast<unsigned>(a.chunks), static_cast<unsigned>(p.batch));
    // each kernel starts while the one before it drains, and waits for it before it reads anything
    if (p.max_seqlen * a.group <= kScoreRows) {
        launch_dependent(attn_weight_stats_kernel<DH, 1>, grid, dim3(kThreads), 0, stream, a);
        const int rc = check_launch("attn_weight_stats_kernel");
        if (rc != PPLB200_SUCCESS) {
            return rc;
        }
        const dim3 spread(grid.x, static_cast<unsigned>((p.max_kvlen + kSpread - 1) / kSpread), grid.z);
        launch_dependent(attn_weight_spread_kernel, spread, dim3(256), 0, stream, a);
        return check_launch("attn_weight_spread_kernel");
    }
    launch_dependent(attn_weight_stats_kernel<DH, kRowBlock / 8>, grid, dim3(kThreads), 0, stream, a);
    int rc = check_launch("attn_weight_stats_kernel");
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    const int64_t warps = p.total_tokens * p.num_heads;
    launch_dependent(attn_weight_merge_kernel, dim3(static_cast<unsigned>((warps * 32 + 255) / 256)), dim3(256), 0, stream, a,
                     static_cast<int32_t>(p.batch));
    rc = check_launch("attn_weight_merge_kernel");
    if (rc != PPLB200_SUCCESS) {
        return rc;
    }
    launch_dependent(attn_weight_apply_kernel<DH, kRowBlock / 8>, grid, dim3(kThreads), 0, stream, a);
    return check_launch("attn_weight_apply_kernel");
}

}  // namespace

int make_weight_plan(const pplb200_attn_params& p, WeightPlan* plan) {
    // With kept scores a CTA's start (lengths, rows and queries, each waiting for the one before) is worth longer chunks
    // as long as there are some 8 CTAs for each place on the chip.
    const bool kept = p.max_seqlen > 0 && p.max_seqlen * (p.num_heads / p.num_kv_heads) <= kScoreRows;
    plan->chunk = kChunk;
    while (kept && plan->chunk < 8 * kChunk &&
           p.batch * p.num_kv_heads * ((p.max_kvlen + 2 * plan->chunk - 1) / (2 * plan->chunk)) >= 148 * 4 * 8) {
        plan->chunk *= 2;
    }
    plan->chunks = (p.max_kvlen + plan->chunk - 1) / plan->chunk;
    const uint64_t rows = static_cast<uint64_t>(p.total_tokens) * p.num_heads;
    plan->off_norm = 256;  // behind the status word
    plan->off_part = plan->off_norm + (rows * 8 + 255) / 256 * 256;
    plan->off_score = plan->off_part + (rows * plan->chunks * 8 + 255) / 256 * 256;
    plan->score_rows = static_cast<int32_t>(p.max_seqlen * (p.num_heads / p.num_kv_heads));
    const uint64_t positions = static_cast<uint64_t>(p.batch) * p.num_kv_heads * p.max_kvlen;
    plan->bytes = plan->off_score + (kept ? (positions * plan->score_rows * 4 + 255) / 256 * 256 : 0);
    return plan->chunks > 65535 ? PPLB200_UNSUPPORTED : PPLB200_SUCCESS;  // a grid dimension
}

int launch_attn_weight(const pplb200_attn_params& p, const CacheGeom& geom, const WeightPlan& plan, const void* query,
                       const int64_t* seqstarts, const int64_t* cachestarts, const int64_t* start_pos,
                       const void* cache, const void* scale, float* weight, void* workspace, cudaStream_t stream) {
    if (plan.chunks <= 0 || p.max_seqlen <= 0) {
        return PPLB200_SUCCESS;
    }
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
    return p.head_dim == 128 ? launch_dh<128>(p, a, stream) : launch_dh<64>(p, a, stream);
}

}  // namespace pplb200
