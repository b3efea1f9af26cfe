// What the kernels of the accumulated attention weight share: their arguments, what a CTA works on, and the join of a
// row's chunks.
#pragma once

#include "common.cuh"
#include "launch.h"

namespace pplb200 {

constexpr int kScoreRows = 32;      // up to so many query rows per kv head the scores are kept
constexpr int kWindowChunk = 1024;  // positions of a CTA where they are formed twice
constexpr float kWeightNegBig = -1.0e30f;

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
    float* score;    // [batch][Hkv][max_kvlen][score_rows]: raw scores, -inf where hidden; up to kScoreRows rows
    int32_t score_rows;
    uint32_t* status;
    CacheGeom geom;
    int64_t max_seqlen, max_kvlen, max_tokens, total_tokens;
    int32_t num_heads, num_kv_heads, group, causal, chunks;
    int32_t chunk;   // positions of a chunk
    float scale_log2;
};

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
    bool cut = s.tok0 < 0 || n < 0 || n > a.total_tokens - s.tok0;  // not rows of the query: no tokens
    n = cut ? 0 : n;
    cut = cut || n > a.max_seqlen;
    n = n > a.max_seqlen ? a.max_seqlen : n;
    s.start = a.start_pos[b];
    if (s.start < 0) {  // no such position: no tokens
        cut = cut || n > 0;
        n = 0;
    }
    if (s.start > a.max_kvlen - n) {
        s.start = s.start > a.max_kvlen ? a.max_kvlen : s.start;
        cut = cut || n > 0;
    }
    int64_t len = s.start + n;
    len = len > a.max_kvlen ? a.max_kvlen : len;
    if (cut && threadIdx.x == 0) {
        atomicOr(a.status, kDevLengthClamped);
    }
    s.rows = static_cast<int32_t>(n) * a.group;
    s.len = n > 0 ? static_cast<int32_t>(len) : 0;
    return s;
}

// Maximum and reciprocal sum of row `at` over its chunks; all lanes of a warp call it.
__device__ __forceinline__ float2 join_chunks(const WeightArgs& a, int64_t at, int32_t chunks, int lane) {
    float m = kWeightNegBig, l = 0.0f;
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

// One addition to a weight; nothing waits for it (measured against atomicAdd: 150 against 890 cycles per 64 positions).
__device__ __forceinline__ void add_weight(float* w, float x) {
    asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(w), "f"(x) : "memory");
}

// More than kScoreRows query rows per kv head: statistics, join and weights (attn_window.cu).
int launch_weight_window(const pplb200_attn_params& p, WeightArgs a, cudaStream_t stream);

}  // namespace pplb200
