// From INT8 cache rows to the swizzled fp16 tiles of a tcgen05 operand: the tensor copy of a raw block (codes and scales
// of 64 rows of one head) into shared memory, and the four converter warps' share of it.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "tensor_map.h"

namespace pplb200 {

constexpr int kTileRows = 64;  // cache rows of a block

// 16 codes -> 16 halves of value, scaled by two groups' scales (s = scale of channels 0..7 | 8..15 << 16)
__device__ __forceinline__ void dequant16(const uint4& c, uint32_t s, uint4& lo, uint4& hi) {
    const __half2 s0 = u32_as_h2(prmt(s, 0u, 0x1010u)), s1 = u32_as_h2(prmt(s, 0u, 0x3232u));
    const uint32_t x0 = c.x ^ 0x80808080u, x1 = c.y ^ 0x80808080u, x2 = c.z ^ 0x80808080u, x3 = c.w ^ 0x80808080u;
    lo.x = h2_as_u32(__hmul2(biased_bytes_to_half2<0x5140u>(x0), s0));
    lo.y = h2_as_u32(__hmul2(biased_bytes_to_half2<0x5342u>(x0), s0));
    lo.z = h2_as_u32(__hmul2(biased_bytes_to_half2<0x5140u>(x1), s0));
    lo.w = h2_as_u32(__hmul2(biased_bytes_to_half2<0x5342u>(x1), s0));
    hi.x = h2_as_u32(__hmul2(biased_bytes_to_half2<0x5140u>(x2), s1));
    hi.y = h2_as_u32(__hmul2(biased_bytes_to_half2<0x5342u>(x2), s1));
    hi.z = h2_as_u32(__hmul2(biased_bytes_to_half2<0x5140u>(x3), s1));
    hi.w = h2_as_u32(__hmul2(biased_bytes_to_half2<0x5342u>(x3), s1));
}

// 16 codes -> 16 halves of fp16(code * scale) and the 16 exact remainders (of a product of a 7-bit and an 11-bit number)
__device__ __forceinline__ void split16(const uint4& c, uint32_t s, uint4& lo, uint4& hi, uint4& lo_rest, uint4& hi_rest) {
    const __half2 s0 = u32_as_h2(prmt(s, 0u, 0x1010u)), s1 = u32_as_h2(prmt(s, 0u, 0x3232u));
    auto split = [](uint32_t word, __half2 sc, uint32_t& k0, uint32_t& k1, uint32_t& e0, uint32_t& e1) {
        const uint32_t x = word ^ 0x80808080u;
        const __half2 c0 = biased_bytes_to_half2<0x5140u>(x), c1 = biased_bytes_to_half2<0x5342u>(x);
        const __half2 p0 = __hmul2(c0, sc), p1 = __hmul2(c1, sc);
        k0 = h2_as_u32(p0);
        k1 = h2_as_u32(p1);
        e0 = h2_as_u32(__hfma2(c0, sc, __hneg2(p0)));
        e1 = h2_as_u32(__hfma2(c1, sc, __hneg2(p1)));
    };
    split(c.x, s0, lo.x, lo.y, lo_rest.x, lo_rest.y);
    split(c.y, s0, lo.z, lo.w, lo_rest.z, lo_rest.w);
    split(c.z, s1, hi.x, hi.y, hi_rest.x, hi_rest.y);
    split(c.w, s1, hi.z, hi.w, hi_rest.z, hi_rest.w);
}

__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// One thread's share of a raw K or V block: 16-byte piece `piece` of the rows row, row + kRowsPerStep, ..
template <int DH>
struct Raw {
    static constexpr int kPieces = DH / 16;            // 16-byte pieces of a row
    static constexpr int kRowsPerStep = 32 / kPieces;  // rows of a warp at once
    static constexpr int kRows = 16 / kRowsPerStep;    // steps over the warp's 16 rows
    uint4 code[kRows];
    uint32_t sc[kRows];

    __device__ __forceinline__ void load(uint32_t raw, int32_t row, int32_t piece, int32_t rows) {
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int32_t r = row + k * kRowsPerStep;
            const int32_t chunk = DH == 128 ? piece ^ (r & 7) : piece;  // as the 128-byte swizzle of the copy left it
            code[k] = lds128(raw + r * DH + chunk * 16);
            sc[k] = lds32(raw + kTileRows * DH + r * (DH / 4) + piece * 4);
            if (r >= rows) {  // rows behind the sequence's end may hold anything
                code[k] = make_uint4(0u, 0u, 0u, 0u);
                sc[k] = 0u;
            }
        }
    }

    // -> the swizzled fp16 tile at `tile`: [64 rows][64 halves] blocks, 16-byte chunk c of row r at chunk c ^ (r & 7)
    __device__ __forceinline__ void store(uint32_t tile, int32_t row, int32_t piece) const {
        const int32_t cb = piece >> 2, c = (piece & 3) * 2;
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int32_t r = row + k * kRowsPerStep;
            const uint32_t at = tile + cb * (kTileRows * 128) + r * 128;
            uint4 lo, hi;
            dequant16(code[k], sc[k], lo, hi);
            const uint32_t c0 = at + ((c ^ (r & 7)) << 4), c1 = at + (((c + 1) ^ (r & 7)) << 4);
            // the two column blocks start with different chunks: eight lanes then fill all banks once
            const bool odd = cb != 0;
            sts128(odd ? c1 : c0, odd ? hi : lo);
            sts128(odd ? c0 : c1, odd ? lo : hi);
        }
    }

    // The same with the remainders in a second tile at `rest`
    __device__ __forceinline__ void store_split(uint32_t tile, uint32_t rest, int32_t row, int32_t piece) const {
        const int32_t cb = piece >> 2, c = (piece & 3) * 2;
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int32_t r = row + k * kRowsPerStep;
            const uint32_t at = cb * (kTileRows * 128) + r * 128;
            uint4 lo, hi, lo_rest, hi_rest;
            split16(code[k], sc[k], lo, hi, lo_rest, hi_rest);
            const uint32_t c0 = at + ((c ^ (r & 7)) << 4), c1 = at + (((c + 1) ^ (r & 7)) << 4);
            const bool odd = cb != 0;
            sts128(tile + (odd ? c1 : c0), odd ? hi : lo);
            sts128(tile + (odd ? c0 : c1), odd ? lo : hi);
            sts128(rest + (odd ? c1 : c0), odd ? hi_rest : lo_rest);
            sts128(rest + (odd ? c0 : c1), odd ? lo_rest : hi_rest);
        }
    }
};

// One head's cache rows from `row` on, K (0) or V (1), by a tensor copy whose box says how many
__device__ __forceinline__ void load_rows(void* dst, const CUtensorMap* map, uint64_t* bar, const CacheMapOrder& order,
                                          int row, int head, int kv, int64_t layer) {
    int c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = i + 1;
        c[i] = order.pos_row == pos ? row : (order.pos_head == pos ? head : (order.pos_kv == pos ? kv : static_cast<int>(layer)));
    }
    tma_load_5d(dst, map, bar, 0, c[0], c[1], c[2], c[3]);
}

// A thread has stored its share of the operand tiles at `full` and is done with the raw slot of `empty`.  The proxy fence
// orders both for what comes next: the stores ahead of the MMAs that read the tiles, and the loads from the slot ahead of
// the tensor copy that overwrites it.  (An arrival behind a fence of ordinary accesses alone lets such a copy overtake the
// loads: seen as wrong scores in up to half of the runs of a busy kernel.)
__device__ __forceinline__ void hand_over(uint64_t* full, uint64_t* empty) {
    fence_proxy_async_smem();
    mbar_arrive(empty);
    mbar_arrive(full);
}

}  // namespace pplb200
