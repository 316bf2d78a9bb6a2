// int4_tile.h — sixteen rows of one kv head quantised into a 4-bit pool by a 256-thread workgroup: the
// step that gg_kv_append and gg_qk_norm_rope_append share.
//
// LPR lanes hold a row, two runs of four dims each (16 rows of one head at LPR 16, of two heads at 8;
// at 32 two rounds of eight rows). FULL: head_dim is 8 * LPR; else it is a smaller one of whole eights,
// and the lanes past it hold nothing. Sixteen rows that are one block in order meet in LDS, and the block's
// K tile, V tile (a byte to a token) and words go out in 16-byte runs, whole lines; other rows go out
// two bytes of K and single bytes of V at a time, each a partial line. Workgroups of one row group are
// neighbours, so that whole source rows are read at a time.
#pragma once
#include "int4.h"
#include "lanes.h"

#include <type_traits>

namespace gg {

constexpr int int4_tile_head_group(int head_dim) { return head_dim <= 64 ? 2 : 1; }  // heads of a workgroup
// (head_dims of whole eights up to 256)
constexpr bool int4_tile_dim(int head_dim) { return head_dim % 8 == 0 && head_dim <= 256; }
// Groups of sixteen rows: one more than the rows fill, as the first block may be entered anywhere.
inline unsigned int4_tile_groups(int n_rows) { return (unsigned)((n_rows + 15 + 15) / 16); }
inline unsigned int4_tile_heads(int heads, int head_dim) {
    const int g = int4_tile_head_group(head_dim);
    return (unsigned)((heads + g - 1) / g);
}

// Calls f with the type as a constant.
template <class F>
inline void with_float(gg_dtype_t t, F f) {
    switch (t) {
        case GG_DTYPE_F32: f(std::integral_constant<gg_dtype_t, GG_DTYPE_F32>{}); break;
        case GG_DTYPE_F16: f(std::integral_constant<gg_dtype_t, GG_DTYPE_F16>{}); break;
        default: f(std::integral_constant<gg_dtype_t, GG_DTYPE_BF16>{}); break;
    }
}

#ifdef __HIPCC__
template <int LPR>
struct Int4Tile {
    static constexpr int kD = 8 * LPR;
    static constexpr int kHeads = LPR == 8 ? 2 : 1;
    __align__(16) uint8_t kv[kHeads][kD * 16];  // K tile, V tile (head_dim * 8 bytes each)
    __align__(16) uint32_t words[kHeads][16];
};

// Four codes in 16 bits.
__device__ __forceinline__ uint32_t int4_codes4(const float (&x)[4], const Int4Scale& p) {
    return int4_code(x[0], p) | (int4_code(x[1], p) << 4) | (int4_code(x[2], p) << 8) | (int4_code(x[3], p) << 12);
}

// A unit of a row as it was loaded: two runs of the key and two of the value.
template <gg_dtype_t T>
struct Int4Raw {
    Raw4<T> ka, kb, va, vb;
};

// Group `group` of rows and head group `hg`. fetch(r, h, u) loads row r, head h, unit u (an Int4Raw): the
// key's runs of dims oa .. oa + 3 and ob .. ob + 3 and the value's of 4u .. and D/2 + 4u .. ; it is
// called before the row's slot is known. make(raw, r, h, u, ka, kb, va, vb, oa, ob) gives the values to be
// stored, called with every lane of a row or none.
template <gg_dtype_t T, int LPR, bool FULL, class FETCH, class MAKE>
__device__ __forceinline__ void int4_tile_rows(const Int4View& p, const int32_t* slots, int n_rows, int group, int hg,
                                               Int4Tile<LPR>& tile, FETCH fetch, MAKE make) {
    constexpr int kRows = 256 / LPR;
    const int D = FULL ? Int4Tile<LPR>::kD : p.D;
    constexpr int kRounds = LPR == 32 ? 2 : 1;
    // A prompt's groups start where its blocks do (rows that are not a prompt's may be grouped anyhow).
    const int s0 = slots[0];
    const int r0 = group * 16 - (s0 < 0 ? 0 : s0 % p.bs % 16);
    const int u = threadIdx.x % LPR;
    const bool live = FULL || 8 * u < D;
    Int4Raw<T> raw[kRounds];
    int slot_of[kRounds];
    const int lead = slots[min(max(r0, 0), n_rows - 1)];
    bool in_order = p.bs == 16 && r0 >= 0 && lead >= 0 && lead % 16 == 0;
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
        const int i = round * kRows + threadIdx.x / LPR, r = r0 + (i & 15), h = hg * Int4Tile<LPR>::kHeads + (i >> 4);
        slot_of[round] = slots[min(max(r, 0), n_rows - 1)];
        if constexpr (!FULL) raw[round] = Int4Raw<T>{};
        if (live) raw[round] = fetch(min(max(r, 0), n_rows - 1), min(h, p.Hkv - 1), u);
    }
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
        const int row = (round * kRows + (int)threadIdx.x / LPR) & 15, r = r0 + row;
        if (r < 0 || r >= n_rows) slot_of[round] = -1;
        in_order = in_order && slot_of[round] == lead + row;
    }
    const bool whole = __syncthreads_and(in_order && lead + 15 < p.num_slots) != 0;
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
        const int i = round * kRows + threadIdx.x / LPR, row = i & 15, hl = i >> 4;
        const int r = r0 + row, h = hg * Int4Tile<LPR>::kHeads + hl;
        const int slot = h < p.Hkv ? slot_of[round] : -1;
        if (slot >= 0 && slot < p.num_slots) {
            float ka[4], kb[4], va[4], vb[4];
            int oa, ob;
            make(raw[round], r, h, u, ka, kb, va, vb, oa, ob);
            Int4Extremes kx, vx;
            auto extremes = [&] {
                kx = vx = Int4Extremes{};
                kx.take(ka[0], ka[1]), kx.take(ka[2], ka[3]), kx.take(kb[0], kb[1]), kx.take(kb[2], kb[3]);
                vx.take(va[0], va[1]), vx.take(va[2], va[3]), vx.take(vb[0], vb[1]), vx.take(vb[2], vb[3]);
            };
            extremes();
            if (__builtin_expect(__any(kx.replaced() || vx.replaced()), 0)) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    ka[e] = int4_clean(ka[e]), kb[e] = int4_clean(kb[e]), va[e] = int4_clean(va[e]), vb[e] = int4_clean(vb[e]);
                extremes();
            }
            auto scale = [](const Int4Extremes& x) {
                return int4_scale(__uint_as_float(group_max_int<LPR>(x.lo)), __uint_as_float((uint32_t)group_max_int<LPR>(x.hi)));
            };
            const Int4Scale ks = scale(kx), vs = scale(vx);
            const int blk = slot / p.bs, off = slot % p.bs;
            const uint32_t k01 = int4_codes4(ka, ks), k23 = int4_codes4(kb, ks), word = ks.half | (vs.half << 16);
            uint32_t vb4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) vb4[e] = int4_code(va[e], vs) | (int4_code(vb[e], vs) << 4);
            if (!live) continue;
            if (whole) {
                *(uint16_t*)&tile.kv[hl][row * (D / 2) + oa / 2] = (uint16_t)k01;
                *(uint16_t*)&tile.kv[hl][row * (D / 2) + ob / 2] = (uint16_t)k23;
#pragma unroll
                for (int e = 0; e < 4; ++e) tile.kv[hl][8 * D + (4 * u + e) * 16 + row] = (uint8_t)vb4[e];
                if (u == 0) tile.words[hl][row] = word;
            } else {
                uint8_t* kt = p.kc + p.tile0(blk, h) + (size_t)off * (D / 2);
                *(uint16_t*)(kt + oa / 2) = (uint16_t)k01;
                *(uint16_t*)(kt + ob / 2) = (uint16_t)k23;
                uint8_t* vt = p.vc + p.tile0(blk, h) + off;
#pragma unroll
                for (int e = 0; e < 4; ++e) vt[(size_t)(4 * u + e) * p.bs] = (uint8_t)vb4[e];
                if (u == 0) p.words[p.word(blk, h, off)] = word;
            }
        }
    }
    if (!whole) return;
    __syncthreads();
    // (The two tiles are neighbours in the pool.)
    for (int i = threadIdx.x; i < Int4Tile<LPR>::kHeads * (D + 4); i += 256) {
        const int hl = i / (D + 4), j = i % (D + 4), h = hg * Int4Tile<LPR>::kHeads + hl;
        if (h >= p.Hkv) break;
        if (j < D) *(uint4*)(p.kc + p.tile0(lead / 16, h) + (size_t)j * 16) = *(const uint4*)&tile.kv[hl][j * 16];
        else ((uint4*)(p.words + p.word(lead / 16, h, 0)))[j - D] = ((const uint4*)tile.words[hl])[j - D];
    }
}
#endif

}  // namespace gg
