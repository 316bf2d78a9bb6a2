// int4.h — the 4-bit code of PER_TOKEN pools: a row's scale and zero point, and its codes.
//
// Of a row x (fp32; NaN as 0, |x| at most 1e36): lo = min(0, x), hi = max(0, x), s = (hi - lo) / 15
// rounded up to five significant bits, z = rint(-lo / s), n = rint(x / s) + z clamped to 0..15,
// and n stands for s * (n - z). Zero lies in the range and z is a whole number, so zero is exact;
// a scale of five bits rounded up covers the range at a step at most 1/16 longer, and scale and
// zero point of K and V fit one 32-bit word per (token, head): 4.125 bits an element at
// head_dim 128. The quotients are those of correctly rounded division: rows of 8 or 11 significant
// bits meet exact ties often (x and s are short), and a tie decided by the rounding of a
// reciprocal would fall either way.
#pragma once
#include "gg_common.h"

namespace gg {

struct Int4Scale {
    float s, inv, z;  // inv: 1 / s, correctly rounded
    uint32_t half;    // the 16 bits kept of it
};

__device__ __forceinline__ float int4_clean(float x) {
    return x == x ? __builtin_amdgcn_fmed3f(x, -1e36f, 1e36f) : 0.f;
}

// x / s, correctly rounded: one Newton step on x * (1 / s). The remainder x - q s is exact (s has
// five significant bits), and no quotient of a 24-bit by a 5-bit number lies within 2^-34 of a
// midpoint between two fp32 numbers, while the corrected quotient is within 2^-45 of the true one.
__device__ __forceinline__ float int4_div(float x, const Int4Scale& p) {
    const float q = x * p.inv;
    return __builtin_fmaf(__builtin_fmaf(-q, p.s, x), p.inv, q);
}

// lo <= 0 <= hi: the row's extremes. The quotient by 15 as in int4_div; 1 / s from the hardware's
// reciprocal (1 ulp) and one Newton step, which gives the correctly rounded one for each of the sixteen
// significands s can have (the codes of rows with every one of them are tested bit for bit).
__device__ __forceinline__ Int4Scale int4_scale(float lo, float hi) {
    Int4Scale p;
    const float d = hi - lo, q = d * (1.0f / 15.0f);
    const float r = __builtin_fmaf(__builtin_fmaf(-q, 15.0f, d), 1.0f / 15.0f, q);
    p.s = fmaxf(__uint_as_float((__float_as_uint(r) + 0x7ffffu) & 0xfff80000u), 0x1p-100f);
    const float y = __builtin_amdgcn_rcpf(p.s);
    p.inv = __builtin_fmaf(__builtin_fmaf(-p.s, y, 1.0f), y, y);
    p.z = __builtin_rintf(int4_div(-lo, p));
    p.half = ((__float_as_uint(p.s) >> 19) << 4) | (uint32_t)(int)p.z;
    return p;
}

// (x: int4_clean, within the row's extremes, so that rint(x / s) + z is 0 at least and 16 at most. Adding
// 1.5 * 2^23 rounds a quotient below 2^22 to a whole number, ties to even, and leaves it in the low bits.)
__device__ __forceinline__ uint32_t int4_code(float x, const Int4Scale& p) {
    const uint32_t n = __float_as_uint(int4_div(x, p) + 12582912.0f);
    return min(n + ((uint32_t)(int)p.z - 0x4b400000u), 15u);
}

// The extremes of a row by whole-number maxima: positive floats order as signed integers and are
// above all negative ones, negative floats order as unsigned integers and are above all positive ones.
// (fminf and fmaxf quiet each operand first, and are not merged with the lane exchanges.) A NaN or a
// value past 1e36 comes out past its bound: `replaced`.
struct Int4Extremes {
    int hi = 0;                    // 0.0
    uint32_t lo = 0x80000000u;     // -0.0
    __device__ __forceinline__ void take(float a, float b) {
        hi = max(hi, max((int)__float_as_uint(a), (int)__float_as_uint(b)));
        lo = max(lo, max(__float_as_uint(a), __float_as_uint(b)));
    }
    __device__ __forceinline__ bool replaced() const { return hi > 0x7b4097ce || lo > 0xfb4097ceu; }  // 1e36f, -1e36f
};

// A token's word: K in the low half, V in the high half.
__device__ __forceinline__ float int4_k_scale(uint32_t w) { return __uint_as_float((w & 0xfff0u) << 15); }
__device__ __forceinline__ float int4_v_scale(uint32_t w) { return __uint_as_float((w >> 1) & 0x7ff80000u); }
__device__ __forceinline__ int int4_k_zero(uint32_t w) { return (int)(w & 15u); }
__device__ __forceinline__ int int4_v_zero(uint32_t w) { return (int)((w >> 16) & 15u); }

// One layer of a 4-bit pool.
struct Int4View {
    uint8_t* kc;      // K tile of (block 0, head 0): [bs][D / 2], byte i = dims 2i, 2i + 1
    uint8_t* vc;      // V tile: [D / 2][bs], byte (i, t) = dims i, i + D / 2 of token t
    uint32_t* words;  // [blocks][Hkv][bs]
    int Hkv, D, bs;
    long long num_slots;

    __device__ __forceinline__ size_t tile0(int blk, int h) const { return ((size_t)blk * Hkv + h) * ((size_t)bs * D); }
    __device__ __forceinline__ size_t word(int blk, int h, int off) const { return ((size_t)blk * Hkv + h) * bs + off; }
};

__device__ __forceinline__ float wave_min(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fminf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// A whole wave quantises one row, kx(d) and vx(d) giving element d (any even head_dim), and writes
// it to offset `off` of block `blk`, head h.
template <class KX, class VX>
__device__ __forceinline__ void int4_write_row(const Int4View& p, int blk, int h, int off, KX kx, VX vx) {
    const int lane = threadIdx.x & 63, half = p.D / 2;
    float klo = 0.f, khi = 0.f, vlo = 0.f, vhi = 0.f;
    for (int i = lane; i < p.D; i += 64) {
        const float k = int4_clean(kx(i)), v = int4_clean(vx(i));
        klo = fminf(klo, k);
        khi = fmaxf(khi, k);
        vlo = fminf(vlo, v);
        vhi = fmaxf(vhi, v);
    }
    const Int4Scale ks = int4_scale(wave_min(klo), wave_max(khi)), vs = int4_scale(wave_min(vlo), wave_max(vhi));
    uint8_t* kt = p.kc + p.tile0(blk, h) + (size_t)off * half;
    uint8_t* vt = p.vc + p.tile0(blk, h) + off;
    for (int i = lane; i < half; i += 64) {
        kt[i] = (uint8_t)(int4_code(int4_clean(kx(2 * i)), ks) | (int4_code(int4_clean(kx(2 * i + 1)), ks) << 4));
        vt[(size_t)i * p.bs] = (uint8_t)(int4_code(int4_clean(vx(i)), vs) | (int4_code(int4_clean(vx(i + half)), vs) << 4));
    }
    if (lane == 0) p.words[p.word(blk, h, off)] = ks.half | (vs.half << 16);
}

inline Int4View int4_view(const KV* kv, int layer) {
    Int4View v{};
    v.kc = kv->k_pool + (size_t)layer * kv->layer_stride;
    v.vc = kv->v_pool + (size_t)layer * kv->layer_stride;
    v.words = (uint32_t*)kv->k_scales + (size_t)layer * kv->scale_layer_elems;
    v.Hkv = kv->num_kv_heads;
    v.D = kv->head_dim;
    v.bs = kv->block_size;
    v.num_slots = (long long)kv->num_blocks * kv->block_size;
    return v;
}

}  // namespace gg
