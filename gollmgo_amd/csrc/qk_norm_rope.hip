// qk_norm_rope.hip — norm of each query and key head and the rotation of its positions, in one pass;
// keys to a dense output or, with the values, to a cache.
//
// Bound: each element is read and written once and costs about ten operations, so a prompt is bound by
// memory and a step's few rows by the launch. The angle is the dear part (40 instructions in 64 bits a
// pair) and belongs to a row, not to a head: lanes hold the same pairs for every head they go through
// and form their angles once. bf16, heads of 128, kernel time: 32768 rows of 32 + 8 heads, three position
// axes, 671 MB 126.5 µs, 5.3 TB/s; 8192 rows with keys and values into a 4-bit pool, 177 MB 36.1 µs,
// 4.9 TB/s; five rows 3.7 µs. Where pairs are not whole fours or rows are unaligned, a wave to a row and
// head forms its own angles: 8192 rows of 40 heads 240 µs against 29.
#include "gg_common.h"
#include "int4.h"
#include "int4_tile.h"
#include "lanes.h"

namespace gg {
namespace {

constexpr int kRowsMaxD = 1024;
constexpr int kRopeWaves = 4096;  // waves that fill the machine (heads_per_wave)

// cos and sin of position times frequency, in 64 bits to the last step: the angle in turns, its whole and
// quarter turns taken off (at position 2^31 the product still keeps 2^-21 of a turn), then the Taylor sums
// on [-pi/4, pi/4], whose remainders are below 2^-33. Rounded once, to fp32; fp64 runs at fp32's rate here.
__device__ __forceinline__ void turn_of(int pos, float freq, float& c, float& s) {
    constexpr double kTurn = 0.15915494309189533577, kRadians = 6.283185307179586477;  // 1 / (2 pi), 2 pi
    double t = (double)pos * ((double)freq * kTurn);
    t -= __builtin_rint(t);
    const double quarter = __builtin_rint(4.0 * t);
    const double x = __builtin_fma(quarter, -0.25, t) * kRadians, y = x * x;
    double u = __builtin_fma(y, -1.0 / 39916800.0, 1.0 / 362880.0);
    u = __builtin_fma(y, u, -1.0 / 5040.0);
    u = __builtin_fma(y, u, 1.0 / 120.0);
    u = __builtin_fma(y, u, -1.0 / 6.0);
    const float sx = (float)__builtin_fma(x * y, u, x);
    double v = __builtin_fma(y, -1.0 / 3628800.0, 1.0 / 40320.0);
    v = __builtin_fma(y, v, -1.0 / 720.0);
    v = __builtin_fma(y, v, 1.0 / 24.0);
    v = __builtin_fma(y, v, -0.5);
    const float cx = (float)__builtin_fma(y, v, 1.0);
    const int n = (int)quarter;  // -2 .. 2
    c = n & 1 ? sx : cx;
    s = n & 1 ? cx : sx;
    c = (n + 1) & 2 ? -c : c;
    s = n & 2 ? -s : s;
}

// 1 / sqrt(m): the fp32 function's (1 ulp) and a Newton step in 64 bits, rounded once.
__device__ __forceinline__ float inv_sqrt(float m) {
    const double y = (double)rsqrtf(m);
    return m > 0.f && m < INFINITY ? (float)(y * __builtin_fma((double)m * y, -0.5 * y, 1.5)) : (float)y;
}

// A normed element, and a pair turned: every kernel here rounds the same products in the same order, one
// by one and not fused. A 4-bit code turns on the last bit of its key, so the keys are those of the
// formula evaluated in fp32 step by step, with exact angles and norms: of 33.5 M codes of 32 k rows none
// differs from that (fp32 sine and cosine, fused products and the hardware's 1 / sqrt: one in 7 M, and
// one bf16 output in 26 k), in the same time.
__device__ __forceinline__ float normed(float x, float r, float w) {
#pragma clang fp contract(off)
    return x * r * w;
}
__device__ __forceinline__ void turn_pair(float& p, float& q, float c, float s) {
#pragma clang fp contract(off)
    const float x = p * c - q * s, y = q * c + p * s;
    p = x;
    q = y;
}

__device__ __forceinline__ int pair_axis(const RopeArgs& a, int j) { return (a.axis[j >> 3] >> (4 * (j & 7))) & 15; }

__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Where keys and values go when they are cached.
struct PoolOut {
    Int4View i4;            // 4-bit pools
    gg_dtype_t dt;
    uint8_t* kc;
    uint8_t* vc;
    const float* k_inv;     // FP8: 1 / per-head scale
    const float* v_inv;
    int bs;
    long long num_slots;
};

__device__ __forceinline__ void pool_store(uint8_t* base, gg_dtype_t dt, size_t i, float x, float inv) {
    if (dt == GG_DTYPE_FP8_E4M3) base[i] = f32_to_fp8e4m3_sat(x * inv);
    else store_from_f32(base, dt, i, x);
}

// One wave per (row, head): any head_dim, pair count, style and alignment. The turned row goes
// through LDS only where it is written to a 4-bit pool, whose scale needs all of it.
__device__ __forceinline__ void rows_wave(const RopeArgs& a, const PoolOut& p, int t, int hh, float* s_row) {
    const int lane = threadIdx.x & 63, D = a.D, P = a.pairs;
    const bool is_q = hh < a.Hq;
    const int h = is_q ? hh : hh - a.Hq;
    const void* src = is_q ? a.q : a.k;
    const void* weight = is_q ? a.q_weight : a.k_weight;
    const size_t at = (size_t)t * (is_q ? a.q_stride : a.k_stride) + (size_t)h * D;
    float norm = 1.f;
    if (weight) {
        float sum = 0.f;
        for (int d = lane; d < D; d += 64) {
            const float x = load_as_f32(src, a.dt, at + d);
            sum = __builtin_fmaf(x, x, sum);
        }
        norm = inv_sqrt(wave_sum(sum) / (float)D + a.eps);
    }
    const bool cached = !is_q && !a.k_out;
    int blk = 0, off = 0;
    if (cached) {
        const int slot = a.slots[t];
        if (slot < 0 || slot >= p.num_slots) return;
        blk = slot / p.bs;
        off = slot % p.bs;
    }
    const bool to_int4 = cached && p.dt == GG_DTYPE_INT4;
    void* out = is_q ? a.q_out : a.k_out;
    const size_t to = ((size_t)t * (is_q ? a.Hq : a.Hkv) + h) * D;
    const size_t tile = ((size_t)blk * a.Hkv + h) * (2 * (size_t)p.bs * D);
    const float kinv = cached && p.dt == GG_DTYPE_FP8_E4M3 ? p.k_inv[h] : 1.f;
    auto value = [&](int d) {
        const float x = load_as_f32(src, a.dt, at + d);
        return weight ? normed(x, norm, load_as_f32(weight, a.dt, d)) : x;
    };
    auto put = [&](int d, float y) {
        if (to_int4) s_row[d] = y;
        else if (cached) pool_store(p.kc, p.dt, tile + (size_t)off * D + d, y, kinv);
        else store_from_f32(out, a.dt, to + d, y);
    };
    for (int u = lane; u < D - P; u += 64) {
        if (u >= P) {
            put(P + u, value(P + u));
            continue;
        }
        const int da = a.style == GG_ROPE_PAIRS ? 2 * u : u, db = a.style == GG_ROPE_PAIRS ? 2 * u + 1 : u + P;
        float c, s;
        turn_of(a.positions[(size_t)pair_axis(a, u) * a.n + t], a.inv_freq[u], c, s);
        float x = value(da), y = value(db);
        turn_pair(x, y, c, s);
        put(da, x);
        put(db, y);
    }
    if (!cached) return;
    const size_t vat = (size_t)t * a.v_stride + (size_t)h * D;
    if (to_int4) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        int4_write_row(p.i4, blk, h, off, [&](int d) { return s_row[d]; },
                       [&](int d) { return load_as_f32(a.v, a.dt, vat + d); });
    } else {
        const float vinv = p.dt == GG_DTYPE_FP8_E4M3 ? p.v_inv[h] : 1.f;
        for (int d = lane; d < D; d += 64)
            pool_store(p.vc, p.dt, tile + (size_t)d * p.bs + off, load_as_f32(a.v, a.dt, vat + d), vinv);
    }
}

__global__ void __launch_bounds__(256) qk_norm_rope_rows_kernel(RopeArgs a, PoolOut p) {
    __shared__ float s_row[4][kRowsMaxD];
    const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int heads = a.Hq + a.Hkv;
    if (i < (long long)a.n * heads) rows_wave(a, p, (int)(i / heads), (int)(i % heads), s_row[threadIdx.x >> 6]);
}

// ---- head_dims of whole eights up to 256: LPR lanes a row, eight dims a lane ----
//
// Lane u of a row holds two runs of four dims, at oa and ob, loaded and stored as vectors:
//   HALVES, u < P / 4 : dims 4u .. and P + 4u .. (pairs 4u .. 4u + 3, both ends in the lane)
//   PAIRS,  u < P / 4 : dims 8u .. and 8u + 4 .. (the same pairs)
//   past the pairs    : eight dims that only the norm touches
struct Unit {
    int oa, ob;
    bool live, turned;
};
__device__ __forceinline__ Unit unit_of(const RopeArgs& a, int u) {
    const int P = a.pairs;
    Unit x;
    x.live = 8 * u < a.D;
    x.turned = 4 * u < P;
    const bool halves = a.style == GG_ROPE_HALVES && x.turned;
    x.oa = halves ? 4 * u : 8 * u;
    x.ob = halves ? P + 4 * u : 8 * u + 4;
    return x;
}
// Pairs 4u .. 4u + 3 of row t (c = 1, s = 0 past the pairs). Positions and frequencies are all asked for
// before the first angle is formed.
struct Turn {
    float c[4], s[4];
};
__device__ __forceinline__ Turn turn4(const RopeArgs& a, const Unit& x, int u, int t) {
    Turn r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        r.c[e] = 1.f;
        r.s[e] = 0.f;
    }
    if (!x.turned) return r;
    const float4 f = *(const float4*)(a.inv_freq + 4 * u);
    int pos[4];
    if (a.axes == 1) {
        pos[0] = pos[1] = pos[2] = pos[3] = a.positions[t];
    } else {
        const uint32_t ax = a.axis[u >> 1] >> (16 * (u & 1));
#pragma unroll
        for (int e = 0; e < 4; ++e) pos[e] = a.positions[(size_t)((ax >> (4 * e)) & 15u) * a.n + t];
    }
    const float freq[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) turn_of(pos[e], freq[e], r.c[e], r.s[e]);
    return r;
}
__device__ __forceinline__ void apply_turn(const RopeArgs& a, const Unit& x, const Turn& r, float (&fa)[4], float (&fb)[4]) {
    if (!x.turned) return;
    if (a.style == GG_ROPE_HALVES) {
#pragma unroll
        for (int e = 0; e < 4; ++e) turn_pair(fa[e], fb[e], r.c[e], r.s[e]);
    } else {
        turn_pair(fa[0], fa[1], r.c[0], r.s[0]);
        turn_pair(fa[2], fa[3], r.c[1], r.s[1]);
        turn_pair(fb[0], fb[1], r.c[2], r.s[2]);
        turn_pair(fb[2], fb[3], r.c[3], r.s[3]);
    }
}
// A row's two runs, normed (w: the weight's runs), by the row's LPR lanes together. The squares are summed
// by dim wherever a row's pairs are whole: four in sequence, then neighbours, neighbours of those and so
// on, which is as accurate as it is fixed. (Products of 16-bit types are exact, fused or not.)
template <gg_dtype_t T>
__device__ __forceinline__ float squares4(const float (&f)[4]) {
#pragma clang fp contract(off)
    if constexpr (T == GG_DTYPE_F32) return f[0] * f[0] + f[1] * f[1] + f[2] * f[2] + f[3] * f[3];
    else return __builtin_fmaf(f[3], f[3], __builtin_fmaf(f[2], f[2], __builtin_fmaf(f[1], f[1], f[0] * f[0])));
}
template <gg_dtype_t T, int LPR>
__device__ __forceinline__ void norm_runs(const RopeArgs& a, const float (&wa)[4], const float (&wb)[4], float (&fa)[4], float (&fb)[4]) {
    const float sa = squares4<T>(fa), sb = squares4<T>(fb);
    const float sum = a.style == GG_ROPE_HALVES ? group_sum<LPR>(sa) + group_sum<LPR>(sb) : group_sum<LPR>(sa + sb);
    const float r = inv_sqrt(__builtin_fmaf(sum, a.inv_d, a.eps));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        fa[e] = normed(fa[e], r, wa[e]);
        fb[e] = normed(fb[e], r, wb[e]);
    }
}
template <gg_dtype_t T>
__device__ __forceinline__ void weight_runs(const void* w, const Unit& x, float (&wa)[4], float (&wb)[4]) {
    to_f32<T>(load4<T>(w, x.oa), wa);
    to_f32<T>(load4<T>(w, x.ob), wb);
}

// Heads [h0, h1) of one side (queries or keys) of row t by one wave, 64 / LPR at a time, four steps in
// flight.
template <gg_dtype_t T, int LPR>
__device__ __forceinline__ void dense_side(const RopeArgs& a, const Unit& x, const Turn& r, const void* rows, long long stride,
                                           const void* weight, void* out, int heads, int t, int h0, int h1) {
    constexpr int kRPW = 64 / LPR, kAhead = 4;
    constexpr size_t kEB = T == GG_DTYPE_F32 ? 4 : 2;
    const int sub = (threadIdx.x & 63) / LPR;
    const uint8_t* src = (const uint8_t*)rows + ((size_t)t * stride + (size_t)(h0 + sub) * a.D) * kEB;
    uint8_t* dst = (uint8_t*)out + (((size_t)t * heads + h0 + sub) * a.D) * kEB;
    const int n = x.live ? h1 - h0 - sub : 0;  // the lane's heads: 0, kRPW, ... below n
    const size_t step = (size_t)kRPW * a.D * kEB;
    Raw4<T> ra[kAhead], rb[kAhead];
    auto fetch = [&](int i, int h) {
        ra[i].w = rb[i].w = make_uint4(0, 0, 0, 0);
        if (h < n) {
            ra[i] = load4<T>(src, x.oa);
            rb[i] = load4<T>(src, x.ob);
        }
        src += step;
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(i, i * kRPW);
    float wa[4] = {1.f, 1.f, 1.f, 1.f}, wb[4] = {1.f, 1.f, 1.f, 1.f};
    if (weight && x.live) weight_runs<T>(weight, x, wa, wb);
    for (int hb = 0; hb < h1 - h0; hb += kAhead * kRPW) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = hb + i * kRPW;
            if (h >= h1 - h0) break;
            float fa[4], fb[4];
            to_f32<T>(ra[i], fa);
            to_f32<T>(rb[i], fb);
            fetch(i, h + kAhead * kRPW);
            if (weight) norm_runs<T, LPR>(a, wa, wb, fa, fb);
            apply_turn(a, x, r, fa, fb);
            if (h < n) {
                store4<T>(dst, x.oa, fa);
                store4<T>(dst, x.ob, fb);
            }
            dst += step;
        }
    }
}

// Wave (t, part): heads [h0, h1) of row t; the first Hq heads are queries.
template <gg_dtype_t T, int LPR>
__device__ __forceinline__ void dense_wave(const RopeArgs& a, int t, int h0, int h1) {
    const int u = threadIdx.x % LPR;
    const Unit x = unit_of(a, u);
    const Turn r = turn4(a, x, u, t);
    if (h0 < a.Hq) dense_side<T, LPR>(a, x, r, a.q, a.q_stride, a.q_weight, a.q_out, a.Hq, t, h0, min(h1, a.Hq));
    if (h1 > a.Hq) dense_side<T, LPR>(a, x, r, a.k, a.k_stride, a.k_weight, a.k_out, a.Hkv, t, max(h0 - a.Hq, 0), h1 - a.Hq);
}

template <gg_dtype_t T, int LPR>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(RopeArgs a, int heads, int parts, int per) {
    const unsigned i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = (int)(i / parts), part = (int)(i % parts);
    if (t >= a.n) return;
    dense_wave<T, LPR>(a, t, part * per, min(heads, part * per + per));
}

// The same into a 4-bit pool: the first q_blocks workgroups do the queries as above, the others
// sixteen rows of a kv head (or two) each, as gg_kv_append does (int4_tile.h).
template <gg_dtype_t T, int LPR, bool FULL>
__global__ void __launch_bounds__(256) qk_norm_rope_int4_kernel(RopeArgs a, Int4View p, int q_blocks, int parts, int per,
                                                                int hg) {
    __shared__ Int4Tile<LPR> tile;
    if ((int)blockIdx.x < q_blocks) {
        const unsigned i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int t = (int)(i / parts), part = (int)(i % parts);
        if (t >= a.n) return;
        dense_wave<T, LPR>(a, t, part * per, min(a.Hq, part * per + per));
        return;
    }
    const int b = (int)blockIdx.x - q_blocks;
    float wa[4] = {1.f, 1.f, 1.f, 1.f}, wb[4] = {1.f, 1.f, 1.f, 1.f};
    const Unit x = unit_of(a, threadIdx.x % LPR);
    if (a.k_weight && (FULL || x.live)) weight_runs<T>(a.k_weight, x, wa, wb);
    int4_tile_rows<T, LPR, FULL>(
        p, a.slots, a.n, b / hg, b % hg, tile,
        [&](int t, int h, int u) {
            const size_t at = (size_t)t * a.k_stride + (size_t)h * a.D, vat = (size_t)t * a.v_stride + (size_t)h * a.D;
            return Int4Raw<T>{load4<T>(a.k, at + x.oa), load4<T>(a.k, at + x.ob), load4<T>(a.v, vat + 4 * u),
                              load4<T>(a.v, vat + a.D / 2 + 4 * u)};
        },
        [&](const Int4Raw<T>& w, int t, int, int u, float (&ka)[4], float (&kb)[4], float (&va)[4], float (&vb)[4], int& oa, int& ob) {
            const Turn r = turn4(a, x, u, t);
            to_f32<T>(w.ka, ka);
            to_f32<T>(w.kb, kb);
            to_f32<T>(w.va, va);
            to_f32<T>(w.vb, vb);
            if (a.k_weight) norm_runs<T, LPR>(a, wa, wb, ka, kb);
            apply_turn(a, x, r, ka, kb);
            oa = x.oa;
            ob = x.ob;
        });
}

// Into pools of one value an element (EB bytes): queries as above, sixteen rows of a kv head (two at LPR
// 8) per workgroup of the others. Where those are one block in order, its K and V tiles, neighbours in the
// pool, meet in LDS and go out in 16-byte runs; other rows go out in fours of K and single elements of V.
// (A V tile is [D][16]: a wave to a row and head wrote each of its values to a line of its own. 8192
// rows of 32 + 8 heads of 128, bf16 pool 69 -> 38 µs, FP8 67 -> 37.)
template <int LPR, int EB>
struct PoolTile {
    static constexpr int kHeads = LPR == 8 ? 2 : 1, kD = 8 * LPR;
    // V: four dims' runs, then 16 bytes not used (the runs of lanes then lie in other banks).
    __align__(16) uint8_t k[kHeads][16 * kD * EB];
    __align__(16) uint8_t v[kHeads][16 * kD * EB + kD / 4 * 16];
};
template <int EB>
__device__ __forceinline__ uint32_t pool_bits(gg_dtype_t dt, float x, float inv) {
    if constexpr (EB == 1) return f32_to_fp8e4m3_sat(x * inv);
    else if constexpr (EB == 2) return dt == GG_DTYPE_F16 ? f32_to_f16_bits(x) : f32_to_bf16_bits(x);
    else return __float_as_uint(x);
}
template <int EB>
__device__ __forceinline__ void put_bits(uint8_t* p, uint32_t x) {
    if constexpr (EB == 1) *p = (uint8_t)x;
    else if constexpr (EB == 2) *(uint16_t*)p = (uint16_t)x;
    else *(uint32_t*)p = x;
}
template <int EB>
__device__ __forceinline__ void put4(uint8_t* p, const uint32_t (&x)[4]) {
    if constexpr (EB == 1) *(uint32_t*)p = x[0] | (x[1] << 8) | (x[2] << 16) | (x[3] << 24);
    else if constexpr (EB == 2) *(uint2*)p = make_uint2(x[0] | (x[1] << 16), x[2] | (x[3] << 16));
    else *(uint4*)p = make_uint4(x[0], x[1], x[2], x[3]);
}

template <gg_dtype_t T, int LPR, int EB>
__global__ void __launch_bounds__(256) qk_norm_rope_tile_kernel(RopeArgs a, PoolOut p, int q_blocks, int parts, int per, int hg) {
    constexpr int kHeads = PoolTile<LPR, EB>::kHeads, kRows = 256 / LPR, kRounds = LPR == 32 ? 2 : 1;
    __shared__ PoolTile<LPR, EB> tile;
    if ((int)blockIdx.x < q_blocks) {
        const unsigned i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int t = (int)(i / parts), part = (int)(i % parts);
        if (t < a.n) dense_wave<T, LPR>(a, t, part * per, min(a.Hq, part * per + per));
        return;
    }
    const int group = ((int)blockIdx.x - q_blocks) / hg, h0 = ((int)blockIdx.x - q_blocks) % hg * kHeads;
    const int D = a.D, u = threadIdx.x % LPR;
    const Unit x = unit_of(a, u);
    // A prompt's groups start where its blocks do (rows that are not a prompt's may be grouped anyhow).
    const int s0 = a.slots[0];
    const int r0 = group * 16 - (s0 < 0 ? 0 : s0 % p.bs % 16);
    const int lead = a.slots[min(max(r0, 0), a.n - 1)];
    bool in_order = p.bs == 16 && r0 >= 0 && lead >= 0 && lead % 16 == 0;
    float wa[4] = {1.f, 1.f, 1.f, 1.f}, wb[4] = {1.f, 1.f, 1.f, 1.f};
    if (a.k_weight && x.live) weight_runs<T>(a.k_weight, x, wa, wb);
    Raw4<T> ka[kRounds], kb[kRounds], va[kRounds], vb[kRounds];
    int slot_of[kRounds];
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
        const int i = round * kRows + (int)threadIdx.x / LPR, r = r0 + (i & 15), h = min(h0 + (i >> 4), a.Hkv - 1);
        const int t = min(max(r, 0), a.n - 1);
        ka[round].w = kb[round].w = va[round].w = vb[round].w = make_uint4(0, 0, 0, 0);
        if (x.live) {
            const size_t at = (size_t)t * a.k_stride + (size_t)h * D, vat = (size_t)t * a.v_stride + (size_t)h * D + 8 * u;
            ka[round] = load4<T>(a.k, at + x.oa);
            kb[round] = load4<T>(a.k, at + x.ob);
            va[round] = load4<T>(a.v, vat);
            vb[round] = load4<T>(a.v, vat + 4);
        }
        slot_of[round] = r >= 0 && r < a.n ? a.slots[t] : -1;
        in_order = in_order && slot_of[round] == lead + (i & 15);
    }
    const bool whole = __syncthreads_and(in_order && lead + 15 < p.num_slots) != 0;
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
        const int i = round * kRows + (int)threadIdx.x / LPR, row = i & 15, hl = i >> 4, h = h0 + hl, slot = slot_of[round];
        if (h >= a.Hkv || slot < 0 || slot >= p.num_slots) continue;
        float fa[4], fb[4], ga[4], gb[4];
        to_f32<T>(ka[round], fa);
        to_f32<T>(kb[round], fb);
        to_f32<T>(va[round], ga);
        to_f32<T>(vb[round], gb);
        if (a.k_weight) norm_runs<T, LPR>(a, wa, wb, fa, fb);
        apply_turn(a, x, turn4(a, x, u, r0 + row), fa, fb);
        if (!x.live) continue;
        const float kinv = EB == 1 ? p.k_inv[h] : 1.f, vinv = EB == 1 ? p.v_inv[h] : 1.f;
        uint32_t k0[4], k1[4], v0[4], v1[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            k0[e] = pool_bits<EB>(p.dt, fa[e], kinv);
            k1[e] = pool_bits<EB>(p.dt, fb[e], kinv);
            v0[e] = pool_bits<EB>(p.dt, ga[e], vinv);
            v1[e] = pool_bits<EB>(p.dt, gb[e], vinv);
        }
        if (whole) {
            put4<EB>(&tile.k[hl][(row * D + x.oa) * EB], k0);
            put4<EB>(&tile.k[hl][(row * D + x.ob) * EB], k1);
            uint8_t* v = &tile.v[hl][8 * u * 16 * EB + 2 * u * 16 + row * EB];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                put_bits<EB>(v + e * 16 * EB, v0[e]);
                put_bits<EB>(v + (4 + e) * 16 * EB + 16, v1[e]);
            }
        } else {
            const int blk = slot / p.bs, off = slot % p.bs;
            const size_t t0 = ((size_t)blk * a.Hkv + h) * (2 * (size_t)p.bs * D);
            uint8_t* k = p.kc + (t0 + (size_t)off * D) * EB;
            put4<EB>(k + x.oa * EB, k0);
            put4<EB>(k + x.ob * EB, k1);
            uint8_t* v = p.vc + (t0 + (size_t)(8 * u) * p.bs + off) * EB;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                put_bits<EB>(v + (size_t)e * p.bs * EB, v0[e]);
                put_bits<EB>(v + (size_t)(4 + e) * p.bs * EB, v1[e]);
            }
        }
    }
    if (!whole) return;
    __syncthreads();
    const int runs = D * EB;  // of 16 bytes, in a tile
    for (int i = threadIdx.x; i < 2 * kHeads * runs; i += 256) {
        const int hl = i / (2 * runs), j = i % (2 * runs), h = h0 + hl;
        if (h >= a.Hkv) break;
        const int jv = j - runs;
        const uint4 w = j < runs ? *(const uint4*)&tile.k[hl][j * 16] : *(const uint4*)&tile.v[hl][(jv + jv / (4 * EB)) * 16];
        *(uint4*)(p.kc + (((size_t)(lead / 16) * a.Hkv + h) * (32 * (size_t)D)) * EB + (size_t)j * 16) = w;
    }
}

// Heads of a row for one wave: all of them where the rows alone fill the machine (one set of angles
// a row), else as few as bring the waves there.
int heads_per_wave(int n, int heads, int rows_per_wave) {
    const int steps = (heads + rows_per_wave - 1) / rows_per_wave;
    const int parts = n >= kRopeWaves ? 1 : (kRopeWaves + n - 1) / n;
    return (steps + parts - 1) / parts * rows_per_wave;
}

// Whether the vector kernels take the call.
bool vectors_fit(const RopeArgs& a) {
    const size_t align = a.dt == GG_DTYPE_F32 ? 16 : 8;
    const long long unit = (long long)(align / dtype_bytes(a.dt));
    auto ok = [&](const void* p) { return (uintptr_t)p % align == 0; };
    return a.D % 8 == 0 && a.D <= 256 && a.pairs % 4 == 0 && a.q_stride % unit == 0 && a.k_stride % unit == 0 &&
           a.v_stride % unit == 0 && ok(a.q) && ok(a.k) && ok(a.v) && ok(a.q_out) && ok(a.k_out) && ok(a.q_weight) &&
           ok(a.k_weight) && (uintptr_t)a.inv_freq % 16 == 0;
}

template <gg_dtype_t T, int LPR>
gg_status_t launch_vectors(const RopeArgs& a, const KV* kv, const PoolOut& p, hipStream_t s) {
    const int heads = kv ? a.Hq : a.Hq + a.Hkv;
    const int per = heads ? heads_per_wave(a.n, heads, 64 / LPR) : 1, parts = heads ? (heads + per - 1) / per : 0;
    const long long blocks = ((long long)a.n * parts + 3) / 4;
    const int hg = LPR == 8 ? (a.Hkv + 1) / 2 : a.Hkv;
    const long long all = blocks + (kv ? (long long)int4_tile_groups(a.n) * hg : 0);
    if (all > max_blocks_of(256)) return fail(GG_ERR_INVALID, "qk_norm_rope: too many rows for one call");
    const unsigned grid = (unsigned)all;
    const int some = parts > 0 ? parts : 1, qb = (int)blocks;
    if (!kv) qk_norm_rope_kernel<T, LPR><<<grid, 256, 0, s>>>(a, heads, some, per);
    else if (kv->dtype == GG_DTYPE_INT4 && a.D == 8 * LPR)
        qk_norm_rope_int4_kernel<T, LPR, true><<<grid, 256, 0, s>>>(a, p.i4, qb, some, per, hg);
    else if (kv->dtype == GG_DTYPE_INT4) qk_norm_rope_int4_kernel<T, LPR, false><<<grid, 256, 0, s>>>(a, p.i4, qb, some, per, hg);
    else if (kv->dtype == GG_DTYPE_F32) qk_norm_rope_tile_kernel<T, LPR, 4><<<grid, 256, 0, s>>>(a, p, qb, some, per, hg);
    else if (kv->dtype == GG_DTYPE_FP8_E4M3) qk_norm_rope_tile_kernel<T, LPR, 1><<<grid, 256, 0, s>>>(a, p, qb, some, per, hg);
    else qk_norm_rope_tile_kernel<T, LPR, 2><<<grid, 256, 0, s>>>(a, p, qb, some, per, hg);
    return check_hip(hipGetLastError(), "qk_norm_rope launch");
}

}  // namespace

gg_status_t launch_qk_norm_rope(const RopeArgs& a, KV* kv, int layer, hipStream_t s) {
    PoolOut p{};
    if (kv) {
        p.dt = kv->dtype;
        p.kc = kv->k_pool + (size_t)layer * kv->layer_stride;
        p.vc = kv->v_pool + (size_t)layer * kv->layer_stride;
        p.bs = kv->block_size;
        p.num_slots = (long long)kv->num_blocks * kv->block_size;
        if (kv->dtype == GG_DTYPE_INT4) p.i4 = int4_view(kv, layer);
        if (kv->scale_mode == GG_SCALE_PER_HEAD) {
            p.k_inv = (const float*)kv->k_scales + (size_t)layer * kv->scale_layer_elems + kv->num_kv_heads;
            p.v_inv = (const float*)kv->v_scales + (size_t)layer * kv->scale_layer_elems + kv->num_kv_heads;
        }
    }
    if (vectors_fit(a)) {
        gg_status_t st = GG_OK;
        with_float(a.dt, [&](auto t) {
            constexpr gg_dtype_t T = decltype(t)::value;
            st = a.D <= 64    ? launch_vectors<T, 8>(a, kv, p, s)
                 : a.D <= 128 ? launch_vectors<T, 16>(a, kv, p, s)
                              : launch_vectors<T, 32>(a, kv, p, s);
        });
        return st;
    }
    const long long waves = (long long)a.n * (a.Hq + a.Hkv);
    if ((waves + 3) / 4 > max_blocks_of(256)) return fail(GG_ERR_INVALID, "qk_norm_rope: too many rows for one call");
    qk_norm_rope_rows_kernel<<<(unsigned)((waves + 3) / 4), 256, 0, s>>>(a, p);
    return check_hip(hipGetLastError(), "qk_norm_rope launch");
}

}  // namespace gg
