// qk_norm_rope.hip — norm of each query and key head and the rotation of its positions, in one pass;
// keys to a dense output or, with the values, to a cache.
#include "gg_common.h"
#include "int4.h"

namespace gg {
namespace {

constexpr int kRowsMaxD = 1024;

// cos and sin of position times frequency. The angle in turns, and its whole turns taken off, in 64
// bits (at position 2^31 the product still keeps 2^-21 of a turn); the rest is exact enough in fp32.
__device__ __forceinline__ void turn_of(int pos, float freq, float& c, float& s) {
    constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
    double t = (double)pos * ((double)freq * kTurn);
    t -= __builtin_rint(t);
    sincospif((float)(2.0 * t), &s, &c);
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
__global__ void __launch_bounds__(256) qk_norm_rope_rows_kernel(RopeArgs a, PoolOut p) {
    __shared__ float s_row[4][kRowsMaxD];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long i = (long long)blockIdx.x * 4 + wave;
    const int heads = a.Hq + a.Hkv, D = a.D, P = a.pairs;
    if (i >= (long long)a.n * heads) return;
    const int t = (int)(i / heads), hh = (int)(i % heads);
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
        norm = rsqrtf(wave_sum(sum) / (float)D + a.eps);
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
        return weight ? x * norm * load_as_f32(weight, a.dt, d) : x;
    };
    auto put = [&](int d, float y) {
        if (to_int4) s_row[wave][d] = y;
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
        const float x = value(da), y = value(db);
        put(da, x * c - y * s);
        put(db, y * c + x * s);
    }
    if (!cached) return;
    const size_t vat = (size_t)t * a.v_stride + (size_t)h * D;
    if (to_int4) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        int4_write_row(p.i4, blk, h, off, [&](int d) { return s_row[wave][d]; },
                       [&](int d) { return load_as_f32(a.v, a.dt, vat + d); });
    } else {
        const float vinv = p.dt == GG_DTYPE_FP8_E4M3 ? p.v_inv[h] : 1.f;
        for (int d = lane; d < D; d += 64)
            pool_store(p.vc, p.dt, tile + (size_t)d * p.bs + off, load_as_f32(a.v, a.dt, vat + d), vinv);
    }
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
    const long long waves = (long long)a.n * (a.Hq + a.Hkv);
    if ((waves + 3) / 4 > 0x7fffffffLL) return fail(GG_ERR_INVALID, "qk_norm_rope: too many rows for one call");
    qk_norm_rope_rows_kernel<<<(unsigned)((waves + 3) / 4), 256, 0, s>>>(a, p);
    return check_hip(hipGetLastError(), "qk_norm_rope launch");
}

}  // namespace gg
