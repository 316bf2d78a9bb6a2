// attention_rows.h — one partition of one (row, head) of the verify attention by one wave, keys
// and dims in fp32: the phase-1 step of the per-row kernel, and of pieces of the MFMA kernels
// that are computed row by row (piece_by_rows).
#pragma once
#include "gg_common.h"
#include "attention_common.h"

namespace gg {
namespace {

// One pool element as f32 (raw, before its block / head scale), pool type fixed.
template <gg_dtype_t DT>
__device__ __forceinline__ float pool_elem(const uint8_t* base, size_t i) {
    if constexpr (DT == GG_DTYPE_F32) return ((const float*)base)[i];
    else if constexpr (DT == GG_DTYPE_F16) return f16_bits_to_f32(((const uint16_t*)base)[i]);
    else if constexpr (DT == GG_DTYPE_BF16) return bf16_bits_to_f32(((const uint16_t*)base)[i]);
    else if constexpr (DT == GG_DTYPE_FP8_E4M3) return fp8e4m3_to_f32(base[i]);
    else if constexpr (DT == GG_DTYPE_INT4) return (float)((base[i >> 1] >> (4 * (i & 1))) & 15u);
    else return (float)((const int8_t*)base)[i];
}

// The pool elements in 16 bytes, as f32.
template <gg_dtype_t DT>
struct Pool16 {
    static constexpr int kN = DT == GG_DTYPE_F32                              ? 4
                              : (DT == GG_DTYPE_F16 || DT == GG_DTYPE_BF16) ? 8
                              : DT == GG_DTYPE_INT4                         ? 32
                                                                            : 16;
    __device__ static __forceinline__ void decode(const uint4 r, float (&f)[kN]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int k = 0; k < kN; ++k) {
            if constexpr (DT == GG_DTYPE_F32) f[k] = __uint_as_float(w[k]);
            else if constexpr (DT == GG_DTYPE_F16) f[k] = f16_bits_to_f32((uint16_t)(w[k >> 1] >> (16 * (k & 1))));
            else if constexpr (DT == GG_DTYPE_BF16) f[k] = bf16_bits_to_f32((uint16_t)(w[k >> 1] >> (16 * (k & 1))));
            else if constexpr (DT == GG_DTYPE_FP8_E4M3)
                f[k] = (k & 3) == 0   ? fp8e4m3_to_f32<0>(w[k >> 2])
                       : (k & 3) == 1 ? fp8e4m3_to_f32<1>(w[k >> 2])
                       : (k & 3) == 2 ? fp8e4m3_to_f32<2>(w[k >> 2])
                                      : fp8e4m3_to_f32<3>(w[k >> 2]);
            else if constexpr (DT == GG_DTYPE_INT4) f[k] = (float)((w[k >> 3] >> (4 * (k & 7))) & 15u);
            else f[k] = (float)(int8_t)(uint8_t)(w[k >> 2] >> (8 * (k & 3)));
        }
    }
};

// One partition of one (row, head), by one wave: keys in tiles of 64, lane i scoring key i of
// the tile against the whole query (in LDS), one wave max and sum per tile, then P.V with each
// lane owning dims lane + 64c. A tile's K rows and V runs are all requested before its scores
// are needed, so a tile waits for one round trip to its block ids and one to its K and V. V
// comes in 16-byte runs of offsets where blocks are whole runs and tiles whole blocks
// (kVRun), by element elsewhere; the products are added in key order either way.
// Bound by those round trips: with four K vectors and sixteen V elements in flight (V at a
// line per lane and key) and the merge in a launch, 4 x 5 rows of 8 heads over 64-256 fp32 keys
// took 14.0 + 4.2 µs, now 8.8; per call on one box, four fp32 sequences of 100-700 keys at
// head_dim 128 64 -> 25 µs, eight bf16 ones at head_dim 96 132 -> 24.
// 4-bit pools: codes less their token's zero point, its scales on the score and on p. A V run of sixteen
// tokens holds two dims; a lane takes its own half of each byte. (V by element: 16 sequences of
// 1024 keys, four rows of 16 heads at head_dim 96 145 µs, by runs 37.)
template <gg_dtype_t DT, int DC, bool kVRun>
__device__ __forceinline__ void generic_partition(const AttnArgs& a, const KVView& kv, int b, int kvh, int t0, int t1,
                                                  const float* s_q, float* s_p, size_t* s_vrow, float (&acc)[DC], float& m,
                                                  float& l) {
    const int lane = threadIdx.x & 63;
    const int D = kv.D;
    const int32_t* bt = a.block_tables + (size_t)b * a.max_blocks;
    const uint8_t* vc = kv.vc;
    constexpr bool kInt4 = DT == GG_DTYPE_INT4;
    constexpr int kN = Pool16<DT>::kN;             // K elements of 16 bytes
    constexpr int kNV = kInt4 ? 16 : kN;           // tokens of a 16-byte V run
    constexpr int kRuns = 64 / kNV;  // 16-byte V runs of a tile per dim
    m = -1e30f;
    l = 0.f;
#pragma unroll
    for (int c = 0; c < DC; ++c) acc[c] = 0.f;
    for (int tb = t0; tb < t1; tb += 64) {
        const int t = tb + lane;
        const int ntile = min(64, t1 - tb);
        int blk = -1, off = 0;
        if (t < t1) {
            blk = bt[t / kv.bs];
            off = t % kv.bs;
            if (blk < 0 || blk >= kv.num_blocks) blk = -1;  // invalid table entry: key skipped
        }
        // (Skipped keys read block 0.)
        const size_t vrow = kInt4 ? kv.tile0(max(blk, 0), kvh) / 2 + off : kv.tile0(max(blk, 0), kvh) + off;
        [[maybe_unused]] uint32_t word = 0;
        if constexpr (kInt4) {
            if (blk >= 0) word = kv.word(blk, kvh, off);
        }
        [[maybe_unused]] const float kzero = kInt4 ? (float)int4_k_zero(word) : 0.f;
        [[maybe_unused]] uint4 vr[kVRun ? DC : 1][kVRun ? kRuns : 1];
        if constexpr (kVRun) {
#pragma unroll
            for (int r = 0; r < kRuns; ++r) {
                const size_t base = ((size_t)__shfl((unsigned)(vrow >> 32), r * kNV) << 32) | (unsigned)__shfl((unsigned)vrow, r * kNV);
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                    const int d = min(lane + 64 * c, D - 1);
                    // (A run past the tile reads its key 0's block: not used.)
                    if constexpr (kInt4) vr[c][r] = *(const uint4*)(vc + base + (size_t)(d >= D / 2 ? d - D / 2 : d) * kv.bs);
                    else vr[c][r] = *(const uint4*)(vc + (base + (size_t)d * kv.bs) * dtype_bytes(DT));
                }
            }
        }
        float sc = -INFINITY;
        if (blk >= 0) {
            // The lane's key row is contiguous: 16-byte loads when rows are whole
            // multiples of 16 bytes (pools are 256-byte aligned), else element loads.
            const size_t krow_i = kv.tile0(blk, kvh) + (size_t)off * D;
            const uint8_t* krow = kv.kc + (kInt4 ? krow_i / 2 : krow_i * dtype_bytes(DT));
            float dot = 0.f;
            if (D % kN == 0) {
#pragma unroll(DT == GG_DTYPE_F32 ? 16 : 4)
                for (int v = 0; v < D / kN; ++v) {
                    float f[kN];
                    Pool16<DT>::decode(((const uint4*)krow)[v], f);
#pragma unroll
                    for (int e = 0; e < kN; ++e) dot += s_q[v * kN + e] * (kInt4 ? f[e] - kzero : f[e]);
                }
            } else if (kInt4 && D % 8 == 0) {
#pragma unroll 4
                for (int v = 0; v < D / 8; ++v) {
                    const uint32_t w = ((const uint32_t*)krow)[v];
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot += s_q[8 * v + e] * ((float)((w >> (4 * e)) & 15u) - kzero);
                }
            } else {
#pragma unroll 16
                for (int d = 0; d < D; ++d)
                    dot += s_q[d] * (kInt4 ? pool_elem<DT>(krow, d) - kzero : pool_elem<DT>(krow, d));
            }
            sc = dot * a.scale * (kInt4 ? int4_k_scale(word) : kv.k_scale(blk, kvh));
        }
        float mt = sc;
        for (int o = 32; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor(mt, o));
        const float m_new = fmaxf(m, mt);
        const float alpha = __expf(m - m_new);
        const float p = blk >= 0 ? __expf(sc - m_new) : 0.f;
        float ps = p;
        for (int o = 32; o > 0; o >>= 1) ps += __shfl_xor(ps, o);
        l = l * alpha + ps;
        m = m_new;
#pragma unroll
        for (int c = 0; c < DC; ++c) acc[c] *= alpha;
        // The tile's probabilities (and by element, V offsets) go through LDS, so the key loop
        // below has no cross-lane operations. (Masked and skipped keys have p = 0.)
        // One wave's own slots: its LDS operations complete in order.
        __builtin_amdgcn_wave_barrier();
        s_p[lane] = blk >= 0 ? p * (kInt4 ? int4_v_scale(word) : kv.v_scale(blk, kvh)) : 0.f;
        if constexpr (kInt4 && kVRun) ((float*)s_vrow)[lane] = (float)int4_v_zero(word);
        else if constexpr (kInt4) s_vrow[lane] = vrow | ((size_t)int4_v_zero(word) << 60);  // (pools are far below 2^60 bytes)
        else if constexpr (!kVRun) s_vrow[lane] = vrow;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if constexpr (kVRun) {
#pragma unroll
            for (int r = 0; r < kRuns; ++r) {
                if (r * kNV >= ntile) break;
                float pi[kNV];
#pragma unroll
                for (int e = 0; e < kNV; ++e) pi[e] = s_p[r * kNV + e];
                if constexpr (kInt4) {
                    // (Codes are finite: masked and skipped keys have p = 0.)
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        const uint32_t w[4] = {vr[c][r].x, vr[c][r].y, vr[c][r].z, vr[c][r].w};
                        const int shift = lane + 64 * c >= D / 2 ? 4 : 0;
#pragma unroll
                        for (int e = 0; e < kNV; ++e)
                            acc[c] += pi[e] * ((float)((w[e >> 2] >> (8 * (e & 3) + shift)) & 15u) - ((const float*)s_vrow)[r * kNV + e]);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        float f[kN];
                        Pool16<DT>::decode(vr[c][r], f);
#pragma unroll
                        for (int e = 0; e < kN; ++e) acc[c] += pi[e] * (r * kN + e < ntile ? f[e] : 0.f);
                    }
                }
            }
        } else {
#pragma unroll 16
            for (int i = 0; i < ntile; ++i) {
                const float pi = s_p[i];
                const size_t vr0 = s_vrow[i];
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                    const int d = lane + 64 * c;
                    if constexpr (kInt4) {
                        const bool up = d >= D / 2;
                        const uint8_t* q = vc + (vr0 & (((size_t)1 << 60) - 1)) + (size_t)(up ? d - D / 2 : d) * kv.bs;
                        if (d < D) acc[c] += pi * ((float)((*q >> (up ? 4 : 0)) & 15u) - (float)(int)(vr0 >> 60));
                    } else if (d < D) {
                        acc[c] += pi * pool_elem<DT>(vc, vr0 + (size_t)d * kv.bs);
                    }
                }
            }
        }
    }
}

}  // namespace
}  // namespace gg
