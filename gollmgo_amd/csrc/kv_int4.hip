// kv_int4.hip — rows written to 4-bit pools (gg_kv_append), and rows of any pool read back
// (gg_kv_read).
//
// Bound: memory. 32768 bf16 rows of 8 heads of 128, in block order (134 MB of rows, 35 MB of pool):
// written in 39 µs (4.3 TB/s; 75 % of that is vector instructions, the quotients), read back in 33 µs
// (5.1 TB/s). 8192 rows in order 11.9 and 11.5 µs, in shuffled slots, partial lines, 26 and 14. The
// five rows of one step 3.3 and 3.6 µs, the launch.
#include "gg_common.h"
#include "attention_common.h"
#include "int4.h"
#include "int4_tile.h"
#include "lanes.h"

namespace gg {
namespace {

// One wave per (row, head), any even head_dim.
__global__ void __launch_bounds__(256) append_int4_rows_kernel(Int4View p, const void* k, const void* v, gg_dtype_t src,
                                                               const int32_t* slots, int n_rows) {
    const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int r = (int)(i / p.Hkv), h = (int)(i % p.Hkv);
    if (r >= n_rows) return;
    const int slot = slots[r];
    if (slot < 0 || slot >= p.num_slots) return;
    const size_t at = ((size_t)r * p.Hkv + h) * p.D;
    int4_write_row(p, slot / p.bs, h, slot % p.bs, [&](int d) { return load_as_f32(k, src, at + d); },
                   [&](int d) { return load_as_f32(v, src, at + d); });
}

// Sixteen rows of one head (or of 16 / LPR heads) per 256-thread workgroup: int4_tile.h.
template <gg_dtype_t SRC, int LPR, bool FULL>
__global__ void __launch_bounds__(256) append_int4_tile_kernel(Int4View p, const void* k, const void* v, const int32_t* slots,
                                                               int n_rows, unsigned hg) {
    __shared__ Int4Tile<LPR> tile;
    const size_t stride = (size_t)p.Hkv * p.D;
    int4_tile_rows<SRC, LPR, FULL>(
        p, slots, n_rows, blockIdx.x / hg, blockIdx.x % hg, tile,
        [&](int r, int h, int u) {
            const size_t at = (size_t)r * stride + (size_t)h * p.D;
            const int oa = 4 * u, ob = p.D / 2 + 4 * u;
            return Int4Raw<SRC>{load4<SRC>(k, at + oa), load4<SRC>(k, at + ob), load4<SRC>(v, at + oa), load4<SRC>(v, at + ob)};
        },
        [&](const Int4Raw<SRC>& w, int, int, int u, float (&ka)[4], float (&kb)[4], float (&va)[4], float (&vb)[4], int& oa, int& ob) {
            oa = 4 * u;
            ob = p.D / 2 + 4 * u;
            to_f32<SRC>(w.ka, ka);
            to_f32<SRC>(w.kb, kb);
            to_f32<SRC>(w.va, va);
            to_f32<SRC>(w.vb, vb);
        });
}

// A 4-bit pool's rows back, sixteen of one head per workgroup of 2 * head_dim threads (HD, or any of whole
// sixteens up to 256 where that is 0): thread (row, c) gives dims 8c .. 8c + 7. Where the rows are a block in order its V tile comes in whole 16-byte
// runs through LDS (each run is sixteen tokens of two dims); else V byte by byte.
template <gg_dtype_t DST, int HD>
__global__ void __launch_bounds__(HD ? 2 * HD : 512) read_int4_tile_kernel(Int4View p, void* k_out, void* v_out, const int32_t* slots, int n_rows) {
    constexpr int kMost = HD ? HD : 256;
    const int D = HD ? HD : p.D, kC = D / 8;
    __shared__ uint32_t s_v[kMost / 2 * 4 + kMost / 16];  // run i at word 4 i + i / 8 (eight runs apart: other banks)
    const int h = blockIdx.x % p.Hkv, group = blockIdx.x / p.Hkv, row = threadIdx.x / kC, c = threadIdx.x % kC;
    const int first = slots[0] < 0 ? 0 : slots[0] % p.bs;  // a prompt's groups start where its blocks do
    const int r = group * 16 - first % 16 + row;
    const int slot = r >= 0 && r < n_rows ? slots[r] : -1;
    const bool live = slot >= 0 && slot < p.num_slots;
    const int blk = live ? slot / p.bs : 0, off = live ? slot % p.bs : 0;
    const int lead = slots[min(max(group * 16 - first % 16, 0), n_rows - 1)];
    const bool whole = __syncthreads_and(live && p.bs == 16 && slot == lead + row && lead % 16 == 0) != 0;
    const uint8_t* vt = p.vc + p.tile0(blk, h);
    if (whole && v_out) {
        if ((int)threadIdx.x < D / 2) {
            const uint4 x = *(const uint4*)(vt + (size_t)threadIdx.x * 16);
            uint32_t* d = s_v + 4 * threadIdx.x + threadIdx.x / 8;
            d[0] = x.x, d[1] = x.y, d[2] = x.z, d[3] = x.w;
        }
        __syncthreads();
    }
    if (!live) return;
    const uint32_t w = p.words[p.word(blk, h, off)];
    const size_t to = ((size_t)r * p.Hkv + h) * D + 8 * c;
    auto put = [&](void* out, const float (&f)[8]) {
        if constexpr (DST == GG_DTYPE_F32) {
            ((float4*)((float*)out + to))[0] = make_float4(f[0], f[1], f[2], f[3]);
            ((float4*)((float*)out + to))[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *(uint4*)((uint16_t*)out + to) =
                make_uint4(pack2<DST>(f[0], f[1]), pack2<DST>(f[2], f[3]), pack2<DST>(f[4], f[5]), pack2<DST>(f[6], f[7]));
        }
    };
    float f[8];
    if (k_out) {
        const uint32_t x = *(const uint32_t*)(p.kc + p.tile0(blk, h) + (size_t)off * (D / 2) + 4 * c);
        const float s = int4_k_scale(w);
        const int z = int4_k_zero(w);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = s * (float)((int)((x >> (4 * e)) & 15u) - z);
        put(k_out, f);
    }
    if (v_out) {
        const float s = int4_v_scale(w);
        const int z = int4_v_zero(w);
        const int i0 = 8 * (c % (kC / 2)), shift = c < kC / 2 ? 0 : 4;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t b = whole ? ((const uint8_t*)(s_v + 4 * (i0 + e) + i0 / 8))[off] : vt[(size_t)(i0 + e) * p.bs + off];
            f[e] = s * (float)((int)((b >> shift) & 15u) - z);
        }
        put(v_out, f);
    }
}

// One thread per element, row after row: K rows are contiguous; V elements of a row lie bs apart.
__global__ void __launch_bounds__(256) read_rows_kernel(KVView kv, void* k_out, void* v_out, gg_dtype_t dst,
                                                        const int32_t* slots, int n_rows) {
    const int per = kv.Hkv * kv.D;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)n_rows * per) return;
    const int r = (int)(i / per), h = (int)(i % per) / kv.D, d = (int)(i % kv.D);
    const int slot = slots[r];
    if (slot < 0 || slot >= (long long)kv.num_blocks * kv.bs) return;
    const int blk = slot / kv.bs, off = slot % kv.bs;
    if (k_out) store_from_f32(k_out, dst, (size_t)i, kv.k_value(blk, h, off, d));
    if (v_out) store_from_f32(v_out, dst, (size_t)i, kv.v_value(blk, h, off, d));
}

}  // namespace

gg_status_t launch_kv_append_int4(KV* kv, int layer, const void* k, const void* v, gg_dtype_t src, const int32_t* slots,
                                  int n_rows, hipStream_t s) {
    const Int4View p = int4_view(kv, layer);
    const char* too_many = "gg_kv_append: too many rows for one call";
    // By tiles of sixteen rows: head_dims of up to 32 lanes of eight dims, vector loads. (8192 bf16 rows of
    // 8 heads in order, a wave to a row and head / by tiles: head_dim 96 42 / 12 µs.)
    const size_t align = src == GG_DTYPE_F32 ? 16 : 8;
    if (int4_tile_dim(p.D) && (uintptr_t)k % align == 0 && (uintptr_t)v % align == 0) {
        const unsigned hg = int4_tile_heads(p.Hkv, p.D);
        const long long blocks = (long long)int4_tile_groups(n_rows) * hg;
        if (blocks > max_blocks_of(256)) return fail(GG_ERR_INVALID, too_many);
        const unsigned grid = (unsigned)blocks;
        with_float(src, [&](auto t) {
            constexpr gg_dtype_t T = decltype(t)::value;
            auto launch = [&](auto lpr) {
                constexpr int LPR = decltype(lpr)::value;
                if (p.D == 8 * LPR) append_int4_tile_kernel<T, LPR, true><<<grid, 256, 0, s>>>(p, k, v, slots, n_rows, hg);
                else append_int4_tile_kernel<T, LPR, false><<<grid, 256, 0, s>>>(p, k, v, slots, n_rows, hg);
            };
            if (p.D <= 64) launch(std::integral_constant<int, 8>{});
            else if (p.D <= 128) launch(std::integral_constant<int, 16>{});
            else launch(std::integral_constant<int, 32>{});
        });
        return check_hip(hipGetLastError(), "kv_append launch");
    }
    const long long waves = (long long)n_rows * p.Hkv;
    if ((waves + 3) / 4 > max_blocks_of(256)) return fail(GG_ERR_INVALID, too_many);
    append_int4_rows_kernel<<<(unsigned)((waves + 3) / 4), 256, 0, s>>>(p, k, v, src, slots, n_rows);
    return check_hip(hipGetLastError(), "kv_append launch");
}

gg_status_t launch_kv_read(KV* kv, int layer, void* k_out, void* v_out, gg_dtype_t dst, const int32_t* slots, int n_rows,
                           hipStream_t s) {
    // (8192 bf16 rows of 8 heads of 96 in order, an element a thread / by tiles: 31 / 10.5 µs.)
    if (kv->dtype == GG_DTYPE_INT4 && kv->head_dim % 16 == 0 && kv->head_dim <= 256 &&
        (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0) {
        const Int4View p = int4_view(kv, layer);
        const long long blocks = (long long)int4_tile_groups(n_rows) * p.Hkv;
        if (blocks > max_blocks_of(2 * p.D)) return fail(GG_ERR_INVALID, "gg_kv_read: too many rows for one call");
        const unsigned grid = (unsigned)blocks;
        with_float(dst, [&](auto t) {
            constexpr gg_dtype_t T = decltype(t)::value;
            if (p.D == 64) read_int4_tile_kernel<T, 64><<<grid, 128, 0, s>>>(p, k_out, v_out, slots, n_rows);
            else if (p.D == 128) read_int4_tile_kernel<T, 128><<<grid, 256, 0, s>>>(p, k_out, v_out, slots, n_rows);
            else if (p.D == 256) read_int4_tile_kernel<T, 256><<<grid, 512, 0, s>>>(p, k_out, v_out, slots, n_rows);
            else read_int4_tile_kernel<T, 0><<<grid, 2 * p.D, 0, s>>>(p, k_out, v_out, slots, n_rows);
        });
        return check_hip(hipGetLastError(), "kv_read launch");
    }
    const KVView view = make_kv_view(kv, layer);
    const long long n = (long long)n_rows * view.Hkv * view.D;
    if ((n + 255) / 256 > max_blocks_of(256)) return fail(GG_ERR_INVALID, "gg_kv_read: too many rows for one call");
    read_rows_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(view, k_out, v_out, dst, slots, n_rows);
    return check_hip(hipGetLastError(), "kv_read launch");
}

}  // namespace gg
