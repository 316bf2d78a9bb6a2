// kv_int4.hip — rows written to 4-bit pools (gg_kv_append), and rows of any pool read back
// (gg_kv_read).
#include "gg_common.h"
#include "attention_common.h"
#include "int4.h"

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
    const long long waves = (long long)n_rows * p.Hkv;
    append_int4_rows_kernel<<<(unsigned)((waves + 3) / 4), 256, 0, s>>>(p, k, v, src, slots, n_rows);
    return check_hip(hipGetLastError(), "kv_append launch");
}

gg_status_t launch_kv_read(KV* kv, int layer, void* k_out, void* v_out, gg_dtype_t dst, const int32_t* slots, int n_rows,
                           hipStream_t s) {
    const KVView view = make_kv_view(kv, layer);
    const long long n = (long long)n_rows * view.Hkv * view.D;
    if ((n + 255) / 256 > 0x7fffffffLL) return fail(GG_ERR_INVALID, "gg_kv_read: too many elements for one call");
    read_rows_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(view, k_out, v_out, dst, slots, n_rows);
    return check_hip(hipGetLastError(), "kv_read launch");
}

}  // namespace gg
