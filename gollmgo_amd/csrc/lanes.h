// lanes.h — reductions over groups of neighbouring lanes, result in every lane of the group.
#pragma once
#include "gg_common.h"

#ifdef __HIPCC__
namespace gg {

template <int CTRL, class V>
__device__ __forceinline__ V dpp(V v) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// N = 8, 16 or 32 lanes. Steps 1 and 2 exchange within a quad; then a mirror of eight and one of
// sixteen lanes, where the halves already agree, stand for the exchanges by 4 and 8: all of it in the
// vector unit (a shuffle is a trip through LDS).
template <int N, class V, class F>
__device__ __forceinline__ V group_reduce(V v, F f) {
    static_assert(N == 8 || N == 16 || N == 32, "group size");
    v = f(v, dpp<0xb1>(v));   // quad_perm [1, 0, 3, 2]
    v = f(v, dpp<0x4e>(v));   // quad_perm [2, 3, 0, 1]
    v = f(v, dpp<0x141>(v));  // row_half_mirror
    if constexpr (N >= 16) v = f(v, dpp<0x140>(v));  // row_mirror
    if constexpr (N == 32) v = f(v, __shfl_xor(v, 16));
    return v;
}
template <int N>
__device__ __forceinline__ float group_sum(float v) {
    return group_reduce<N>(v, [](float a, float b) { return a + b; });
}
template <int N>
__device__ __forceinline__ float group_max(float v) {
    return group_reduce<N>(v, [](float a, float b) { return fmaxf(a, b); });
}

template <int N, class V>
__device__ __forceinline__ V group_max_int(V v) {
    return group_reduce<N>(v, [](V a, V b) { return max(a, b); });
}

// Four consecutive elements of a float type, and back.
template <gg_dtype_t DT>
struct Raw4 {
    uint4 w;  // 16-bit types: the low two words
};
template <gg_dtype_t DT>
__device__ __forceinline__ Raw4<DT> load4(const void* p, size_t i) {
    Raw4<DT> r;
    if constexpr (DT == GG_DTYPE_F32) {
        r.w = *(const uint4*)((const float*)p + i);
    } else {
        const uint2 x = *(const uint2*)((const uint16_t*)p + i);
        r.w = make_uint4(x.x, x.y, 0, 0);
    }
    return r;
}
template <gg_dtype_t DT>
__device__ __forceinline__ void to_f32(const Raw4<DT>& r, float (&f)[4]) {
    if constexpr (DT == GG_DTYPE_F32) {
        f[0] = __uint_as_float(r.w.x), f[1] = __uint_as_float(r.w.y), f[2] = __uint_as_float(r.w.z), f[3] = __uint_as_float(r.w.w);
    } else if constexpr (DT == GG_DTYPE_BF16) {
        f[0] = __uint_as_float(r.w.x << 16), f[1] = __uint_as_float(r.w.x & 0xffff0000u);
        f[2] = __uint_as_float(r.w.y << 16), f[3] = __uint_as_float(r.w.y & 0xffff0000u);
    } else {
        f[0] = f16_bits_to_f32((uint16_t)r.w.x), f[1] = f16_bits_to_f32((uint16_t)(r.w.x >> 16));
        f[2] = f16_bits_to_f32((uint16_t)r.w.y), f[3] = f16_bits_to_f32((uint16_t)(r.w.y >> 16));
    }
}
// (A pair by the hardware's round-to-nearest-even conversion.)
template <gg_dtype_t DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = {a, b};
    if constexpr (DT == GG_DTYPE_BF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2));
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
    }
}
template <gg_dtype_t DT>
__device__ __forceinline__ void store4(void* p, size_t i, const float (&f)[4]) {
    if constexpr (DT == GG_DTYPE_F32) *(float4*)((float*)p + i) = make_float4(f[0], f[1], f[2], f[3]);
    else *(uint2*)((uint16_t*)p + i) = make_uint2(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]));
}

}  // namespace gg
#endif
