// e4m3 codes in blocks of 128 with fp32 scales: helpers shared by the quantising kernels and the product.
#pragma once
#include <type_traits>

#include "ldot_common.h"

namespace ldot {

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;         // the largest e4m3 value

// op over groups of LANES neighbouring lanes (16, 32 or 64), the same result in all of them: four moves inside rows of 16 (neighbour, pair,
// mirrored halves, mirrored row), then swaps of rows — no trip through LDS
template <int LANES, typename F>
__device__ __forceinline__ float lanes_reduce(float v, F op) {
    auto moved = [](float x, auto ctrl) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
    v = op(v, moved(v, std::integral_constant<int, 0xb1>()));       // lane ^ 1
    v = op(v, moved(v, std::integral_constant<int, 0x4e>()));       // lane ^ 2
    v = op(v, moved(v, std::integral_constant<int, 0x141>()));      // 7 - lane in 8
    v = op(v, moved(v, std::integral_constant<int, 0x140>()));      // 15 - lane in 16
    if (LANES >= 32) {
        auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    if (LANES >= 64) {
        auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    return v;
}

// scale of a block from its largest magnitude: 1 where the block is all zeros
__device__ __forceinline__ float fp8_scale(float amax) { return amax > 0.f ? amax / kFp8Max : 1.f; }

// what a value is multiplied by before it is rounded; 0: the reciprocal is no normal number and the value is divided instead
__device__ __forceinline__ float fp8_inverse(float scale) { return scale >= 1.17549435e-38f && scale < 8.5e37f ? 1.f / scale : 0.f; }

__device__ __forceinline__ float fp8_scaled(float x, float scale, float inv) {
    const float q = x * inv, v = inv != 0.f ? __builtin_fmaf(__builtin_fmaf(-q, scale, x), inv, q) : x / scale;    // (x / scale, rounded once)
    const float c = fminf(fmaxf(v, -kFp8Max), kFp8Max);      // (rounding of the product must not leave the range)
    return v != v ? v : c;
}

// eight scaled values, rounded to the nearest code (ties to even), the first in the lowest byte
__device__ __forceinline__ uint2 fp8_pack(const float (&v)[8]) {
    uint2 r;
    r.x = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    r.x = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r.x, true);
    r.y = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
    r.y = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], r.y, true);
    return r;
}

template <int DT>
__device__ __forceinline__ float fp8_load(const void* p, int64_t i) {
    if (DT == LDOT_F32) return ((const float*)p)[i];
    if (DT == LDOT_BF16) return (float)((const __bf16*)p)[i];
    return (float)((const _Float16*)p)[i];
}
template <int DT>
__device__ __forceinline__ void fp8_store(void* p, int64_t i, float v) {
    if (DT == LDOT_F32) ((float*)p)[i] = v;
    else if (DT == LDOT_BF16) ((__bf16*)p)[i] = (__bf16)v;
    else ((_Float16*)p)[i] = (_Float16)v;
}

// two consecutive elements, aligned to their bytes
template <int DT>
__device__ __forceinline__ void fp8_load2(const void* p, int64_t i, float& x, float& y) {
    union {
        uint2 w;
        uint32_t u;
        float f[2];
        __bf16 b[2];
        _Float16 h[2];
    } v;
    if (DT == LDOT_F32) v.w = *(const uint2*)((const float*)p + i);
    else v.u = *(const uint32_t*)((const uint16_t*)p + i);
    x = DT == LDOT_F32 ? v.f[0] : DT == LDOT_BF16 ? (float)v.b[0] : (float)v.h[0];
    y = DT == LDOT_F32 ? v.f[1] : DT == LDOT_BF16 ? (float)v.b[1] : (float)v.h[1];
}
template <int DT>
__device__ __forceinline__ void fp8_store2(void* p, int64_t i, float x, float y) {
    union {
        uint2 w;
        uint32_t u;
        float f[2];
        __bf16 b[2];
        _Float16 h[2];
    } v;
    if (DT == LDOT_F32) v.f[0] = x, v.f[1] = y, *(uint2*)((float*)p + i) = v.w;
    else if (DT == LDOT_BF16) v.b[0] = (__bf16)x, v.b[1] = (__bf16)y, *(uint32_t*)((uint16_t*)p + i) = v.u;
    else v.h[0] = (_Float16)x, v.h[1] = (_Float16)y, *(uint32_t*)((uint16_t*)p + i) = v.u;
}

union Fp8Vec {
    uint4 u[2];
    float f[8];
    __bf16 b[8];
    _Float16 h[8];
};
// eight consecutive elements, 16-byte aligned
template <int DT>
__device__ __forceinline__ void fp8_load8(const void* p, int64_t i, float (&x)[8]) {
    Fp8Vec v;
    if (DT == LDOT_F32) {
        v.u[0] = ((const uint4*)((const float*)p + i))[0];
        v.u[1] = ((const uint4*)((const float*)p + i))[1];
    } else {
        v.u[0] = *(const uint4*)((const uint16_t*)p + i);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = DT == LDOT_F32 ? v.f[j] : DT == LDOT_BF16 ? (float)v.b[j] : (float)v.h[j];
}
template <int DT>
__device__ __forceinline__ void fp8_store8(void* p, int64_t i, const float (&x)[8]) {
    Fp8Vec v;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (DT == LDOT_F32) v.f[j] = x[j];
        else if (DT == LDOT_BF16) v.b[j] = (__bf16)x[j];
        else v.h[j] = (_Float16)x[j];
    }
    if (DT == LDOT_F32) {
        ((uint4*)((float*)p + i))[0] = v.u[0];
        ((uint4*)((float*)p + i))[1] = v.u[1];
    } else {
        *(uint4*)((uint16_t*)p + i) = v.u[0];
    }
}

}  // namespace ldot
