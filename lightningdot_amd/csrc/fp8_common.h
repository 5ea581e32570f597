// e4m3 codes in blocks of 128 with fp32 scales: helpers shared by the quantising kernels and the product.
#pragma once
#include <type_traits>

#include "ldot_common.h"

namespace ldot {

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;         // the largest e4m3 value

// a value of another lane, by a move between registers: 64-bit values in two halves
template <int CTRL>
__device__ __forceinline__ float lane_moved(float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true)); }
template <int CTRL>
__device__ __forceinline__ double lane_moved(double x) {
    return __hiloint2double(__builtin_amdgcn_mov_dpp(__double2hiint(x), CTRL, 0xf, 0xf, true), __builtin_amdgcn_mov_dpp(__double2loint(x), CTRL, 0xf, 0xf, true));
}
template <bool ROWS_OF_32>
__device__ __forceinline__ auto lane_swap(uint32_t x) {
    if constexpr (ROWS_OF_32) return __builtin_amdgcn_permlane32_swap(x, x, false, false);
    else return __builtin_amdgcn_permlane16_swap(x, x, false, false);
}
template <bool ROWS_OF_32, typename F>
__device__ __forceinline__ float lanes_join(float v, F op) {
    auto a = lane_swap<ROWS_OF_32>(__float_as_uint(v));
    return op(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
template <bool ROWS_OF_32, typename F>
__device__ __forceinline__ double lanes_join(double v, F op) {
    auto lo = lane_swap<ROWS_OF_32>((uint32_t)__double2loint(v)), hi = lane_swap<ROWS_OF_32>((uint32_t)__double2hiint(v));
    return op(__hiloint2double((int)hi[0], (int)lo[0]), __hiloint2double((int)hi[1], (int)lo[1]));
}

// op over groups of LANES neighbouring lanes (16, 32 or 64), the same result in all of them: four moves inside rows of 16 (neighbour, pair,
// mirrored halves, mirrored row), then swaps of rows — no trip through LDS
template <int LANES, typename V, typename F>
__device__ __forceinline__ V lanes_reduce(V v, F op) {
    v = op(v, lane_moved<0xb1>(v));        // lane ^ 1
    v = op(v, lane_moved<0x4e>(v));        // lane ^ 2
    v = op(v, lane_moved<0x141>(v));       // 7 - lane in 8
    v = op(v, lane_moved<0x140>(v));       // 15 - lane in 16
    if (LANES >= 32) v = lanes_join<false>(v, op);
    if (LANES >= 64) v = lanes_join<true>(v, op);
    return v;
}

// scale of a block from its largest magnitude: 1 where the block is all zeros
__device__ __forceinline__ float fp8_scale(float amax) { return amax > 0.f ? amax / kFp8Max : 1.f; }

// what a value is multiplied by before it is rounded; 0: the reciprocal is no normal number and the value is divided instead
__device__ __forceinline__ float fp8_inverse(float scale) { return scale >= 1.17549435e-38f && scale < 8.5e37f ? 1.f / scale : 0.f; }

__device__ __forceinline__ float fp8_limit(float v) {
    const float c = fminf(fmaxf(v, -kFp8Max), kFp8Max);
    return v != v ? v : c;
}
__device__ __forceinline__ float fp8_scaled(float x, float scale, float inv) {
    const float q = x * inv, v = inv != 0.f ? __builtin_fmaf(__builtin_fmaf(-q, scale, x), inv, q) : x / scale;    // (x / scale, rounded once)
    return fp8_limit(v);                 // (rounding of the product must not leave the range)
}

// a 64-bit value in 32 bits, cut off with its last bit set if anything was lost: a later rounding to fewer bits then sees on which side of
// the middle between two of its results the value lies
__device__ __forceinline__ float fp8_cut(double v) {
    const uint32_t lo = (uint32_t)__double2loint(v), below = 0x1fffffffu;
    return (float)__hiloint2double(__double2hiint(v), (int)((lo | ((lo & below) + below)) & ~below));
}

// x / by, rounded once, from 1 / by; by 0 and inv 0: 0, and NaN for what is infinite
__device__ __forceinline__ double fp8_quotient(double x, double by, double inv) {
    const double q = x * inv;
    return __builtin_fma(__builtin_fma(-q, by, x), inv, q);
}
// 1 / by: the hardware's reciprocal, twice improved; 0 where `undo`, else by itself, is 0 (an infinite divisor)
__device__ __forceinline__ double fp8_reciprocal(double by, double undo) {
    double r = __builtin_amdgcn_rcp(by);
    r = __builtin_fma(__builtin_fma(-undo, r, 1.), r, r);
    return __builtin_fma(__builtin_fma(-undo, r, 1.), r, r);
}

// 1 / sqrt(x), the same way; x = 0 and x = infinity as the hardware gives them
__device__ __forceinline__ double fp8_rsqrt(double x) {
    const double r = __builtin_amdgcn_rsq(x), e = __builtin_fma(-x * r, r, 1.), s = __builtin_fma(0.5 * r, e, r), f = __builtin_fma(-x * s, s, 1.);
    return x > 0. && x < 1e300 ? __builtin_fma(0.5 * s, f, s) : r;
}
// the larger of a and |x|, as fmax has it (NaN: the other one), without the instruction that makes a signalling NaN a quiet one first
__device__ __forceinline__ double fp8_larger(double a, double x) {
    double r;
    asm("v_max_f64 %0, %1, |%2|" : "=v"(r) : "v"(a), "v"(x));
    return r;
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
