// Activations and weights into 8 bits (e4m3, a scale for each block of 128), alone or behind the towers' residual norm
// (uniter_model/model/layer.py:103-113,144-154: LayerNorm(dense(x) + residual)):
//     z = x + r,  mean = sum z / k,  var = sum (z - mean)^2 / k,  y = (z - mean) / sqrt(var + eps) * w + b,
//     scale_b = max_{i in block b} |y_i| / 448,  code_i = e4m3(y_i / scale_b)
// Bound by memory: a row is read once, kept in registers (mean, then variance around it, then the block's largest value: three passes
// over registers, none over memory) and written once in both forms.  86011 x 768 in bf16: 111 us, 4.2 TB/s (95 us,
// a large copy's rate, without the check of codes next to a border).
#include <algorithm>

#include "fp8_common.h"

namespace ldot {
namespace {

struct NormArgs {
    const void *x, *r;
    int64_t ldx, ldr, m;
    int k;
    const float *w, *b;
    float eps;
    void *y, *codes;
    float* scales;
};

// a row per LANES lanes (16 to 64 of a wave, or the whole workgroup).  TOGETHER 8: rows start on 16 bytes and k is a multiple of 8; lane i takes
// the groups of eight elements i, i + LANES, ...: 16 lanes hold one block of 128.  Else neighbouring lanes take neighbouring pairs (TOGETHER 2) or
// elements (1): 16 lanes hold a row of one block, or a wave holds a block at a time, two elements per lane (37394 x 262 in fp16, before codes were
// checked: 33 us by pairs, 38 by elements; with eight elements in a row per lane, each load over eight cache lines, 82)
template <int DT, int LANES, int ITER, bool NORM, int TOGETHER>
__global__ __launch_bounds__(256) void norm_e4m3_kernel(const NormArgs a) {
    constexpr bool VEC = TOGETHER == 8;
    __shared__ float sh[2][4];
    const int lane = (int)threadIdx.x % LANES;
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    if (row >= a.m) return;             // (whole rows leave: lanes that exchange values stay together)
    // a pair's elements lie together where rows can be pairs, and otherwise half a piece apart, so that neighbouring lanes read neighbours
    const bool pairs = TOGETHER == 2 || (a.k & 1) == 0;
    constexpr int kPiece = LANES == 16 ? 16 : 64;
    const int place = pairs ? 2 * (lane % kPiece) : lane % kPiece, other = pairs ? 1 : kPiece;
    auto column = [&](int i, int j) {                  // of this lane's element (i, j)
        if (VEC) return (lane + i * LANES) * 8 + j;
        if (LANES == 16) return 32 * (j >> 1) + place + (j & 1) * other;
        const int t = 8 * i + j;
        return ((t >> 1) * (LANES / 64) + lane / 64) * kFp8Block + place + (t & 1) * other;
    };
    float z[ITER][8];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (lane + i * LANES) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[i][j] = 0.f;
        if (VEC) {
            if (c < a.k) {
                fp8_load8<DT>(a.x, row * a.ldx + c, z[i]);
                if (NORM && a.r) {
                    float t[8];
                    fp8_load8<DT>(a.r, row * a.ldr + c, t);
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[i][j] += t[j];
                }
            }
        } else if (TOGETHER == 2) {
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                if (column(i, j) < a.k) {
                    fp8_load2<DT>(a.x, row * a.ldx + column(i, j), z[i][j], z[i][j + 1]);
                    if (NORM && a.r) {
                        float t, u;
                        fp8_load2<DT>(a.r, row * a.ldr + column(i, j), t, u);
                        z[i][j] += t;
                        z[i][j + 1] += u;
                    }
                }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (column(i, j) < a.k) {
                    z[i][j] = fp8_load<DT>(a.x, row * a.ldx + column(i, j));
                    if (NORM && a.r) z[i][j] += fp8_load<DT>(a.r, row * a.ldr + column(i, j));
                }
        }
    }
    if (NORM) {
        auto row_sum = [&](float v, int which) {
            v = lanes_reduce<(LANES < 64 ? LANES : 64)>(v, [](float a, float b) { return a + b; });
            if (LANES <= 64) return v;
            if ((threadIdx.x & 63) == 0) sh[which][threadIdx.x >> 6] = v;
            __syncthreads();
            return (sh[which][0] + sh[which][1]) + (sh[which][2] + sh[which][3]);
        };
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += z[i][j];
        const float mean = row_sum(s, 0) / (float)a.k;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (lane + i * LANES) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                z[i][j] -= mean;
                if (VEC ? c < a.k : column(i, j) < a.k) s = __builtin_fmaf(z[i][j], z[i][j], s);
            }
        }
        const float inv = 1.f / sqrtf(row_sum(s, 1) / (float)a.k + a.eps);
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (lane + i * LANES) * 8;
            if (VEC) {
                float w[8], b[8];
                if (c < a.k) {
                    fp8_load8<LDOT_F32>(a.w, c, w);
                    fp8_load8<LDOT_F32>(a.b, c, b);
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[i][j] = __builtin_fmaf(z[i][j] * inv, w[j], b[j]);
                    if (a.y) fp8_store8<DT>(a.y, row * a.k + c, z[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[i][j] = 0.f;
                }
            } else if (TOGETHER == 2) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int e = column(i, j);
                    if (e < a.k) {
                        float w0, w1, b0, b1;
                        fp8_load2<LDOT_F32>(a.w, e, w0, w1);
                        fp8_load2<LDOT_F32>(a.b, e, b0, b1);
                        z[i][j] = __builtin_fmaf(z[i][j] * inv, w0, b0);
                        z[i][j + 1] = __builtin_fmaf(z[i][j + 1] * inv, w1, b1);
                        if (a.y) fp8_store2<DT>(a.y, row * a.k + e, z[i][j], z[i][j + 1]);
                    } else {
                        z[i][j] = z[i][j + 1] = 0.f;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = column(i, j);
                    if (e < a.k) {
                        z[i][j] = __builtin_fmaf(z[i][j] * inv, a.w[e], a.b[e]);
                        if (a.y) fp8_store<DT>(a.y, row * a.k + e, z[i][j]);
                    } else {
                        z[i][j] = 0.f;
                    }
                }
            }
        }
    }
    // A value next to the middle between two codes can fall on the wrong side by its own last bits (the difference, the product, the scale, its
    // largest element's two and the quotient: 7 halves of one at most).  Rows that have one within 4 of them are done over in 64 bits, one
    // wave in 85: the codes are those of the exact values (86011 x 768 in bf16: 111 us against 95, no code in 10^6 off instead of one)
    uint32_t border = ~0u;
    const int kb = (a.k + kFp8Block - 1) / kFp8Block;
    uint8_t* const out = (uint8_t*)a.codes + row * a.k;
    constexpr int kOwn = VEC || LANES == 16 ? 8 : 2, kOver = VEC || LANES == 16 ? 16 : 64;      // elements of a block per lane, lanes of a block
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += kOwn) {
            float amax = 0.f;
#pragma unroll
            for (int j = j0; j < j0 + kOwn; ++j) amax = fmaxf(amax, fabsf(z[i][j]));
            amax = lanes_reduce<kOver>(amax, [](float a, float b) { return fmaxf(a, b); });
            const float scale = fp8_scale(amax), inv = fp8_inverse(scale);
            const int c = column(i, j0), blk = c / kFp8Block;
            if (blk >= kb) continue;
            if ((lane & (kOver - 1)) == 0) a.scales[row * kb + blk] = scale;
#pragma unroll
            for (int j = j0; j < j0 + kOwn; ++j) {
                z[i][j] = fp8_scaled(z[i][j], scale, inv);
            }
            if (NORM)
#pragma unroll
                for (int j = j0; j < j0 + kOwn; j += 2)        // (the 20 bits below a code's, less the middle's and 4)
                    border = min(border, min((__float_as_uint(z[i][j]) << 12) - ((0x80000u - 4u) << 12),
                                             (__float_as_uint(z[i][j + 1]) << 12) - ((0x80000u - 4u) << 12)));
            if (VEC) {
                if (c < a.k) *(uint2*)(out + c) = fp8_pack(z[i]);
            } else {
#pragma unroll
                for (int j = j0; j < j0 + kOwn; j += 2) {
                    const int two = __builtin_amdgcn_cvt_pk_fp8_f32(z[i][j], z[i][j + 1], 0, false);
                    const int e = column(i, j), f = column(i, j + 1);
                    if (TOGETHER == 2) {
                        if (e < a.k) *(uint16_t*)(out + e) = (uint16_t)two;
                    } else {
                        if (e < a.k) out[e] = (uint8_t)two;
                        if (f < a.k) out[f] = (uint8_t)(two >> 8);
                    }
                }
            }
        }
    if (!NORM) return;
    const bool over = border < 8u << 12;
    if (LANES > 64 ? !__syncthreads_or(over) : !__any(over)) return;
    __shared__ double wide[2][4];
    auto add = [&](double v, int which) {
        for (int o = 1; o < (LANES < 64 ? LANES : 64); o <<= 1) v += __shfl_xor(v, o);
        if (LANES <= 64) return v;
        if ((threadIdx.x & 63) == 0) wide[which][threadIdx.x >> 6] = v;
        __syncthreads();
        return (wide[which][0] + wide[which][1]) + (wide[which][2] + wide[which][3]);
    };
    // (16-bit operands: their sums are exact in 32 bits but where one is far smaller than the other's last bit)
    typename std::conditional<DT == LDOT_F32, double, float>::type again[ITER][8];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        float x[8] = {}, r[8] = {};
        if (VEC) {
            if (column(i, 0) < a.k) {
                fp8_load8<DT>(a.x, row * a.ldx + column(i, 0), x);
                if (a.r) fp8_load8<DT>(a.r, row * a.ldr + column(i, 0), r);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (column(i, j) < a.k) {
                    x[j] = fp8_load<DT>(a.x, row * a.ldx + column(i, j));
                    if (a.r) r[j] = fp8_load<DT>(a.r, row * a.ldr + column(i, j));
                }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) again[i][j] = DT == LDOT_F32 ? (double)x[j] + (double)r[j] : x[j] + r[j];
    }
    double s = 0.;
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += again[i][j];
    const double mean = add(s, 0) / a.k;
    s = 0.;
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double d = column(i, j) < a.k ? again[i][j] - mean : 0.;
            s = __builtin_fma(d, d, s);
        }
    const double inv = 1. / sqrt(add(s, 1) / a.k + a.eps);
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += kOwn) {
            double y[kOwn], amax = 0.;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                const int e = column(i, j0 + j);
                y[j] = e < a.k ? __builtin_fma((again[i][j0 + j] - mean) * inv, (double)a.w[e], (double)a.b[e]) : 0.;
                amax = fmax(amax, fabs(y[j]));
            }
            for (int o = 1; o < kOver; o <<= 1) amax = fmax(amax, __shfl_xor(amax, o));
            const double scale = amax > 0. ? amax / kFp8Max : 1.;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                const int e = column(i, j0 + j);
                const double v = y[j] / scale;
                float f = __double2float_rz(v);        // (rounded to odd: the rounding to a code then sees on which side v lies)
                if ((double)f != v) f = __uint_as_float(__float_as_uint(f) | 1u);
                if (e < a.k) out[e] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(f, 0.f, 0, false);
            }
        }
}

// one workgroup per block of 128 x 128 (weights: once per model, not on any hot path)
template <int DT>
__global__ __launch_bounds__(256) void quantize_tile_kernel(const void* __restrict__ x, int64_t m, int64_t k, int64_t ld, uint8_t* __restrict__ codes,
                                                            float* __restrict__ scales) {
    __shared__ float sh[4];
    const int64_t r0 = (int64_t)blockIdx.y * kFp8Block, c0 = (int64_t)blockIdx.x * kFp8Block;
    const int64_t c = c0 + (threadIdx.x & 127);
    float amax = 0.f;
    if (c < k)
        for (int64_t r = r0 + (threadIdx.x >> 7); r < min(m, r0 + kFp8Block); r += 2) amax = fmaxf(amax, fabsf(fp8_load<DT>(x, r * ld + c)));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
    const float scale = fp8_scale(amax), inv = fp8_inverse(scale);
    if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = scale;
    if (c < k)
        for (int64_t r = r0 + (threadIdx.x >> 7); r < min(m, r0 + kFp8Block); r += 2)
            codes[r * k + c] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(fp8_scaled(fp8_load<DT>(x, r * ld + c), scale, inv), 0.f, 0, false);
}

template <int DT, int LANES, int ITER, bool NORM, int TOGETHER>
void norm_launch_v(const NormArgs& a, hipStream_t st) {
    // (a launch has fewer than 2^32 threads in x: more rows go on in y)
    const int64_t n = (a.m + 256 / LANES - 1) / (256 / LANES);
    const dim3 grid((unsigned)std::min<int64_t>(n, 1 << 23), (unsigned)((n + (1 << 23) - 1) >> 23));
    hipLaunchKernelGGL((norm_e4m3_kernel<DT, LANES, ITER, NORM, TOGETHER>), grid, dim3(256), 0, st, a);
}

template <int DT, bool NORM, int TOGETHER>
void norm_launch_ragged(const NormArgs& a, int groups, hipStream_t st) {
    // (fp16, before codes were checked, a wave per row against a workgroup: 60000 x 513 96 us and 152, 20000 x 1500 112 and 65, 5000 x 4095 140 and 59)
    if (groups <= 16) norm_launch_v<DT, 16, 1, NORM, TOGETHER>(a, st);
    else if (groups <= 64) norm_launch_v<DT, 64, 1, NORM, TOGETHER>(a, st);
    else if (groups <= 128) norm_launch_v<DT, 64, 2, NORM, TOGETHER>(a, st);
    else if (groups <= 256) norm_launch_v<DT, 256, 1, NORM, TOGETHER>(a, st);
    else if (groups <= 512) norm_launch_v<DT, 256, 2, NORM, TOGETHER>(a, st);
    else if (groups <= 1024) norm_launch_v<DT, 256, 4, NORM, TOGETHER>(a, st);
    else norm_launch_v<DT, 256, 8, NORM, TOGETHER>(a, st);
}

template <int DT, bool NORM>
void norm_launch(const NormArgs& a, int together, hipStream_t st) {
    // up to 64 elements per lane, and as few lanes as leave none idle: rows of 768 take half a wave with three groups each, twice the loads
    // in flight of a whole wave with one and a half
    const int groups = (a.k + 7) / 8;
    if (together == 1) norm_launch_ragged<DT, NORM, 1>(a, groups, st);
    else if (together == 2) norm_launch_ragged<DT, NORM, 2>(a, groups, st);
    else if (groups <= 16) norm_launch_v<DT, 16, 1, NORM, 8>(a, st);
    else if (groups <= 32) norm_launch_v<DT, 32, 1, NORM, 8>(a, st);
    else if (groups <= 64) norm_launch_v<DT, 32, 2, NORM, 8>(a, st);
    else if (groups <= 96) norm_launch_v<DT, 32, 3, NORM, 8>(a, st);
    else if (groups <= 128) norm_launch_v<DT, 32, 4, NORM, 8>(a, st);
    else if (groups <= 192) norm_launch_v<DT, 64, 3, NORM, 8>(a, st);
    else if (groups <= 256) norm_launch_v<DT, 64, 4, NORM, 8>(a, st);
    else if (groups <= 512) norm_launch_v<DT, 64, 8, NORM, 8>(a, st);
    else if (groups <= 1024) norm_launch_v<DT, 256, 4, NORM, 8>(a, st);
    else norm_launch_v<DT, 256, 8, NORM, 8>(a, st);
}

bool on(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <bool NORM>
int norm_entry(const NormArgs& a, int dtype, hipStream_t st) {
    const int64_t es = dtype == LDOT_F32 ? 4 : 2;
    // n elements of every operand at once: rows of a multiple of n, each of whose addresses is one of n elements' bytes (of 16 for eight)
    auto together = [&](int n) {
        const uintptr_t b = std::min<uintptr_t>(n * es, 16), f = std::min<uintptr_t>(n * 4, 16);
        return a.k % n == 0 && on(a.x, b) && a.ldx * es % b == 0 && on(a.codes, n) &&
               (!NORM || (on(a.y, b) && on(a.w, f) && on(a.b, f) && (!a.r || (on(a.r, b) && a.ldr * es % b == 0))));
    };
    const int n = together(8) ? 8 : together(2) ? 2 : 1;
    if (dtype == LDOT_F32) norm_launch<LDOT_F32, NORM>(a, n, st);
    else if (dtype == LDOT_BF16) norm_launch<LDOT_BF16, NORM>(a, n, st);
    else norm_launch<LDOT_F16, NORM>(a, n, st);
    LDOT_HIP_CHECK(hipGetLastError());
    return LDOT_OK;
}

constexpr int64_t kNormWidth = 16384;

}  // namespace
}  // namespace ldot

using namespace ldot;

extern "C" {

int ldot_quantize_e4m3(const void* x, int dtype, int64_t m, int64_t k, int64_t ld, int block_rows, void* codes, float* scales, void* stream) {
    LDOT_REQUIRE(dtype == LDOT_F32 || dtype == LDOT_BF16 || dtype == LDOT_F16, LDOT_EINVAL, "bad dtype %d", dtype);
    LDOT_REQUIRE(m >= 0 && k > 0 && ld >= k && m < (1ll << 31), LDOT_EINVAL, "bad shape %lld x %lld (row stride %lld)", (long long)m, (long long)k, (long long)ld);
    LDOT_REQUIRE(block_rows == 1 || block_rows == kFp8Block, LDOT_EINVAL, "blocks of %d rows: 1 or 128 are supported", block_rows);
    if (m == 0) return LDOT_OK;
    LDOT_REQUIRE(x && codes && scales, LDOT_EINVAL, "NULL buffer");
    hipStream_t st = (hipStream_t)stream;
    if (block_rows == 1) {
        LDOT_REQUIRE(k <= kNormWidth, LDOT_EINVAL, "rows of %lld elements: 16384 at most", (long long)k);
        NormArgs a{};
        a.x = x;
        a.ldx = ld;
        a.m = m;
        a.k = (int)k;
        a.codes = codes;
        a.scales = scales;
        return norm_entry<false>(a, dtype, st);
    }
    const int64_t gx = (k + kFp8Block - 1) / kFp8Block, gy = (m + kFp8Block - 1) / kFp8Block;
    LDOT_REQUIRE(gy <= 65535 && gx < (1ll << 31), LDOT_EINVAL, "weights of %lld x %lld: too many blocks", (long long)m, (long long)k);
    const dim3 grid((unsigned)gx, (unsigned)gy);
    if (dtype == LDOT_F32) hipLaunchKernelGGL(quantize_tile_kernel<LDOT_F32>, grid, dim3(256), 0, st, x, m, k, ld, (uint8_t*)codes, scales);
    else if (dtype == LDOT_BF16) hipLaunchKernelGGL(quantize_tile_kernel<LDOT_BF16>, grid, dim3(256), 0, st, x, m, k, ld, (uint8_t*)codes, scales);
    else hipLaunchKernelGGL(quantize_tile_kernel<LDOT_F16>, grid, dim3(256), 0, st, x, m, k, ld, (uint8_t*)codes, scales);
    LDOT_HIP_CHECK(hipGetLastError());
    return LDOT_OK;
}

int ldot_add_layer_norm_e4m3(const void* x, int64_t ldx, const void* residual, int64_t ldr, int dtype, int64_t m, int64_t k, const float* weight,
                             const float* bias, float eps, void* y, void* codes, float* scales, void* stream) {
    LDOT_REQUIRE(dtype == LDOT_F32 || dtype == LDOT_BF16 || dtype == LDOT_F16, LDOT_EINVAL, "bad dtype %d", dtype);
    LDOT_REQUIRE(m >= 0 && m < (1ll << 31) && k > 0 && k <= kNormWidth && ldx >= k && (!residual || ldr >= k), LDOT_EINVAL,
                 "bad shape %lld x %lld (16384 columns at most)", (long long)m, (long long)k);
    LDOT_REQUIRE(eps >= 0.f, LDOT_EINVAL, "eps has to be >= 0");
    if (m == 0) return LDOT_OK;
    LDOT_REQUIRE(x && weight && bias && codes && scales, LDOT_EINVAL, "NULL buffer");
    NormArgs a{x, residual, ldx, ldr, m, (int)k, weight, bias, eps, y, codes, scales};
    return norm_entry<true>(a, dtype, (hipStream_t)stream);
}

}  // extern "C"
