// Activations and weights into 8 bits (e4m3, a scale for each block of 128), alone or behind the towers' residual norm
// (uniter_model/model/layer.py:103-113,144-154: LayerNorm(dense(x) + residual)):
//     z = x + r,  mean = sum z / k,  var = sum (z - mean)^2 / k,  y = (z - mean) / sqrt(var + eps) * w + b,
//     scale_b = max_{i in block b} |y_i| / 448,  code_i = e4m3(y_i / scale_b)
// A row is read once, kept in registers (mean, then variance around it, then the block's largest value: three passes over registers, none
// over memory) and written once in both forms.  All of it in 64 bits, rounded where it is stored: in 32 bits a mean that is large beside the
// row's spread leaves its own rounding in every value (768 times 1.3 came out as 0.23 instead of 0), and a value next to the middle between two
// codes falls on either side.  64-bit instructions are as fast as 32-bit ones here.  Bound by memory in fp32 (46073 x 768: 95 us, 4.8 TB/s;
// 17277 x 2048: 86 us, 5.4 TB/s); in 16 bits, half the bytes for as many instructions, the vector instructions are busy for 60 % of the time
// beside it (bf16, 86011 x 768: 110 us, 4.2 TB/s; 32087 x 2048: 97 us, 4.75 TB/s; 256696 x 256: 95 us, 4.8 TB/s; 400000 x 64: 60 us, 3.0 TB/s).
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
    double share;        // 1 / k
    void *y, *codes;
    float* scales;
};

// a row per LANES lanes (16 to 64 of a wave, or the whole workgroup).  TOGETHER 8: rows start on 16 bytes and k is a multiple of 8; lane i takes
// the groups of eight elements i, i + LANES, ...: 16 lanes hold one block of 128.  Else neighbouring lanes take neighbouring pairs (TOGETHER 2) or
// elements (1): 16 lanes hold a row of one block, or a wave holds a block at a time, two elements per lane
template <int DT, int LANES, int ITER, bool NORM, int TOGETHER>
__global__ __launch_bounds__(256) void norm_e4m3_kernel(const NormArgs a) {
    constexpr bool VEC = TOGETHER == 8;
    __shared__ double sh[2][4];
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
    typedef typename std::conditional<NORM, double, float>::type V;
    V z[ITER][8];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int c = (lane + i * LANES) * 8;
        auto sum = [&](int j, float x, float r) { z[i][j] = (V)x + (V)r; };
        if (VEC) {
            if (c < a.k) {
                float x[8], r[8];
                fp8_load8<DT>(a.x, row * a.ldx + c, x);
                if (NORM && a.r) {
                    fp8_load8<DT>(a.r, row * a.ldr + c, r);
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum(j, x[j], r[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[i][j] = x[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) z[i][j] = 0;
            }
        } else if (TOGETHER == 2) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float x[2] = {}, r[2] = {};
                if (column(i, j) < a.k) {
                    fp8_load2<DT>(a.x, row * a.ldx + column(i, j), x[0], x[1]);
                    if (NORM && a.r) fp8_load2<DT>(a.r, row * a.ldr + column(i, j), r[0], r[1]);
                }
                sum(j, x[0], r[0]);
                sum(j + 1, x[1], r[1]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float x = 0.f, r = 0.f;
                if (column(i, j) < a.k) {
                    x = fp8_load<DT>(a.x, row * a.ldx + column(i, j));
                    if (NORM && a.r) r = fp8_load<DT>(a.r, row * a.ldr + column(i, j));
                }
                sum(j, x, r);
            }
        }
    }
    if constexpr (NORM) {
        auto row_sum = [&](double v, int which) {
            v = lanes_reduce<(LANES < 64 ? LANES : 64)>(v, [](double a, double b) { return a + b; });
            if (LANES <= 64) return v;
            if ((threadIdx.x & 63) == 0) sh[which][threadIdx.x >> 6] = v;
            __syncthreads();
            return (sh[which][0] + sh[which][1]) + (sh[which][2] + sh[which][3]);
        };
        double s = 0.;
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += z[i][j];
        const double mean = fp8_quotient(row_sum(s, 0), (double)a.k, a.share);
        s = 0.;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            double from = 0.;              // (columns past the row's end stay zeros)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j % TOGETHER == 0) from = column(i, j) < a.k ? mean : 0.;
                z[i][j] -= from;
                s = __builtin_fma(z[i][j], z[i][j], s);
            }
        }
        const double inv = fp8_rsqrt(__builtin_fma(row_sum(s, 1), a.share, (double)a.eps));
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int c = (lane + i * LANES) * 8;
            float y[8];
            auto value = [&](int j, float w, float b) {
                z[i][j] = __builtin_fma(z[i][j] * inv, (double)w, (double)b);
                y[j] = (float)z[i][j];
                asm("" : "+v"(y[j]));      // (rounded to 16 bits from here: in one step from 64 bits it takes seven instructions more)
            };
            if (VEC) {
                if (c < a.k) {
                    float w[8], b[8];
                    fp8_load8<LDOT_F32>(a.w, c, w);
                    fp8_load8<LDOT_F32>(a.b, c, b);
#pragma unroll
                    for (int j = 0; j < 8; ++j) value(j, w[j], b[j]);
                    if (a.y) fp8_store8<DT>(a.y, row * a.k + c, y);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[i][j] = 0.;
                }
            } else if (TOGETHER == 2) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const int e = column(i, j);
                    if (e < a.k) {
                        float w[2], b[2];
                        fp8_load2<LDOT_F32>(a.w, e, w[0], w[1]);
                        fp8_load2<LDOT_F32>(a.b, e, b[0], b[1]);
                        value(j, w[0], b[0]);
                        value(j + 1, w[1], b[1]);
                        if (a.y) fp8_store2<DT>(a.y, row * a.k + e, y[j], y[j + 1]);
                    } else {
                        z[i][j] = z[i][j + 1] = 0.;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = column(i, j);
                    if (e < a.k) {
                        value(j, a.w[e], a.b[e]);
                        if (a.y) fp8_store<DT>(a.y, row * a.k + e, y[j]);
                    } else {
                        z[i][j] = 0.;
                    }
                }
            }
        }
    }
    const int kb = (a.k + kFp8Block - 1) / kFp8Block;
    uint8_t* const out = (uint8_t*)a.codes + row * a.k;
    constexpr int kOwn = VEC || LANES == 16 ? 8 : 2, kOver = VEC || LANES == 16 ? 16 : 64;      // elements of a block per lane, lanes of a block
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += kOwn) {
            V amax = 0;
#pragma unroll
            for (int j = j0; j < j0 + kOwn; ++j) {
                if constexpr (NORM) amax = fp8_larger(amax, z[i][j]);
                else amax = fmaxf(amax, fabsf(z[i][j]));
            }
            amax = lanes_reduce<kOver>(amax, [](V a, V b) {
                if constexpr (NORM) return fp8_larger(a, b);
                else return fmaxf(a, b);
            });
            const int c = column(i, j0), blk = c / kFp8Block;
            if (blk >= kb) continue;
            float v[kOwn];
            if constexpr (NORM) {
                // (what is stored is the scale in 32 bits, off by 2^-24 of it; where that is no normal number, the codes are made with it)
                const double exact = amax < 1e300 ? amax > 0. ? fp8_quotient(amax, (double)kFp8Max, 1. / kFp8Max) : 1. : amax;
                const bool coarse = (float)exact < 1.17549435e-38f;
                const float scale = (float)exact > 0.f ? (float)exact : 1.f;
                const double by = coarse ? (double)scale : exact, undo = by < 1e300 ? by : 0., inv = fp8_reciprocal(by, undo);
                if ((lane & (kOver - 1)) == 0) a.scales[row * kb + blk] = scale;
#pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    v[j] = fp8_cut(fp8_quotient(z[i][j0 + j], undo, inv));      // (infinite scales: 0, and NaN for what is infinite too)
                }
                if (__any(coarse)) {
#pragma unroll
                    for (int j = 0; j < kOwn; ++j) v[j] = fp8_limit(v[j]);
                }
            } else {
                const float scale = fp8_scale(amax), inv = fp8_inverse(scale);
                if ((lane & (kOver - 1)) == 0) a.scales[row * kb + blk] = scale;
#pragma unroll
                for (int j = 0; j < kOwn; ++j) v[j] = fp8_scaled(z[i][j0 + j], scale, inv);
            }
            if constexpr (VEC) {
                if (c < a.k) *(uint2*)(out + c) = fp8_pack(v);
            } else {
#pragma unroll
                for (int j = 0; j < kOwn; j += 2) {
                    const int two = __builtin_amdgcn_cvt_pk_fp8_f32(v[j], v[j + 1], 0, false);
                    const int e = column(i, j0 + j), f = column(i, j0 + j + 1);
                    if (TOGETHER == 2) {
                        if (e < a.k) *(uint16_t*)(out + e) = (uint16_t)two;
                    } else {
                        if (e < a.k) out[e] = (uint8_t)two;
                        if (f < a.k) out[f] = (uint8_t)(two >> 8);
                    }
                }
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
    // (norm of 460 MB in bf16, us: 513 columns 64 x 2 241, 256 x 1 358; 1022 64 x 2 143, 256 x 1 193; 1500 256 x 1 174, 64 x 4 208; 4095 256 x 2 227, 256 x 4 387)
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
    // As few elements per lane as leave few lanes idle: registers are what limits the loads in flight (norm of 460 MB in bf16, us: 512 columns
    // 64 x 1 93, 32 x 2 94, 16 x 4 109; 768 32 x 3 109, 64 x 2 116; 1024 64 x 2 94, 32 x 4 108; 1536 256 x 1 107, 64 x 3 108 (fp32 86 and 96);
    // 2048 256 x 1 95, 64 x 4 110; 4096 256 x 2 104, 256 x 4 123, 64 x 8 151).  Without the norm a value is 32 bits (512 columns 32 x 2 82, 64 x 1 87;
    // 1536 64 x 3 81, 256 x 1 95; 4096 256 x 2 79, 64 x 8 102)
    const int groups = (a.k + 7) / 8;
    if (together == 1) norm_launch_ragged<DT, NORM, 1>(a, groups, st);
    else if (together == 2) norm_launch_ragged<DT, NORM, 2>(a, groups, st);
    else if (groups <= 16) norm_launch_v<DT, 16, 1, NORM, 8>(a, st);
    else if (groups <= 32) norm_launch_v<DT, 32, 1, NORM, 8>(a, st);
    else if (groups <= 64) norm_launch_v<DT, NORM ? 64 : 32, NORM ? 1 : 2, NORM, 8>(a, st);
    else if (groups <= 96) norm_launch_v<DT, 32, 3, NORM, 8>(a, st);
    else if (groups <= 128) norm_launch_v<DT, 64, 2, NORM, 8>(a, st);
    else if (groups <= 192) norm_launch_v<DT, NORM ? 256 : 64, NORM ? 1 : 3, NORM, 8>(a, st);
    else if (groups <= 256) norm_launch_v<DT, NORM ? 256 : 64, NORM ? 1 : 4, NORM, 8>(a, st);
    else if (groups <= 512) norm_launch_v<DT, 256, 2, NORM, 8>(a, st);
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

// rows are read and written by different workgroups in any order: what is written must not be read.  (An operand that lies exactly where y does
// is another matter: a row is read as a whole by those who then write it.)
int64_t rows_bytes(int64_t m, int64_t k, int64_t ld, int64_t size) { return ((m - 1) * ld + k) * size; }
bool apart(const void* a, int64_t bytes_a, const void* b, int64_t bytes_b) {
    return !a || !b || (uintptr_t)a + (uintptr_t)bytes_a <= (uintptr_t)b || (uintptr_t)b + (uintptr_t)bytes_b <= (uintptr_t)a;
}

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
    const int64_t es = dtype == LDOT_F32 ? 4 : 2, in = rows_bytes(m, k, ld, es), nscales = (m + block_rows - 1) / block_rows * ((k + kFp8Block - 1) / kFp8Block);
    LDOT_REQUIRE(apart(codes, m * k, x, in) && apart(scales, nscales * 4, x, in) && apart(codes, m * k, scales, nscales * 4), LDOT_EINVAL,
                 "codes or scales overlap another tensor");
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
    {
        const int64_t es = dtype == LDOT_F32 ? 4 : 2, ny = m * k * es, ns = m * ((k + kFp8Block - 1) / kFp8Block) * 4;
        const int64_t nx = rows_bytes(m, k, ldx, es), nr = rows_bytes(m, k, ldr, es);
        struct Part { const void* p; int64_t n; } in[4] = {{x, nx}, {residual, nr}, {weight, k * 4}, {bias, k * 4}}, out[3] = {{y, ny}, {codes, m * k}, {scales, ns}};
        for (int i = 0; i < 3; ++i) {
            for (int j = 0; j < 4; ++j) {
                const bool place = i == 0 && j < 2 && in[j].p == y && (m == 1 || (j ? ldr : ldx) == k);
                LDOT_REQUIRE(place || apart(out[i].p, out[i].n, in[j].p, in[j].n), LDOT_EINVAL, "y, codes or scales overlap another tensor");
            }
            for (int j = i + 1; j < 3; ++j) LDOT_REQUIRE(apart(out[i].p, out[i].n, out[j].p, out[j].n), LDOT_EINVAL, "y, codes or scales overlap each other");
        }
    }
    NormArgs a{x, residual, ldx, ldr, m, (int)k, weight, bias, eps, 1. / (double)k, y, codes, scales};
    return norm_entry<true>(a, dtype, (hipStream_t)stream);
}

}  // extern "C"
