// Product of 8-bit activations and weights (e4m3, scales per 1 x 128 and per 128 x 128):
//     out[m][n] = act( sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k]  + bias[n] )
// One v_mfma_f32_16x16x128 takes exactly one block of 128: its result is that block's sum of exact products, which is scaled into the
// fp32 accumulator — the scales cost one vector fma per result element and block, beside the matrix pipe.
// The 8-bit matrix instructions add the products of 8 consecutive k in fixed point, aligned to the largest of the 8, and drop what lies
// below 2^-13 of it (measured, product by product; the groups are then added in fp32).  On normally distributed data that is 2.5e-5 of
// the result: 1/60 of the rounding to bf16, 1/8 of that to fp16.  Results in fp32 do not take it: their codes are widened to bf16 in
// registers (exact) and multiplied by v_mfma_f32_16x16x32_bf16, which keeps fp32 sums, at half the rate (8192 x 4096 x 4096: 316 us, 870
// TFLOP/s, 72 % of the library's bf16 product).
// Weights are the MFMA's A operand: a lane then holds 4 consecutive output columns of ONE row, so both scales of its results are one
// number per 16 rows.
#include <algorithm>

#include "fp8_common.h"

namespace ldot {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(4))) float* const_floats;      // (read through the scalar cache: the kernel does not write them)

struct LinearArgs {
    const char *x, *w;
    const float *xs, *ws, *bias;
    void* out;
    int64_t ldx;
    int64_t m;
    int n, k, kb;        // kb: blocks of 128
};

// operand of one block of 128: 32 codes of a row per lane, or the same widened to bf16
template <bool WIDE>
struct Fp8Frag {
    i32x8 v;
    __device__ __forceinline__ void set(i32x4 lo, i32x4 hi) { v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
};
template <>
struct Fp8Frag<true> {
    bf16x8_t v[4];
    __device__ __forceinline__ void set(i32x4 lo, i32x4 hi) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned w = (unsigned)(q < 2 ? lo : hi)[(2 * q + h) & 3];
                const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true);
                v[q][4 * h] = a[0];
                v[q][4 * h + 1] = a[1];
                v[q][4 * h + 2] = b[0];
                v[q][4 * h + 3] = b[1];
            }
    }
};
__device__ __forceinline__ f32x4 fp8_mma(const Fp8Frag<false>& a, const Fp8Frag<false>& b) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, zero, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 fp8_mma(const Fp8Frag<true>& a, const Fp8Frag<true>& b) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], c, 0, 0, 0);
    return c;
}

// erf-GELU, x Phi(x).  fp32 results: the library's erf.  16-bit results: Phi(-t) = 2^p(t) on [0, 6] with p of degree 7, fitted to
// log2 Phi(-t) so that Phi is off by 5e-7 at most and by 2.6e-5 of itself in the tail; then x Phi(x) = max(x, 0) - |x| Phi(-|x|) (no
// cancellation).  Beyond 6 the second term, 6e-9 and less, stays where it is.  (16384 x 8192 results: 28 us instead of 63 for a
// reciprocal, five terms and an exponential.)
template <int ODT>
__device__ __forceinline__ float fp8_gelu(float x) {
    if (ODT == LDOT_F32) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    const float t = fminf(fabsf(x), 6.f);
    float p = __builtin_fmaf(-1.37215324e-6f, t, 5.26263694e-5f);
    p = __builtin_fmaf(p, t, -8.63727445e-4f);
    p = __builtin_fmaf(p, t, 8.2694537e-3f);
    p = __builtin_fmaf(p, t, -5.3544786e-2f);
    p = __builtin_fmaf(p, t, -4.58783773e-1f);
    p = __builtin_fmaf(p, t, -1.15116653f);
    p = __builtin_fmaf(p, t, -9.99998639e-1f);
    return __builtin_fmaf(-t, __builtin_amdgcn_exp2f(p), __builtin_fmaf(fabsf(x), 0.5f, 0.5f * x));
}

// four consecutive columns: bias and activation
template <int ODT, bool GELU>
__device__ __forceinline__ f32x4 linear_finish(f32x4 v, f32x4 bias) {
    v += bias;
    if (GELU)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = fp8_gelu<ODT>(v[r]);
    return v;
}
__device__ __forceinline__ f32x4 linear_bias(const LinearArgs& a, int col) {
    f32x4 b = {0.f, 0.f, 0.f, 0.f};
    if (a.bias)
#pragma unroll
        for (int r = 0; r < 4; ++r) b[r] = a.bias[min(col + r, a.n - 1)];
    return b;
}
template <int ODT>
struct LinearOut {
    static constexpr int E = ODT == LDOT_F32 ? 4 : 2;
    // four results as they lie in memory
    static __device__ __forceinline__ void put4(char* p, f32x4 v) {
        if (ODT == LDOT_F32) {
            *(f32x4*)p = v;
        } else {
            union {
                uint2 u;
                __bf16 b[4];
                _Float16 h[4];
            } o;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (ODT == LDOT_BF16) o.b[r] = (__bf16)v[r];
                else o.h[r] = (_Float16)v[r];
            *(uint2*)p = o.u;
        }
    }
    static __device__ __forceinline__ void copy(char* to, const char* from) {     // one result
        if (E == 4) *(uint32_t*)to = *(const uint32_t*)from;
        else *(uint16_t*)to = *(const uint16_t*)from;
    }
    static __device__ __forceinline__ void put(const LinearArgs& a, int64_t row, int col, f32x4 v, bool vec) {
        const int64_t at = row * a.n + col;
        if (vec && col + 3 < a.n) {
            put4((char*)a.out + at * E, v);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (col + r < a.n) fp8_store<ODT>(a.out, at + r, v[r]);
        }
    }
};

// ---- many rows: tiles of (16 TM WM) rows x (16 TN WN) columns through LDS ---------------------------------------------------------------
// A K block of a panel lies in LDS as rows of 128 bytes; 16-byte chunk c of row r at place c ^ (r & 6).  A fragment takes chunks g and g + 4
// of its row (g: the lane's group; which k a lane holds is free as long as both operands agree): the 16 lanes that LDS serves at once, 8 rows
// of two groups, then hit every bank once (0 conflicts counted; chunks 2 g and 2 g + 1 took twice the cycles, with any permutation).  The
// permutation is applied to the SOURCE address of the direct-to-LDS loads (16 bytes per lane,
// 8 rows per instruction).
template <int WM, int WN, int TM, int TN>
struct LinearTile {
    static constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
    static constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
    static constexpr int kX = BM * 128, kStage = (BM + BN) * 128, kScales = 2 * kStage, kLds = kScales + BM * 128;
    static constexpr int kPieces = (BM + BN) / 8;              // 1 KiB loads of a stage
};

// a tile of results: its first row and column, and how many it has
struct LinearPlace {
    int64_t m0;
    int n0, rows_m, rows_n;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t linear_buffer(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000);
}

// threadIdx.x, made anew: what is computed from it behind a tile's products is not kept in registers beside them
__device__ __forceinline__ int linear_thread() {
    int t = (int)threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// A workgroup works on one tile after another: the next tile's first block of codes is loaded under the last block's products, and its
// second one, like the stores of the results, under the first block's.  (m x k x n, bf16 results: 21513 x 768 x 2304 50 us against 63 with a
// workgroup per tile, 86011 x 768 x 768 66 against 84, 8192^3 467 against 515: 2360 TFLOP/s, 87 % of the library's product without scales.)
// Bound by the matrix pipe where k is long, by the results' bytes where it is short (21513 x 128 x 2304: 28 us, 3.6 TB/s).
template <int WM, int WN, int TM, int TN, int ODT, bool GELU>
__global__ __launch_bounds__(WM* WN * 64, 2) void linear_tile_kernel(const LinearArgs a, int tiles_m, int tiles_n, int vec_arg) {
    const bool vec = vec_arg != 0;
    typedef LinearTile<WM, WN, TM, TN> G;
    typedef Fp8Frag<ODT == LDOT_F32> Frag;
    typedef LinearOut<ODT> Out;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    // an XCD (blockIdx % 8) takes a contiguous eighth of the tiles; inside it, 8 tiles of rows under each tile of columns share the
    // weight panel, and the activations' panels stay in the XCD's L2
    const unsigned n_all = (unsigned)tiles_m * (unsigned)tiles_n, xcd = blockIdx.x % 8, step = gridDim.x / 8;
    const unsigned first = xcd * (n_all / 8) + min(xcd, n_all % 8), count = n_all / 8 + (xcd < n_all % 8 ? 1u : 0u);
    unsigned id = blockIdx.x / 8;
    if (id >= count) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int wm = wave % WM, wn = wave / WM;
    const int src_row = lane >> 3, src_col = ((lane & 7) ^ (src_row & 6)) << 4;   // (a piece is 8 rows)
    const int vx = src_row * (int)a.ldx + src_col, vw = src_row * a.k + src_col;
    constexpr int kMine = G::kPieces / G::kWaves, kMineX = G::BM / 8 / G::kWaves;

    auto place = [&](unsigned i) {
        const unsigned at = first + i, band = 8u * (unsigned)tiles_n, b0 = at / band, in = at % band, high = min(8u, (unsigned)tiles_m - b0 * 8u);
        LinearPlace t;
        t.m0 = (int64_t)(b0 * 8u + in % high) * G::BM;
        t.n0 = (int)(in / high) * G::BN;
        t.rows_m = (int)min((int64_t)G::BM, a.m - t.m0);
        t.rows_n = min(G::BN, a.n - t.n0);
        return t;
    };
    // A whole tile's loads keep one offset per lane, piece and K block ride in the scalar offset.  At the edges (rows past the panel repeat
    // its last one: their results are not written; chunks past k repeat the row's first one and are cleared in LDS before they are used)
    // the offset is made anew for every load.
    auto issue = [&](const LinearPlace& t, int kb, int buf, int p0, int p1) {            // pieces p0 .. p1 - 1 of this wave
        char* st = lds + buf * G::kStage + wave * 1024;
        const int k0 = kb * 128;
        const __amdgpu_buffer_rsrc_t rx = linear_buffer(a.x + t.m0 * a.ldx, (int)((t.rows_m - 1) * a.ldx + a.k));
        const __amdgpu_buffer_rsrc_t rw = linear_buffer(a.w + (int64_t)t.n0 * a.k, t.rows_n * a.k);
        if (t.rows_m == G::BM && t.rows_n == G::BN && k0 + 128 <= a.k) {
#pragma unroll
            for (int p = p0; p < p1; ++p) {
                const int row = (p * G::kWaves + wave - (p < kMineX ? 0 : G::BM / 8)) * 8;
                if (p < kMineX) __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr)(st + p * G::kWaves * 1024), 16, vx, row * (int)a.ldx + k0, 0, 0);
                else __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr)(st + p * G::kWaves * 1024), 16, vw, row * a.k + k0, 0, 0);
            }
        } else {
            const int col = k0 + src_col < a.k ? k0 + src_col : 0;
#pragma unroll
            for (int p = p0; p < p1; ++p) {
                const int row = (p * G::kWaves + wave - (p < kMineX ? 0 : G::BM / 8)) * 8 + src_row;
                if (p < kMineX) __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr)(st + p * G::kWaves * 1024), 16, min(row, t.rows_m - 1) * (int)a.ldx + col, 0, 0, 0);
                else __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr)(st + p * G::kWaves * 1024), 16, min(row, t.rows_n - 1) * a.k + col, 0, 0, 0);
            }
        }
    };
    const int tail = a.k % 128;
    auto clear_tail = [&](int buf, int tid) {                                         // the last block's chunks past k (8 places per row)
        char* st = lds + buf * G::kStage;
        for (int i = tid; i < (G::BM + G::BN) * 8; i += G::kThreads) {
            const int row = i >> 3, c = i & 7;
            if (c * 16 >= tail) *(i32x4*)(st + row * 128 + ((c ^ (row & 6)) << 4)) = i32x4{0, 0, 0, 0};
        }
    };
    const int r = lane & 15, c0 = (g ^ (r & 6)) << 4, c1 = c0 ^ 64;
    auto frag = [&](const char* panel, int row0) {
        const char* p = panel + (row0 + r) * 128;
        Frag f;
        f.set(*(const i32x4*)(p + c0), *(const i32x4*)(p + c1));
        return f;
    };
    // The rows' scales lie in LDS too (read where they are, every one of them was a cache line of its own: as many requests as the codes), 16
    // blocks at a time and the next 16 on their way, the next tile's first ones among them.  Scale b of row r at word 16 r + (b ^ r) % 16:
    // 16 rows are 16 banks
    float* const scales = (float*)(lds + G::kScales);
    const int srow = wm * TM * 16 + r;
    auto scales_issue = [&](const LinearPlace& t, int kb, int half, int l) {          // those of blocks kb to kb + 15, past the last one its own
        const __amdgpu_buffer_rsrc_t rs = linear_buffer(a.xs + t.m0 * a.kb, t.rows_m * a.kb * 4);
        char* const to = (char*)(scales + half * G::BM * 16);
#pragma unroll
        for (int p = 0; p < G::BM / 4 / G::kWaves; ++p) {                             // (64 words a load: four rows)
            const int four = p * G::kWaves + wave, row = 4 * four + (l >> 4), b = (l ^ row) & 15;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(to + four * 256), 4, (min(row, t.rows_m - 1) * a.kb + min(kb + b, a.kb - 1)) * 4, 0, 0, 0);
        }
    };

    LinearPlace cur = place(id);
    int even = 0, half = 0;                            // the buffers of the tile's even blocks, and of its first scales
    issue(cur, 0, 0, 0, kMine);
    scales_issue(cur, 0, 0, lane);
    if (a.kb > 1) issue(cur, 1, 1, 0, kMine);          // (both buffers are free: the second block's loads do not wait for the first's)
    if (a.kb > 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kMine) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    for (;;) {
        if (a.kb == 1 && tail) {
            clear_tail(even, linear_thread());
            __syncthreads();
        }
        const bool last = id + step >= count;
        const LinearPlace next = place(last ? id : id + step);
        const int wrow = cur.n0 + wn * TN * 16;                      // this wave's first column: its columns lie in one block of 128
        const const_floats wsp = (const_floats)(a.ws + (int64_t)min(wrow / kFp8Block, (a.n - 1) / kFp8Block) * a.kb);
        f32x4 acc[TN][TM], part[2][TM];
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int t = 0; t < TM; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        float s_old[TM], s[TM];
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            s[t] = 0.f;
            part[1][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        Frag xf[TM], wf[2];
#pragma unroll
        for (int t = 0; t < TM; ++t) xf[t] = frag(lds + even * G::kStage, wm * TM * 16 + t * 16);
        wf[0] = frag(lds + even * G::kStage + G::kX, wn * TN * 16);
        // Per step: one fragment of weights against all of activations.  Fragments are read a step ahead; the results of a step are scaled
        // into the accumulators during the next one, an fma each while the matrix pipe works.  All of a block's reads are done a step before
        // its end: the barrier stands there, and behind it the next block's first fragments are read and its successor's loads go out, under
        // the matrix instructions that are left.
        for (int kb = 0; kb < a.kb; ++kb) {
            const int buf = (kb & 1) ^ even;
            const char* st = lds + buf * G::kStage;
            const char* nx = lds + (buf ^ 1) * G::kStage;
            const bool more = kb + 1 < a.kb;
            const int now = half ^ ((kb >> 4) & 1);
            if (kb % 16 == 8 && kb + 8 < a.kb) scales_issue(cur, kb + 8, now ^ 1, linear_thread() & 63);
            const float ws = wsp[kb];
#pragma unroll
            for (int t = 0; t < TM; ++t) {
                s_old[t] = s[t];
                s[t] = scales[now * G::BM * 16 + (srow + 16 * t) * 16 + ((kb ^ (srow + 16 * t)) & 15)] * ws;
            }
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                if (i == TN - 1 && more) {
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    if (tail && kb + 2 == a.kb) {
                        clear_tail(buf ^ 1, linear_thread());
                        __syncthreads();
                    }
                }
                // (behind the last block nothing is left to read: its own first fragments once more, unused)
                wf[(i + 1) & 1] = frag((i + 1 < TN || !more ? st : nx) + G::kX, (wn * TN + (i + 1) % TN) * 16);
#pragma unroll
                for (int t = 0; t < TM; ++t) {
                    __builtin_amdgcn_sched_barrier(0);
                    part[i & 1][t] = fp8_mma(wf[i & 1], xf[t]);
                    if (i == TN - 1) xf[t] = frag(more ? nx : st, wm * TM * 16 + t * 16);
                    const int j = (i + TN - 1) % TN;              // the step before (of the block before)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][t][e] = __builtin_fmaf(part[(i + 1) & 1][t][e], i == 0 ? s_old[t] : s[t], acc[j][t][e]);
                    asm volatile("" : "+v"(acc[j][t]));           // (here, not behind the barrier: the partial sums' registers are needed)
                    // the loads go out a quarter per step, from behind the barrier on: all at once they fill the address queue and every
                    // wave waits to issue (16384 x 4096 x 8192: 735 us against 785)
                    if (t == 1 && i < 3 && kb > 0 && more) issue(cur, kb + 1, buf ^ 1, kMine * (i + 1) / 4, kMine * (i + 2) / 4);
                    if (t == 1 && i == TN - 1 && kb + 2 < a.kb) issue(cur, kb + 2, buf, 0, kMine / 4);
                    if (t == 1 && i < 4 && !more && !last) issue(next, 0, buf ^ 1, kMine * i / 4, kMine * (i + 1) / 4);
                    if (t == 2 && i == 0 && !more && !last) scales_issue(next, 0, now ^ 1, linear_thread() & 63);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int t = 0; t < TM; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[TN - 1][t][e] = __builtin_fmaf(part[(TN - 1) & 1][t][e], s[t], acc[TN - 1][t][e]);
        // The results are turned through the last block's place in LDS, each wave's through a part of its own, so that memory sees whole rows
        // in 16-byte stores: stored from where they are, 32 bytes of 16 rows each, the results of a 256 x 256 tile took 30 us, as long as
        // 32 blocks of products.
        const int lane2 = linear_thread() & 63, r2 = lane2 & 15, g2 = lane2 >> 4;
        constexpr int kBias = TN * 16 / 64;
        float bias_in[kBias];
#pragma unroll
        for (int i = 0; i < kBias; ++i) bias_in[i] = a.bias ? a.bias[min(wrow + i * 64 + lane2, a.n - 1)] : 0.f;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                  // (every wave is done with the last block)
        const int gone = (a.kb - 1) & 1 ? even ^ 1 : even;
        constexpr int kRowBytes = TN * 16 * Out::E, kRowChunks = kRowBytes / 16, kSpace = G::kStage / G::kWaves, kAtOnce = kSpace / kRowBytes / 16;
        static_assert(kAtOnce >= 1 && TM % kAtOnce == 0 && kRowChunks >= 8, "a wave's part does not fit its results");
        char* const mine = lds + gone * G::kStage + wave * kSpace;
        f32x4 bias[TN];
#pragma unroll
        for (int i = 0; i < kBias; ++i) ((float*)mine)[i * 64 + lane2] = bias_in[i];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < TN; ++i) bias[i] = *(const f32x4*)(mine + (i * 16 + 4 * g2) * 4);
        __builtin_amdgcn_wave_barrier();
        const int first_row = wm * TM * 16;
        char* const out = (char*)a.out + ((cur.m0 + first_row) * a.n + wrow) * Out::E;
        const int rows = cur.rows_m - first_row, bytes = (a.n - wrow) * Out::E;
#pragma unroll
        for (int t0 = 0; t0 < TM; t0 += kAtOnce) {
#pragma unroll
            for (int t = t0; t < t0 + kAtOnce; ++t)
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    const int row = (t - t0) * 16 + r2, col = i * 16 + 4 * g2;
                    const f32x4 v = linear_finish<ODT, GELU>(acc[i][t], bias[i]);
                    Out::put4(mine + row * kRowBytes + (((col * Out::E >> 4) ^ (row & 7)) << 4) + (col * Out::E & 15), v);
                }
            // the next tile's first block of codes and its scales, which were asked for under the last block's products
            if (t0 == 0 && !last) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
            if (vec) {
#pragma unroll
                for (int q = 0; q < kAtOnce * 16 * kRowChunks / 64; ++q) {
                    const int idx = lane2 + 64 * q, row = idx / kRowChunks, c = idx % kRowChunks;
                    if (t0 * 16 + row < rows && c * 16 < bytes)
                        *(uint4*)(out + (int64_t)(t0 * 16 + row) * a.n * Out::E + c * 16) = *(const uint4*)(mine + row * kRowBytes + ((c ^ (row & 7)) << 4));
                }
            } else {                                   // (rows that begin anywhere: element by element)
#pragma unroll 2
                for (int idx = lane2; idx < kAtOnce * 16 * TN * 16; idx += 64) {
                    const int row = idx / (TN * 16), at = idx % (TN * 16) * Out::E;
                    if (t0 * 16 + row < rows && at < bytes)
                        Out::copy(out + (int64_t)(t0 * 16 + row) * a.n * Out::E + at, mine + row * kRowBytes + (((at >> 4) ^ (row & 7)) << 4) + (at & 15));
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        if (last) break;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        even = gone ^ 1;
        half ^= (((a.kb - 1) >> 4) & 1) ^ 1;
        cur = next;
        id += step;
        if (a.kb > 1) issue(cur, 1, gone, 0, kMine);
    }
}

// ---- few results: 16 columns x up to 64 rows per workgroup, the K blocks dealt to its 8 waves and joined through LDS in a fixed order ---------
// Bound by the weights' bytes and by latency: operands go straight from memory to the MFMA's registers.
template <int TM, int ODT, bool GELU>
__global__ __launch_bounds__(512) void linear_few_kernel(const LinearArgs a, int vec) {
    typedef Fp8Frag<ODT == LDOT_F32> Frag;
    __shared__ f32x4 part[8][TM][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int n0 = (int)blockIdx.x * 16;
    const int64_t m0 = (int64_t)blockIdx.y * (16 * TM);
    const float* wsp = a.ws + (int64_t)(n0 / kFp8Block) * a.kb;
    const char* wp = a.w + (int64_t)min(n0 + r, a.n - 1) * a.k + g * 32;
    const char* xp[TM];
    const float* xsp[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const int64_t row = min(m0 + t * 16 + r, a.m - 1);        // (rows past the end repeat the last one and are not written)
        xp[t] = a.x + row * a.ldx + g * 32;
        xsp[t] = a.xs + row * a.kb;
    }
    f32x4 acc[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](const char* p, int kb) {
        const int left = a.k - kb * 128 - g * 32;                 // bytes of this lane's 32 that there are
        Frag f;
        f.set(left >= 16 ? *(const i32x4*)(p + kb * 128) : i32x4{0, 0, 0, 0}, left >= 32 ? *(const i32x4*)(p + kb * 128 + 16) : i32x4{0, 0, 0, 0});
        return f;
    };
    for (int kb = wave; kb < a.kb; kb += 8) {
        const Frag wf = load(wp, kb);
        const float ws = wsp[kb];
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const f32x4 p = fp8_mma(wf, load(xp[t], kb));
            const float s = xsp[t][kb] * ws;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(p[e], s, acc[t][e]);
        }
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < TM; t += 8) {
        f32x4 v = part[0][t][lane];
#pragma unroll
        for (int w = 1; w < 8; ++w) v += part[w][t][lane];
        const int64_t row = m0 + t * 16 + r;
        const int col = n0 + 4 * g;
        if (row < a.m && col < a.n) LinearOut<ODT>::put(a, row, col, linear_finish<ODT, GELU>(v, linear_bias(a, col)), vec);
    }
}

template <int WM, int WN, int TM, int TN, int ODT, bool GELU>
int launch_tile(const LinearArgs& a, int vec, hipStream_t st) {
    typedef LinearTile<WM, WN, TM, TN> G;
    static bool flags[kAttrDevices];
    LDOT_HIP_CHECK(set_max_dynamic_lds_once((const void*)linear_tile_kernel<WM, WN, TM, TN, ODT, GELU>, G::kLds, flags));
    const int64_t tm = (a.m + G::BM - 1) / G::BM, tn = (a.n + G::BN - 1) / G::BN;
    LDOT_REQUIRE(tm * tn < (1ll << 31), LDOT_EINVAL, "too many tiles");
    const int64_t at_once = 256 * ((160 << 10) / G::kLds);       // workgroups that fit on the chip's 256 CUs, a multiple of 8
    hipLaunchKernelGGL((linear_tile_kernel<WM, WN, TM, TN, ODT, GELU>), dim3((unsigned)std::min(round_up(tm * tn, 8), at_once)), dim3(G::kThreads), G::kLds, st, a,
                       (int)tm, (int)tn, vec);
    LDOT_HIP_CHECK(hipGetLastError());
    return LDOT_OK;
}

template <int ODT, bool GELU>
int launch_linear(const LinearArgs& a, int vec, hipStream_t st) {
    // Few results: operands straight from memory, 7.9e7 multiplications per us whatever the shape, where a single 128 x 128 tile takes 2 us and
    // 1.4 us per block of k.  Both grow with k: the border lies at 10^6 results (m x n, k 768: 1000 x 768 9.6 us
    // against 10.5, 1000 x 2304 22 against 11; k 4096: 300 x 768 15 against 36).
    // As many rows per workgroup as leave 192 of them (128 x 768, k 4096: 32 rows 9.6 us, 64 rows 15.2; 300 x 768: 17.1 and 15.4)
    if (a.m * a.n <= 1000000) {
        const unsigned gn = (unsigned)((a.n + 15) / 16);
        auto groups = [&](int rows) { return dim3(gn, (unsigned)((a.m + rows - 1) / rows)); };
        auto enough = [&](int rows) { return (int64_t)gn * ((a.m + rows - 1) / rows) >= 192; };
        if (enough(64)) hipLaunchKernelGGL((linear_few_kernel<4, ODT, GELU>), groups(64), dim3(512), 0, st, a, vec);
        else if (enough(32)) hipLaunchKernelGGL((linear_few_kernel<2, ODT, GELU>), groups(32), dim3(512), 0, st, a, vec);
        else hipLaunchKernelGGL((linear_few_kernel<1, ODT, GELU>), groups(16), dim3(512), 0, st, a, vec);
        LDOT_HIP_CHECK(hipGetLastError());
        return LDOT_OK;
    }
    if constexpr (ODT != LDOT_F32) {              // (a wave's widened operands and 32 result tiles do not fit the registers)
        // rounds of the chip: 256 large tiles take 1.15 times as long as 512 small ones (two per CU, whose last round is only partly idle):
        // 16000 x 768, k 768: 20.5 us against 23.3 (189 tiles); 2000 x 4096, k 1024: 22.3 against 19.7 (128 tiles)
        const int64_t large = ((a.m + 255) / 256) * ((a.n + 255) / 256), small = ((a.m + 127) / 128) * ((a.n + 127) / 128);
        const double rounds_large = 1.15 * (double)((large + 255) / 256), x = (double)small / 512, rounds_small = ((double)((small + 511) / 512) + x) / 2;
        if (rounds_large < rounds_small) return launch_tile<4, 2, 4, 8, ODT, GELU>(a, vec, st);
    }
    return launch_tile<2, 2, 4, 4, ODT, GELU>(a, vec, st);
}

}  // namespace
}  // namespace ldot

using namespace ldot;

extern "C" int ldot_linear_e4m3(const void* x, const float* x_scale, int64_t ldx, const void* w, const float* w_scale, const float* bias, int gelu,
                                int64_t m, int64_t n, int64_t k, void* out, int out_dtype, void* stream) {
    LDOT_REQUIRE(out_dtype == LDOT_F32 || out_dtype == LDOT_BF16 || out_dtype == LDOT_F16, LDOT_EINVAL, "bad dtype %d", out_dtype);
    LDOT_REQUIRE(m >= 0 && m < (1ll << 31) && n > 0 && n <= (1 << 24) && k > 0 && k <= (1 << 20) && k % 16 == 0 && ldx >= k && ldx <= (1 << 22) && ldx % 16 == 0,
                 LDOT_EINVAL, "bad shape: m %lld, n %lld, k %lld, row stride %lld (k and the stride: multiples of 16)", (long long)m, (long long)n,
                 (long long)k, (long long)ldx);
    if (m == 0) return LDOT_OK;
    LDOT_REQUIRE(x && x_scale && w && w_scale && out, LDOT_EINVAL, "NULL buffer");
    LDOT_REQUIRE((uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0, LDOT_EINVAL, "codes have to be aligned to 16 bytes");
    LinearArgs a{(const char*)x, (const char*)w, x_scale, w_scale, bias, out, ldx, m, (int)n, (int)k, (int)((k + 127) / 128)};
    const int vec = n * (out_dtype == LDOT_F32 ? 4 : 2) % 16 == 0 && (uintptr_t)out % 16 == 0;
    hipStream_t st = (hipStream_t)stream;
    if (out_dtype == LDOT_F32) return gelu ? launch_linear<LDOT_F32, true>(a, vec, st) : launch_linear<LDOT_F32, false>(a, vec, st);
    if (out_dtype == LDOT_BF16) return gelu ? launch_linear<LDOT_BF16, true>(a, vec, st) : launch_linear<LDOT_BF16, false>(a, vec, st);
    return gelu ? launch_linear<LDOT_F16, true>(a, vec, st) : launch_linear<LDOT_F16, false>(a, vec, st);
}
