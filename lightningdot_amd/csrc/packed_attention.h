// Attention over a packed batch: documents of different lengths lie one behind the other in one tensor of tokens, a token sees the
// tokens of its own document.  Per document and head, with X = scale * Q K^T:
//     P = softmax_rows(X),   O = (M o P) V,       M = keep mask / (1 - p) of the dropout, all ones without it
//     dV = (M o P)^T dO,     dP = M o (dO V^T),   delta = rowsum(dO o O),   dX = P o (dP - delta),   dQ = scale dX K,   dK = scale dX^T Q
//
// One family of tiles serves both directions.  A wave keeps 16 * MS rows of the STATIONARY operand in registers (queries forward and for
// dQ, keys for dK / dV) and the workgroup streams 64-row tiles of the other side through LDS.  Scores are computed with the streamed rows
// as the MFMA's A operand: its result leaves every lane with ONE stationary row (lane & 15) and 4 consecutive streamed rows, so that
//   * row statistics of the forward pass are lane-local up to two lane swaps,
//   * two result tiles, rounded, ARE the B operand of the second product (contraction over the streamed rows, whose order may be any as
//     long as both operands agree) — probabilities never pass through LDS; its A operand is the streamed tile, transposed by the LDS read.
// Tiles never span documents: rows of other documents are neither loaded nor multiplied by zero, so an inf or NaN stays in its document.
#pragma once
#include "ldot_common.h"

namespace ldot {

constexpr int kAttnTile = 64;       // rows of a streamed tile, and of an entry of the plan

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// an operand of the attention: element (token, head, e) at token * st + head * sh + e
struct AttnTensor {
    const void* p;
    int64_t st, sh;
};

struct AttnParams {
    AttnTensor q, k, v, o, go;       // go: the output's gradient
    void *out, *dq, *dk, *dv;        // contiguous [total][heads or kv_heads][dim]
    float* lse;                      // [heads][total], base 2: log2 sum exp2(scale2 * q.k)
    float* delta;                    // [heads][total]
    const int4* tiles;               // {first row of the document, rows of the document, tile in it, 1: rows that no document holds}
    int ntiles, heads, kv_heads, dim;
    int64_t total;
    float scale, scale2;             // scale2 = scale * log2(e)
    uint32_t drop;                   // a key is kept iff its 16 random bits are >= drop; 0: no dropout
    float keep_scale;                // 65536 / (65536 - drop)
    const int64_t* seed;
};

template <typename T>
struct AttnType;
template <>
struct AttnType<__bf16> {
    typedef bf16x8_t frag;
    typedef bf16x4_t quad;
};
template <>
struct AttnType<_Float16> {
    typedef f16x8_t frag;
    typedef f16x4_t quad;
};
template <>
struct AttnType<float> {
    typedef f32x8_t frag;
    typedef f32x4 quad;
};

// D[16][16] += A[16][32] B[32][16]; lane l holds 8 of the 32 in each operand (row / column l & 15, group l >> 4): which 8 is free as long
// as A and B agree.  fp32: eight 16x16x4 products, the e-th takes element e of every group.
__device__ __forceinline__ f32x4 attn_mma(bf16x8_t a, bf16x8_t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 attn_mma(f16x8_t a, f16x8_t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 attn_mma(f32x8_t a, f32x8_t b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ bf16x8_t attn_pack(const f32x4& a, const f32x4& b, __bf16) {
    bf16x8_t r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (__bf16)a[e], r[e + 4] = (__bf16)b[e];
    return r;
}
__device__ __forceinline__ f16x8_t attn_pack(const f32x4& a, const f32x4& b, _Float16) {
    f16x8_t r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (_Float16)a[e], r[e + 4] = (_Float16)b[e];
    return r;
}
__device__ __forceinline__ f32x8_t attn_pack(const f32x4& a, const f32x4& b, float) {
    f32x8_t r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = a[e], r[e + 4] = b[e];
    return r;
}

// over the four lanes that share lane & 15
__device__ __forceinline__ float attn_max4(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float attn_sum4(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// the dropout's random bits: a 32-bit mixer (xor-shift, multiply) over (seed, head, row of the packed batch), then over the pair of
// keys; key j of the document takes the lower 16 bits of pair j / 2 if j is even, the upper ones if it is odd
__device__ __forceinline__ uint32_t attn_mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7feb352du;
    x ^= x >> 15;
    x *= 0x846ca68bu;
    return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t attn_head_state(int64_t seed, int head) { return attn_mix((uint32_t)(seed >> 32) ^ ((uint32_t)head * 0x9e3779b9u)); }
__device__ __forceinline__ uint32_t attn_row_state(uint32_t head_state, int64_t seed, int64_t row) {
    return attn_mix(head_state ^ ((uint32_t)row * 0x85ebca6bu + (uint32_t)seed));
}
__device__ __forceinline__ uint32_t attn_pair_bits(uint32_t row_state, uint32_t pair) { return attn_mix(row_state ^ (pair * 0xc2b2ae35u)); }

// blockIdx -> (plan entry, head): heads outermost, and every XCD (blockIdx % 8) takes one contiguous eighth of that order, so that the
// tiles which stream the same document of the same head find it in their own L2
__device__ __forceinline__ void attn_place(unsigned b, unsigned n, int ntiles, int& tile, int& head) {
    const unsigned per = n / 8, more = n % 8, x = b % 8;
    const unsigned at = x * per + min(x, more) + b / 8;
    head = (int)(at / (unsigned)ntiles);
    tile = (int)(at % (unsigned)ntiles);
}

// geometry of a tile in LDS: 64 rows of DP elements, 16 bytes of padding behind each (rows then start 16 bytes apart modulo the banks:
// neither the row-wise 16-byte reads nor the transposing ones conflict)
template <typename T, int NS>
struct AttnGeom {
    static constexpr int DP = NS * 32;                              // head size, padded
    static constexpr int kRow = DP * (int)sizeof(T) + 16;           // bytes
    static constexpr int kTileBytes = kAttnTile * kRow;
    static constexpr int kChunks = DP * (int)sizeof(T) / 16;        // 16-byte chunks of a row
    static constexpr int kPer = kAttnTile * kChunks / 256;          // chunks per thread
    static constexpr int kElems = 16 / (int)sizeof(T);
};

// 64 rows of one operand from memory into registers (rows past the document's end and elements past dim: zeros)
template <typename T, int NS>
struct AttnStage {
    uint4 r[AttnGeom<T, NS>::kPer];
    __device__ __forceinline__ void load(const char* base, int64_t st_bytes, int rows, int dim) {
        typedef AttnGeom<T, NS> G;
#pragma unroll
        for (int i = 0; i < G::kPer; ++i) {
            const int idx = (int)threadIdx.x + 256 * i, row = idx / G::kChunks, c = idx % G::kChunks;
            r[i] = make_uint4(0, 0, 0, 0);
            if (row < rows && c * G::kElems < dim) r[i] = *(const uint4*)(base + row * st_bytes + c * 16);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
        typedef AttnGeom<T, NS> G;
#pragma unroll
        for (int i = 0; i < G::kPer; ++i) {
            const int idx = (int)threadIdx.x + 256 * i, row = idx / G::kChunks, c = idx % G::kChunks;
            *(uint4*)(lds + row * G::kRow + c * 16) = r[i];
        }
    }
};

// A operands out of a tile in LDS
template <typename T, int NS>
struct AttnTile {
    typedef AttnGeom<T, NS> G;
    typedef typename AttnType<T>::frag frag;
    // rows 16 t .. + 15, elements 32 s .. + 31
    static __device__ __forceinline__ frag rows(const char* lds, int t, int s, int lane) {
        const char* p = lds + (16 * t + (lane & 15)) * G::kRow + (s * 32 + (lane >> 4) * 8) * (int)sizeof(T);
        if constexpr (sizeof(T) == 2) {
            return *(const frag*)p;
        } else {
            const f32x4 a = ((const f32x4*)p)[0], b = ((const f32x4*)p)[1];
            return attn_pack(a, b, 0.f);
        }
    }
    // transposed: elements 16 d .. + 15 of rows 32 b .. + 31; a lane's eight rows are the ones whose scores it holds
    static __device__ __forceinline__ frag cols(const char* lds, int b, int d, int lane) {
        const int g = lane >> 4, i = lane & 15;
        if constexpr (sizeof(T) == 2) {
            // a transposing read takes 4 rows x 16 elements per group of 16 lanes: lane i supplies the address of row i / 4, elements
            // 4 (i % 4) .. + 3, and receives element i of the four rows
            const char* p = lds + (32 * b + 4 * g + (i >> 2)) * G::kRow + (16 * d + (i & 3) * 4) * 2;
            typedef __attribute__((address_space(3))) s16x4_t* lptr;
            union {
                s16x4_t h[2];
                frag f;
            } r;
            r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)p);
            r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(p + 16 * G::kRow));
            return r.f;
        } else {
            const char* p = lds + (32 * b + 4 * g) * G::kRow + (16 * d + i) * 4;
            frag r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r[e] = *(const float*)(p + e * G::kRow);
                r[e + 4] = *(const float*)(p + (16 + e) * G::kRow);
            }
            return r;
        }
    }
};

// B operands of a stationary row, from memory (zeros past dim and for a row past the document)
template <typename T, int NS>
__device__ __forceinline__ void attn_load_row(typename AttnType<T>::frag (&f)[NS], const char* row, bool valid, int dim, int lane) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int e = s * 32 + (lane >> 4) * 8;
        if (valid && e < dim)
            f[s] = *(const typename AttnType<T>::frag*)(row + e * (int)sizeof(T));
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) f[s][j] = (T)0.f;
    }
}

// a result tile (element 16 d + 4 g + r of stationary row lane & 15), scaled and rounded once, to memory
template <typename T, int NS>
__device__ __forceinline__ void attn_write_row(const f32x4 (&acc)[2 * NS], float f, T* row, int dim, int lane) {
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d) {
        const int e = 16 * d + 4 * (lane >> 4);
        if (e < dim) {
            typename AttnType<T>::quad o;
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = (T)(acc[d][r] * f);
            *(typename AttnType<T>::quad*)(row + e) = o;
        }
    }
}

// rows that no document holds: zeros
template <typename T>
__device__ __forceinline__ void attn_zero_rows(T* out, int64_t row0, int n, int heads, int head, int dim) {
    for (int i = (int)threadIdx.x; i < n * dim; i += 256) out[((row0 + i / dim) * heads + head) * dim + i % dim] = (T)0.f;
}

template <typename T, int NS, int MQ, bool DROP>
__global__ __launch_bounds__(256) void attn_fwd_kernel(const AttnParams p) {
    typedef AttnGeom<T, NS> G;
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
    __shared__ __attribute__((aligned(16))) char lds[2][2][G::kTileBytes];
    int tile, head;
    attn_place(blockIdx.x, gridDim.x, p.ntiles, tile, head);
    const int4 e = p.tiles[tile];
    const int64_t row0 = (int64_t)e.x + (int64_t)e.z * (kAttnTile * MQ);
    const int nrows = min(kAttnTile * MQ, e.y - e.z * (kAttnTile * MQ));
    if (nrows <= 0) return;                            // (an entry that the plan did not need)
    if (e.w) {
        attn_zero_rows((T*)p.out, row0, nrows, p.heads, head, p.dim);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int kvh = head / (p.heads / p.kv_heads);
    const char* kbase = (const char*)p.k.p + ((int64_t)e.x * p.k.st + kvh * p.k.sh) * (int)sizeof(T);
    const char* vbase = (const char*)p.v.p + ((int64_t)e.x * p.v.st + kvh * p.v.sh) * (int)sizeof(T);
    const int64_t kst = p.k.st * (int)sizeof(T), vst = p.v.st * (int)sizeof(T);
    const int nk = (e.y + kAttnTile - 1) / kAttnTile;

    AttnStage<T, NS> sk, sv;
    sk.load(kbase, kst, e.y, p.dim);
    sv.load(vbase, vst, e.y, p.dim);
    frag q[MQ][NS];
    const int r0 = wave * 16 * MQ + (lane & 15);       // this lane's first row of the tile
    uint32_t state[MQ];
    int64_t seed = 0;
    if (DROP) seed = p.seed[0];
#pragma unroll
    for (int m = 0; m < MQ; ++m) {
        const int r = r0 + 16 * m;
        attn_load_row<T, NS>(q[m], (const char*)p.q.p + ((row0 + r) * p.q.st + head * p.q.sh) * (int)sizeof(T), r < nrows, p.dim, lane);
        if (DROP) state[m] = attn_row_state(attn_head_state(seed, head), seed, row0 + r);
    }
    sk.store(lds[0][0]);
    sv.store(lds[0][1]);
    __syncthreads();

    f32x4 acc[MQ][2 * NS];
    float mx[MQ], sum[MQ];
#pragma unroll
    for (int m = 0; m < MQ; ++m) {
        mx[m] = -INFINITY;
        sum[m] = 0.f;
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) acc[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int kt = 0; kt < nk; ++kt) {
        const int left = e.y - kt * kAttnTile;
        const bool more = kt + 1 < nk;
        if (more) {
            sk.load(kbase + (int64_t)(kt + 1) * kAttnTile * kst, kst, left - kAttnTile, p.dim);
            sv.load(vbase + (int64_t)(kt + 1) * kAttnTile * vst, vst, left - kAttnTile, p.dim);
        }
        const char* kl = lds[kt & 1][0];
        const char* vl = lds[kt & 1][1];
        f32x4 s[MQ][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int m = 0; m < MQ; ++m) s[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                const frag a = Tile::rows(kl, t, st, lane);
#pragma unroll
                for (int m = 0; m < MQ; ++m) s[m][t] = attn_mma(a, q[m][st], s[m][t]);
            }
        }
        if (left < kAttnTile) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * t + 4 * g + r >= left)
#pragma unroll
                        for (int m = 0; m < MQ; ++m) s[m][t][r] = -INFINITY;
        }
        frag b[MQ][2];
#pragma unroll
        for (int m = 0; m < MQ; ++m) {
            float top = s[m][0][0];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, s[m][t][r]);
            const float mnew = fmaxf(mx[m], attn_max4(top) * p.scale2);
            const float ref = mnew == -INFINITY ? 0.f : mnew;      // (every score so far is -inf: their exponentials are 0, not NaN)
            const float fade = __builtin_amdgcn_exp2f(mx[m] - ref);
            float add = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[m][t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m][t][r], p.scale2, -ref));
                    add += s[m][t][r];
                }
            sum[m] = sum[m] * fade + add;
            mx[m] = mnew;
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) acc[m][d] *= fade;
            if (DROP) {
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t bits = attn_pair_bits(state[m], (uint32_t)(kt * 32 + 8 * t + 2 * g + h));
                        if ((bits & 0xffffu) < p.drop) s[m][t][2 * h] = 0.f;
                        if ((bits >> 16) < p.drop) s[m][t][2 * h + 1] = 0.f;
                    }
            }
            // the probabilities are rounded to the operands' type for the second product; their sum is kept in 32 bits unrounded
            b[m][0] = attn_pack(s[m][0], s[m][1], (T)0.f);
            b[m][1] = attn_pack(s[m][2], s[m][3], (T)0.f);
        }
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) {
                const frag a = Tile::cols(vl, blk, d, lane);
#pragma unroll
                for (int m = 0; m < MQ; ++m) acc[m][d] = attn_mma(a, b[m][blk], acc[m][d]);
            }
        if (more) {
            sk.store(lds[(kt + 1) & 1][0]);
            sv.store(lds[(kt + 1) & 1][1]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < MQ; ++m) {
        const float total = attn_sum4(sum[m]);
        const int r = r0 + 16 * m;
        if (r < nrows) {
            const float f = (DROP ? p.keep_scale : 1.f) / total;
            attn_write_row<T, NS>(acc[m], f, (T*)p.out + ((row0 + r) * p.heads + head) * p.dim, p.dim, lane);
            if (p.lse && g == 0) p.lse[head * p.total + row0 + r] = mx[m] + __builtin_amdgcn_logf(total);
        }
    }
}

// KEYS: dK and dV of a tile of keys (the document's queries are streamed, for every query head that shares the key head);
// else: dQ of a tile of queries (its keys are streamed), and delta, which the KEYS launch behind it reads
template <typename T, int NS, int MS, bool DROP, bool KEYS>
__global__ __launch_bounds__(256) void attn_bwd_kernel(const AttnParams p) {
    typedef AttnGeom<T, NS> G;
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
    __shared__ __attribute__((aligned(16))) char lds[2][2][G::kTileBytes];
    __shared__ float row_lse[2][kAttnTile], row_delta[2][kAttnTile];
    __shared__ uint32_t row_state[2][kAttnTile];
    const int heads = KEYS ? p.kv_heads : p.heads;
    int tile, head;
    attn_place(blockIdx.x, gridDim.x, p.ntiles, tile, head);
    const int4 e = p.tiles[tile];
    const int64_t row0 = (int64_t)e.x + (int64_t)e.z * (kAttnTile * MS);
    const int nrows = min(kAttnTile * MS, e.y - e.z * (kAttnTile * MS));
    if (nrows <= 0) return;
    if (e.w) {
        attn_zero_rows((T*)(KEYS ? p.dk : p.dq), row0, nrows, heads, head, p.dim);
        if (KEYS) attn_zero_rows((T*)p.dv, row0, nrows, heads, head, p.dim);
        return;
    }
    constexpr int E = (int)sizeof(T);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int group = p.heads / p.kv_heads;
    const int head_q0 = KEYS ? head * group : head, head_kv = KEYS ? head : head / group;
    const int nt = (e.y + kAttnTile - 1) / kAttnTile;
    const int steps = KEYS ? nt * group : nt;

    // streamed operands: s1 gives the scores, s2 the gradients of the probabilities
    const AttnTensor t1 = KEYS ? p.q : p.k, t2 = KEYS ? p.go : p.v;
    const int64_t st1 = t1.st * E, st2 = t2.st * E;
    AttnStage<T, NS> s1, s2;
    float next_lse = INFINITY, next_delta = 0.f;
    uint32_t next_state = 0;
    int64_t seed = 0;
    if (DROP) seed = p.seed[0];
    auto fetch = [&](int step) {
        const int hq = KEYS ? head_q0 + step / nt : head_kv, at = (KEYS ? step % nt : step) * kAttnTile;
        const int left = e.y - at;
        s1.load((const char*)t1.p + (((int64_t)e.x + at) * t1.st + hq * t1.sh) * E, st1, left, p.dim);
        s2.load((const char*)t2.p + (((int64_t)e.x + at) * t2.st + hq * t2.sh) * E, st2, left, p.dim);
        if (KEYS && threadIdx.x < kAttnTile) {
            const int64_t r = (int64_t)e.x + at + threadIdx.x;
            const bool in = (int)threadIdx.x < left;
            next_lse = in ? p.lse[(int64_t)hq * p.total + r] : INFINITY;      // (probability 0)
            next_delta = in ? p.delta[(int64_t)hq * p.total + r] : 0.f;
            if (DROP) next_state = attn_row_state(attn_head_state(seed, hq), seed, r);
        }
    };
    auto put = [&](int buf) {
        s1.store(lds[buf][0]);
        s2.store(lds[buf][1]);
        if (KEYS && threadIdx.x < kAttnTile) {
            row_lse[buf][threadIdx.x] = next_lse;
            row_delta[buf][threadIdx.x] = next_delta;
            if (DROP) row_state[buf][threadIdx.x] = next_state;
        }
    };
    fetch(0);
    frag b1[MS][NS], b2[MS][NS];
    float my_lse[MS], my_delta[MS];
    uint32_t my_state[MS];
    const int r0 = wave * 16 * MS + (lane & 15);
    const AttnTensor u1 = KEYS ? p.k : p.q, u2 = KEYS ? p.v : p.go;
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int r = r0 + 16 * m;
        const bool in = r < nrows;
        attn_load_row<T, NS>(b1[m], (const char*)u1.p + ((row0 + r) * u1.st + head * u1.sh) * E, in, p.dim, lane);
        attn_load_row<T, NS>(b2[m], (const char*)u2.p + ((row0 + r) * u2.st + head * u2.sh) * E, in, p.dim, lane);
        if (!KEYS) {
            frag o[NS];
            attn_load_row<T, NS>(o, (const char*)p.o.p + ((row0 + r) * p.o.st + head * p.o.sh) * E, in, p.dim, lane);
            float d = 0.f;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) d = __builtin_fmaf((float)o[s][j], (float)b2[m][s][j], d);
            my_delta[m] = attn_sum4(d);
            my_lse[m] = in ? p.lse[(int64_t)head * p.total + row0 + r] : INFINITY;
            if (in && g == 0) p.delta[(int64_t)head * p.total + row0 + r] = my_delta[m];
            if (DROP) my_state[m] = attn_row_state(attn_head_state(seed, head), seed, row0 + r);
        }
    }
    put(0);
    __syncthreads();

    f32x4 acc1[MS][2 * NS], acc2[KEYS ? MS : 1][2 * NS];
#pragma unroll
    for (int m = 0; m < MS; ++m)
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) {
            acc1[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (KEYS) acc2[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    for (int step = 0; step < steps; ++step) {
        const bool more = step + 1 < steps;
        if (more) fetch(step + 1);
        const int buf = step & 1;
        const int at = (KEYS ? step % nt : step) * kAttnTile, left = e.y - at;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            f32x4 s[MS][2], dp[MS][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int m = 0; m < MS; ++m) s[m][t] = dp[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < NS; ++st) {
                    const frag a1 = Tile::rows(lds[buf][0], 2 * blk + t, st, lane), a2 = Tile::rows(lds[buf][1], 2 * blk + t, st, lane);
#pragma unroll
                    for (int m = 0; m < MS; ++m) {
                        s[m][t] = attn_mma(a1, b1[m][st], s[m][t]);
                        dp[m][t] = attn_mma(a2, b2[m][st], dp[m][t]);
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int mr = 16 * (2 * blk + t) + 4 * g;        // this lane's first streamed row of the tile
                f32x4 lse4, delta4;
                uint32_t state4[4];
                if (KEYS) {
                    lse4 = *(const f32x4*)&row_lse[buf][mr];
                    delta4 = *(const f32x4*)&row_delta[buf][mr];
                    if (DROP)
#pragma unroll
                        for (int r = 0; r < 4; ++r) state4[r] = row_state[buf][mr + r];
                }
#pragma unroll
                for (int m = 0; m < MS; ++m) {
                    uint32_t bits[2];
                    if (DROP && !KEYS) {
                        bits[0] = attn_pair_bits(my_state[m], (uint32_t)(at + mr) / 2);
                        bits[1] = attn_pair_bits(my_state[m], (uint32_t)(at + mr) / 2 + 1);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m][t][r], p.scale2, -(KEYS ? lse4[r] : my_lse[m])));
                        if (!KEYS && left < kAttnTile && mr + r >= left) pr = 0.f;
                        float kept = pr, d = dp[m][t][r];
                        if (DROP) {
                            bool keep;
                            if (KEYS) {
                                const uint32_t key = (uint32_t)(e.z * (kAttnTile * MS) + r0 + 16 * m);
                                keep = ((attn_pair_bits(state4[r], key / 2) >> (16 * (key & 1))) & 0xffffu) >= p.drop;
                            } else {
                                keep = ((bits[r >> 1] >> (16 * (r & 1))) & 0xffffu) >= p.drop;
                            }
                            kept = keep ? pr : 0.f;
                            d = keep ? d * p.keep_scale : 0.f;
                        }
                        s[m][t][r] = kept;
                        dp[m][t][r] = pr * (d - (KEYS ? delta4[r] : my_delta[m]));
                    }
                }
            }
            // probabilities and score gradients are rounded to the operands' type for the second products (32-bit sums)
            frag x1[MS], x2[KEYS ? MS : 1];
#pragma unroll
            for (int m = 0; m < MS; ++m) {
                x1[m] = attn_pack(dp[m][0], dp[m][1], (T)0.f);
                if (KEYS) x2[m] = attn_pack(s[m][0], s[m][1], (T)0.f);
            }
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) {
                const frag a1 = Tile::cols(lds[buf][0], blk, d, lane);
#pragma unroll
                for (int m = 0; m < MS; ++m) acc1[m][d] = attn_mma(a1, x1[m], acc1[m][d]);
                if (KEYS) {
                    const frag a2 = Tile::cols(lds[buf][1], blk, d, lane);
#pragma unroll
                    for (int m = 0; m < MS; ++m) acc2[m][d] = attn_mma(a2, x2[m], acc2[m][d]);
                }
            }
        }
        if (more) put(buf ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int r = r0 + 16 * m;
        if (r < nrows) {
            const int64_t o = ((row0 + r) * heads + head) * p.dim;
            attn_write_row<T, NS>(acc1[m], p.scale, (T*)(KEYS ? p.dk : p.dq) + o, p.dim, lane);
            if (KEYS) attn_write_row<T, NS>(acc2[m], DROP ? p.keep_scale : 1.f, (T*)p.dv + o, p.dim, lane);
        }
    }
}

// launches for one element type (one source file each: they compile in parallel); mq: 16-row groups of a wave (the plan's entries are
// 64 * mq rows)
template <typename T>
int attn_launch(const AttnParams& p, bool backward, int mq, hipStream_t st);
extern template int attn_launch<__bf16>(const AttnParams&, bool, int, hipStream_t);
extern template int attn_launch<_Float16>(const AttnParams&, bool, int, hipStream_t);
extern template int attn_launch<float>(const AttnParams&, bool, int, hipStream_t);

template <typename T, int NS, int MQ, bool DROP>
int attn_launch_as(const AttnParams& p, bool backward, hipStream_t st) {
    const unsigned nq = (unsigned)p.ntiles * (unsigned)p.heads, nk = (unsigned)p.ntiles * (unsigned)p.kv_heads;
    if (!backward) {
        hipLaunchKernelGGL((attn_fwd_kernel<T, NS, MQ, DROP>), dim3(nq), dim3(256), 0, st, p);
    } else {
        hipLaunchKernelGGL((attn_bwd_kernel<T, NS, MQ, DROP, false>), dim3(nq), dim3(256), 0, st, p);
        LDOT_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL((attn_bwd_kernel<T, NS, MQ, DROP, true>), dim3(nk), dim3(256), 0, st, p);
    }
    LDOT_HIP_CHECK(hipGetLastError());
    return LDOT_OK;
}

template <typename T, int NS>
int attn_launch_ns(const AttnParams& p, bool backward, int mq, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (mq == 2) return p.drop ? attn_launch_as<T, NS, 2, true>(p, backward, st) : attn_launch_as<T, NS, 2, false>(p, backward, st);
    }
    return p.drop ? attn_launch_as<T, NS, 1, true>(p, backward, st) : attn_launch_as<T, NS, 1, false>(p, backward, st);
}

template <typename T>
int attn_launch(const AttnParams& p, bool backward, int mq, hipStream_t st) {
    switch ((p.dim + 31) / 32) {
        case 1: return attn_launch_ns<T, 1>(p, backward, mq, st);
        case 2: return attn_launch_ns<T, 2>(p, backward, mq, st);
        case 3: return attn_launch_ns<T, 3>(p, backward, mq, st);
        default: return attn_launch_ns<T, 4>(p, backward, mq, st);
    }
}

}  // namespace ldot
