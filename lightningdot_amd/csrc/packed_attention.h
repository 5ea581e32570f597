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
#include <algorithm>
#include <type_traits>

#include "ldot_common.h"

namespace ldot {

constexpr int kAttnTile = 64;       // rows of a streamed tile, and of an entry of the plan
// documents of 65 to 128 rows have kernels of their own where a padded row is up to 128 bytes: two workgroups per CU then hold the four
// operands of 128 rows; with wider rows they are tiles
constexpr bool attn_has_mid(int ns, size_t esize) { return ns * 32 * esize <= 128; }
// 16-row groups of a wave in the backward pass over tiles of 64 * mq rows: two groups halve what is read from LDS for a product (12 heads of
// 64, 8 documents of 4096 rows: 1.67 ms against 1.94), but the accumulators of heads of more than 64 elements then do not fit the registers of
// two waves per SIMD, and one wave per SIMD was slower (16 heads of 128, 5 documents of 1900 to 8192 rows: 5.7 ms against 5.0)
constexpr int attn_bwd_groups(int ns, int mq) { return ns > 2 ? 1 : mq; }

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
    // segment i of the batch: rows [bound[i], bound[i + 1]); the first and the last of the nseg segments hold no document.  Segments of up
    // to 64 rows are found by their number; those of up to 128 are listed as {first row, rows, 0, 1: no document}, longer ones in tiles
    // {first row, rows, tile in it, 1: no document}.  How many there are the device alone knows
    const int* bound;
    const int4 *tiles, *mids;
    const int *ntiles, *nmids;
    int nseg, heads, kv_heads, dim;
    int64_t total;
    float scale, scale2;             // scale2 = scale * log2(e)
    uint32_t drop;                   // a key is kept iff its 16 random bits are >= drop; 0: no dropout
    float keep_scale;                // 65536 / (65536 - drop)
    int shorts;                      // 0: no document of up to 64 rows
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

// t + the sum of what a packed operand holds
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float attn_total(const bf16x8_t& x, float t) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) t = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{x[e], x[e + 1]}, bf16x2_t{(__bf16)1.f, (__bf16)1.f}, t, false);
    return t;
}
__device__ __forceinline__ float attn_total(const f16x8_t& x, float t) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) t = __builtin_amdgcn_fdot2(f16x2_t{x[e], x[e + 1]}, f16x2_t{(_Float16)1.f, (_Float16)1.f}, t, false);
    return t;
}
__device__ __forceinline__ float attn_total(const f32x8_t&, float t) { return t; }      // (nothing was rounded)

// threadIdx.x, made anew: what is computed from it inside a loop over work items is not kept in registers across the loop
__device__ __forceinline__ int attn_thread() {
    int t = (int)threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
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

// fp16 holds no more than 6e-5 to 65504 in full, and probabilities of long documents and gradients of scores are smaller: the second
// products' operands are multiplied by powers of two, and the sums divided by them at the end.  Probabilities (at most 1): by 2^15, which is
// subtracted from the logarithms that they are made with (and so is in the gradients too).  Gradients of scores: by a gain of each owned
// row, large at first; a row's sums so far are scaled down with it whenever a value would pass 2^14, to leave the largest below 2^11, so
// that whatever is normal relative to the row's largest by 2^-24 stays so.  (8192 rows, dO 1e-2 and less: dQ was off by 6e-4, 7e-3, ...)
template <typename T> constexpr float kAttnLift = std::is_same<T, _Float16>::value ? 15.f : 0.f;
template <typename T> constexpr float kAttnUnlift = std::is_same<T, _Float16>::value ? 0x1p-15f : 1.f;     // 2^-lift
template <typename T> constexpr float kAttnGain = std::is_same<T, _Float16>::value ? 0x1p30f : 1.f;
template <typename T, int N>
__device__ __forceinline__ void attn_gain(f32x4& a, f32x4& b, float& gain, float& total, f32x4 (&acc)[N]) {
    if constexpr (std::is_same<T, _Float16>::value) {
        float top = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, fmaxf(fabsf(a[r]), fabsf(b[r])));
        top = attn_max4(top);
        if (top * gain > 0x1p14f) {
            const float next = __builtin_ldexpf(1.f, 11 - __builtin_amdgcn_frexp_expf(top)), by = next / gain;
            if (by < 1.f) {                            // (an infinity's exponent reads as 0)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] *= by;
                total *= by;
                gain = next;
            }
        }
        a *= gain;
        b *= gain;
    }
}

// the dropout's random bits: a 32-bit mixer (xor-shift, multiply; shifts and multipliers from C. Wellons' published search for mixers of
// little bias, 2018) over (seed, head, row of the packed batch), then over the pair of keys, each spread by an odd constant first (2^32 over the
// golden ratio; two multipliers that A. Appleby published for the same purpose); key j of the document takes the lower 16 bits of pair j / 2 if j
// is even, the upper ones if it is odd
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

// Work item b -> (tile, head).  The tiles are listed from the longest document to the shortest and taken in that order (the last ones to
// finish are short), yet those of one document and head belong on one XCD (blockIdx % 8), whose L2 then holds what they stream.  A head's
// tiles are dealt to 8 hands, tile t to hand t % 8; the 8 * heads hands go to the XCDs in equal runs, and an XCD takes one tile of each of
// its hands in turn.
__device__ __forceinline__ unsigned attn_items(int ntiles, int heads) { return 8u * (unsigned)heads * (unsigned)((ntiles + 7) / 8); }
__device__ __forceinline__ bool attn_place(unsigned b, int ntiles, int heads, int& tile, int& head) {
    const unsigned i = b / 8, hand = (b % 8) * (unsigned)heads + i % (unsigned)heads;
    head = (int)(hand >> 3);
    tile = (int)((hand & 7) + 8 * (i / (unsigned)heads));
    return tile < ntiles;
}

// geometry of a tile in LDS: 64 rows of DP elements, a power of two of bytes each; the 16-byte chunk c of a row lies at place c ^ swizzle(row).
// LDS serves 16 lanes at once in a 16-byte read, 8 rows of two neighbouring chunks: the permutations below put them on 16 different places
// of 256 bytes, and likewise the 8 rows of 32 bytes that a transposing read touches (0 conflicts; rows padded by 16 bytes took 1.7 times the
// cycles).
template <typename T, int NS>
struct AttnGeom {
    static constexpr int DP = NS * 32;                              // head size, padded
    static constexpr int kBytes = DP * (int)sizeof(T);              // of a row's elements
    static constexpr int kRow = kBytes <= 64 ? 64 : kBytes <= 128 ? 128 : kBytes <= 256 ? 256 : 512;
    static constexpr int kTileBytes = kAttnTile * kRow;
    static constexpr int kChunks = kBytes / 16;                     // 16-byte chunks of a row
    static constexpr int kPer = kAttnTile * kChunks / 256;          // chunks per thread
    static constexpr int kElems = 16 / (int)sizeof(T);
    static __device__ __forceinline__ int swizzle(int row) {        // (row & 15 alone decides)
        return kRow == 64 ? (row >> 1) & 3 : kRow == 128 ? row & 6 : (2 * (row & 7)) ^ (4 * ((row >> 3) & 1));
    }
    static __device__ __forceinline__ int at(int row, int c) { return row * kRow + ((c ^ swizzle(row)) << 4); }
};

// 64 rows of one operand from memory into registers, by 256 threads (or 128 by 512; rows past the document's end and elements past dim:
// zeros)
template <typename T, int NS, int THREADS = 256>
struct AttnStage {
    uint4 r[AttnGeom<T, NS>::kPer];
    __device__ __forceinline__ void load(const char* base, int64_t st_bytes, int rows, int dim, int thread) {
        typedef AttnGeom<T, NS> G;
#pragma unroll
        for (int i = 0; i < G::kPer; ++i) {
            const int idx = thread + THREADS * i, row = idx / G::kChunks, c = idx % G::kChunks;
            r[i] = make_uint4(0, 0, 0, 0);
            if (row < rows && c * G::kElems < dim) r[i] = *(const uint4*)(base + row * st_bytes + c * 16);
        }
    }
    __device__ __forceinline__ void store(char* lds, int thread) const {
        typedef AttnGeom<T, NS> G;
#pragma unroll
        for (int i = 0; i < G::kPer; ++i) {
            const int idx = thread + THREADS * i, row = idx / G::kChunks, c = idx % G::kChunks;
            *(uint4*)(lds + G::at(row, c)) = r[i];
        }
    }
};

// elements of a row that a lane of group g holds of step s (32 elements): 16-bit types 8 g .. + 7, fp32 4 g .. + 3 and 16 + 4 g .. + 3 (two
// chunks of 16 bytes each); the same for both operands of a product
// A operands out of a tile in LDS
template <typename T, int NS>
struct AttnTile {
    typedef AttnGeom<T, NS> G;
    typedef typename AttnType<T>::frag frag;
    // rows 16 t .. + 15, elements 32 s .. + 31
    static __device__ __forceinline__ frag rows(const char* lds, int t, int s, int lane) {
        const char* p = lds + (16 * t + (lane & 15)) * G::kRow;
        const int c = (lane >> 4) ^ G::swizzle(lane & 15);
        if constexpr (sizeof(T) == 2) {
            return *(const frag*)(p + ((c ^ (4 * s)) << 4));
        } else {
            return attn_pack(*(const f32x4*)(p + ((c ^ (8 * s)) << 4)), *(const f32x4*)(p + ((c ^ (8 * s + 4)) << 4)), 0.f);
        }
    }
    // transposed: elements 16 d .. + 15 of rows 32 b .. + 31; a lane's eight rows are the ones whose scores it holds
    static __device__ __forceinline__ frag cols(const char* lds, int b, int d, int lane) {
        const int g = lane >> 4, i = lane & 15;
        if constexpr (sizeof(T) == 2) {
            // a transposing read takes 4 rows x 16 elements per group of 16 lanes: lane i supplies the address of row i / 4, elements
            // 4 (i % 4) .. + 3, and receives element i of the four rows
            const int row = 4 * g + (i >> 2), c = ((i >> 1) & 1) ^ G::swizzle(row);
            const char* p = lds + (32 * b + row) * G::kRow + ((c ^ (2 * d)) << 4) + (i & 1) * 8;
            typedef __attribute__((address_space(3))) s16x4_t* lptr;
            union {
                s16x4_t h[2];
                frag f;
            } r;
            r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)p);
            r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lptr)(p + 16 * G::kRow));
            return r.f;
        } else {
            frag r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 4 * g + e;
                const char* p = lds + (32 * b + row) * G::kRow + ((((i >> 2) ^ G::swizzle(row)) ^ (4 * d)) << 4) + (i & 3) * 4;
                r[e] = *(const float*)p;
                r[e + 4] = *(const float*)(p + 16 * G::kRow);
            }
            return r;
        }
    }
};

// B operands of a stationary row, from memory (zeros past dim and for a row past the document)
template <typename T, int NS>
__device__ __forceinline__ void attn_load_row(typename AttnType<T>::frag (&f)[NS], const char* row, bool valid, int dim, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        if constexpr (sizeof(T) == 2) {
            const int e = s * 32 + g * 8;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (valid && e < dim) v = *(const uint4*)(row + e * 2);
            union {
                uint4 u;
                typename AttnType<T>::frag f;
            } x;
            x.u = v;
            f[s] = x.f;
        } else {
            const int e = s * 32 + g * 4;
            f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = {0.f, 0.f, 0.f, 0.f};
            if (valid && e < dim) a = *(const f32x4*)(row + e * 4);
            if (valid && e + 16 < dim) b = *(const f32x4*)(row + (e + 16) * 4);
            f[s] = attn_pack(a, b, 0.f);
        }
    }
}

// result rows of a wave (element 16 d + 4 g + r of row lane & 15), scaled and rounded once, to memory: turned through 16 rows of LDS of the
// wave's own, so that whole rows leave in 16-byte stores (32 bytes of 16 rows each, as they lie in registers, keep memory busy four times)
template <typename T, int NS>
__device__ __forceinline__ void attn_write_rows(char* scratch, const f32x4 (&acc)[2 * NS], float f, T* out, int64_t row_elems, int rows, int dim, int lane) {
    typedef AttnGeom<T, NS> G;
    if constexpr (sizeof(T) == 4) {                    // (a lane's four elements are 16 bytes as they are)
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) {
            const int e = 16 * d + 4 * (lane >> 4);
            if ((lane & 15) < rows && e < dim) *(f32x4*)(out + (lane & 15) * row_elems + e) = acc[d] * f;
        }
        return;
    }
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d) {
        typename AttnType<T>::quad o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = (T)(acc[d][r] * f);
        *(typename AttnType<T>::quad*)(scratch + G::at(lane & 15, 2 * d + (lane >> 5)) + ((lane >> 4) & 1) * 8) = o;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 16 * G::kChunks / 64; ++i) {
        const int idx = lane + 64 * i, row = idx / G::kChunks, c = idx % G::kChunks;
        if (row < rows && c * G::kElems < dim) *(uint4*)(out + row * row_elems + c * G::kElems) = *(const uint4*)(scratch + G::at(row, c));
    }
    __builtin_amdgcn_wave_barrier();
}

// rows that no document holds: zeros (n rows of one head, by `threads` threads)
template <typename T>
__device__ __forceinline__ void attn_zero_rows(T* out, int64_t row0, int n, int heads, int head, int dim, int thread, int threads) {
    for (int i = thread; i < n * dim; i += threads) out[((row0 + i / dim) * heads + head) * dim + i % dim] = (T)0.f;
}

// probabilities that the dropout takes out become zeros: four scores of one row, keys from `key` (a multiple of 4) on
__device__ __forceinline__ void attn_drop4(f32x4& p, uint32_t state, uint32_t key, uint32_t drop) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t bits = attn_pair_bits(state, key / 2 + h);
        if ((bits & 0xffffu) < drop) p[2 * h] = 0.f;
        if ((bits >> 16) < drop) p[2 * h + 1] = 0.f;
    }
}

// which of one key's probabilities stay in four rows, whose states lie one behind the other.  A lane and its neighbour hold the two keys of
// a pair: each makes the bits of two rows and hands the other its half (backward of 12 heads of 384 documents of 11 to 101 rows: 95 -> 93 us)
__device__ __forceinline__ void attn_keep4(const uint32_t* states, uint32_t key, uint32_t drop, bool (&keep)[4]) {
    const bool odd = key & 1;
    const uint2 own = *(const uint2*)(states + (odd ? 2 : 0));
    const uint32_t a = attn_pair_bits(own.x, key / 2), b = attn_pair_bits(own.y, key / 2);
    const uint32_t c = __builtin_amdgcn_mov_dpp((int)a, 0xb1, 0xf, 0xf, true), d = __builtin_amdgcn_mov_dpp((int)b, 0xb1, 0xf, 0xf, true);     // (lane ^ 1)
    const uint32_t bits[4] = {odd ? c : a, odd ? d : b, odd ? a : c, odd ? b : d};
#pragma unroll
    for (int r = 0; r < 4; ++r) keep[r] = ((bits[r] >> (odd ? 16 : 0)) & 0xffffu) >= drop;
}

// ---- forward ------------------------------------------------------------------------------------------------------------------------------
// Documents of up to 64 rows: a wave takes one document of one head, all of its keys at once (no running maximum), and nothing is shared, so
// nothing waits for another wave.  Bound by memory: every operand is read once, four heads of a document by one workgroup (bf16, 2048 documents
// of 6 to 62 rows, 12 heads of 64: 83 us, 5.2 TB/s, a large copy's rate).
template <typename T, int NS, bool DROP>
__device__ __forceinline__ void attn_fwd_short(const AttnParams& p, char* lds, unsigned item, int lane) {
    typedef AttnGeom<T, NS> G;
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
    constexpr int E = (int)sizeof(T);
    const unsigned seg = item / (unsigned)p.heads;
    if (seg >= (unsigned)p.nseg) return;
    const int head = (int)(item % (unsigned)p.heads), kvh = head / (p.heads / p.kv_heads), g = lane >> 4;
    const int start = p.bound[seg], len = p.bound[seg + 1] - start;
    if (len <= 0 || len > kAttnTile) return;
    if (seg == 0 || seg == (unsigned)p.nseg - 1) {
        attn_zero_rows((T*)p.out, start, len, p.heads, head, p.dim, lane, 64);
        return;
    }
    char* const scratch = lds + G::kTileBytes;
    const char* kbase = (const char*)p.k.p + ((int64_t)start * p.k.st + kvh * p.k.sh) * E;
    const char* vbase = (const char*)p.v.p + ((int64_t)start * p.v.st + kvh * p.v.sh) * E;
    const char* qbase = (const char*)p.q.p + ((int64_t)start * p.q.st + head * p.q.sh) * E;
    frag k[4][NS], q[NS];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int r = 16 * t + (lane & 15);
        attn_load_row<T, NS>(k[t], kbase + r * p.k.st * E, r < len, p.dim, lane);
    }
    attn_load_row<T, NS>(q, qbase + (lane & 15) * p.q.st * E, (lane & 15) < len, p.dim, lane);
    {
        uint4 v[kAttnTile * G::kChunks / 64];
#pragma unroll
        for (int i = 0; i < kAttnTile * G::kChunks / 64; ++i) {
            const int idx = lane + 64 * i, row = idx / G::kChunks, c = idx % G::kChunks;
            v[i] = make_uint4(0, 0, 0, 0);
            if (row < len && c * G::kElems < p.dim) v[i] = *(const uint4*)(vbase + row * p.v.st * E + c * 16);
        }
#pragma unroll
        for (int i = 0; i < kAttnTile * G::kChunks / 64; ++i) {
            const int idx = lane + 64 * i, row = idx / G::kChunks, c = idx % G::kChunks;
            *(uint4*)(lds + G::at(row, c)) = v[i];
        }
    }
    __builtin_amdgcn_wave_barrier();
    int64_t seed = 0;
    if (DROP) seed = p.seed[0];
    for (int q0 = 0; q0 < len; q0 += 16) {
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (16 * t < len)
#pragma unroll
                for (int st = 0; st < NS; ++st) s[t] = attn_mma(k[t][st], q[st], s[t]);
        }
        const int row = q0 + (lane & 15);
        attn_load_row<T, NS>(q, qbase + (row + 16) * p.q.st * E, row + 16 < len, p.dim, lane);         // (the next 16 rows')
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (16 * t + 4 * g + r >= len) s[t][r] = -INFINITY;
                top = fmaxf(top, s[t][r]);
            }
        const float mx = attn_max4(top) * p.scale2;
        const float ref = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], p.scale2, -ref));
                sum += s[t][r];
            }
        sum = attn_sum4(sum);
        if (DROP) {
            const uint32_t state = attn_row_state(attn_head_state(seed, head), seed, (int64_t)start + row);
#pragma unroll
            for (int t = 0; t < 4; ++t) attn_drop4(s[t], state, (uint32_t)(16 * t + 4 * g), p.drop);
        }
        f32x4 acc[2 * NS];
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            if (32 * blk >= len) continue;
            const frag b = attn_pack(s[2 * blk], s[2 * blk + 1], (T)0.f);
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) acc[d] = attn_mma(Tile::cols(lds, blk, d, lane), b, acc[d]);
        }
        const int64_t at = (int64_t)start + q0;
        attn_write_rows<T, NS>(scratch, acc, (DROP ? p.keep_scale : 1.f) / sum, (T*)p.out + (at * p.heads + head) * p.dim, (int64_t)p.heads * p.dim,
                               len - q0, p.dim, lane);
        if (p.lse && g == 0 && row < len) p.lse[(int64_t)head * p.total + start + row] = mx + __builtin_amdgcn_logf(sum);
    }
}

// Documents of 65 to 128 rows: eight waves share one document of one head, 16 rows of queries each, all keys at once.  Bound by latency: two
// workgroups per CU, one computes while the other loads (161 documents of 65 to 101 rows, 12 heads of 64, dropout: 24 us, 3.3 TB/s).
template <typename T, int NS, bool DROP>
__device__ __forceinline__ void attn_fwd_mid(const AttnParams& p, char* lds, const int4 e, int head) {
    typedef AttnGeom<T, NS> G;
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
    constexpr int E = (int)sizeof(T);
    const int start = e.x, len = e.y;
    if (e.w) {
        attn_zero_rows((T*)p.out, start, len, p.heads, head, p.dim, (int)threadIdx.x, 512);
        return;
    }
    const int tid = attn_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, kvh = head / (p.heads / p.kv_heads);
    char *const lk = lds, *const lv = lds + 2 * G::kTileBytes;
    AttnStage<T, NS, 512> a, b;
    a.load((const char*)p.k.p + ((int64_t)start * p.k.st + kvh * p.k.sh) * E, p.k.st * E, len, p.dim, tid);
    b.load((const char*)p.v.p + ((int64_t)start * p.v.st + kvh * p.v.sh) * E, p.v.st * E, len, p.dim, tid);
    const int row = 16 * wave + (lane & 15);
    const bool mine = 16 * wave < len;
    frag q[NS];
    attn_load_row<T, NS>(q, (const char*)p.q.p + (((int64_t)start + row) * p.q.st + head * p.q.sh) * E, row < len, p.dim, lane);
    a.store(lk, tid);
    b.store(lv, tid);
    __syncthreads();
    f32x4 s[8], acc[2 * NS];
    float top = -INFINITY, sum = 0.f;
    if (mine) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (16 * t < len)
#pragma unroll
                for (int st = 0; st < NS; ++st) s[t] = attn_mma(Tile::rows(lk, t, st, lane), q[st], s[t]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (16 * t + 4 * g + r >= len) s[t][r] = -INFINITY;
                top = fmaxf(top, s[t][r]);
            }
        }
        top = attn_max4(top) * p.scale2;
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], p.scale2, -ref));
                sum += s[t][r];
            }
        sum = attn_sum4(sum);
        if (DROP) {
            const int64_t seed = p.seed[0];
            const uint32_t state = attn_row_state(attn_head_state(seed, head), seed, (int64_t)start + row);
#pragma unroll
            for (int t = 0; t < 8; ++t) attn_drop4(s[t], state, (uint32_t)(16 * t + 4 * g), p.drop);
        }
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) {
            if (32 * blk >= len) continue;
            const frag x = attn_pack(s[2 * blk], s[2 * blk + 1], (T)0.f);
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) acc[d] = attn_mma(Tile::cols(lv, blk, d, lane), x, acc[d]);
        }
    }
    __syncthreads();                                   // (the rows leave through the keys' place)
    if (mine) {
        attn_write_rows<T, NS>(lk + wave * 16 * G::kRow, acc, (DROP ? p.keep_scale : 1.f) / sum,
                               (T*)p.out + (((int64_t)start + 16 * wave) * p.heads + head) * p.dim, (int64_t)p.heads * p.dim, len - 16 * wave, p.dim, lane);
        if (p.lse && g == 0 && row < len) p.lse[(int64_t)head * p.total + start + row] = top + __builtin_amdgcn_logf(sum);
    }
}

// Longer ones: 64 * MQ rows of queries per workgroup, keys streamed.  Bound by the matrix pipe and, as much, by the exponentials beside it
// (bf16, 16 heads of 128, 4 key heads, 5 documents of 1900 to 8192 rows: 0.84 ms, 860 TFLOP/s; 12 heads of 64, 8 documents of 4096: 0.58 ms,
// 710 TFLOP/s).
template <typename T, int NS, int MQ, bool DROP>
__device__ __forceinline__ void attn_fwd_tile(const AttnParams& p, char* lds, const int4 e, int head) {
    typedef AttnGeom<T, NS> G;
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
    const int64_t row0 = (int64_t)e.x + (int64_t)e.z * (kAttnTile * MQ);
    const int nrows = min(kAttnTile * MQ, e.y - e.z * (kAttnTile * MQ));
    if (nrows <= 0) return;
    if (e.w) {
        attn_zero_rows((T*)p.out, row0, nrows, p.heads, head, p.dim, (int)threadIdx.x, 256);
        return;
    }
    const int tid = attn_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const int kvh = head / (p.heads / p.kv_heads);
    const char* kbase = (const char*)p.k.p + ((int64_t)e.x * p.k.st + kvh * p.k.sh) * (int)sizeof(T);
    const char* vbase = (const char*)p.v.p + ((int64_t)e.x * p.v.st + kvh * p.v.sh) * (int)sizeof(T);
    const int64_t kst = p.k.st * (int)sizeof(T), vst = p.v.st * (int)sizeof(T);
    const int nk = (e.y - 1) / kAttnTile + 1;
    auto kl = [&](int i) { return lds + (i & 1) * 2 * G::kTileBytes; };

    AttnStage<T, NS> sk, sv;
    sk.load(kbase, kst, e.y, p.dim, tid);
    sv.load(vbase, vst, e.y, p.dim, tid);
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
    sk.store(kl(0), tid);
    sv.store(kl(0) + G::kTileBytes, tid);
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
            sk.load(kbase + (int64_t)(kt + 1) * kAttnTile * kst, kst, left - kAttnTile, p.dim, tid);
            sv.load(vbase + (int64_t)(kt + 1) * kAttnTile * vst, vst, left - kAttnTile, p.dim, tid);
        }
        const char* kl0 = kl(kt);
        const char* vl0 = kl0 + G::kTileBytes;
        f32x4 s[MQ][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int m = 0; m < MQ; ++m) s[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                const frag a = Tile::rows(kl0, t, st, lane);
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
        // The maximum that is taken out of the exponent is not the running one: it stays until a score passes it by 2^8 (a factor that
        // neither fp32 sums nor the rounding of the probabilities notice), so that the accumulators are hardly ever rescaled
        float top[MQ];
        bool grow = false;
#pragma unroll
        for (int m = 0; m < MQ; ++m) {
            top[m] = fmaxf(s[m][0][0], s[m][0][1]);
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; r += 2) top[m] = fmaxf(fmaxf(top[m], s[m][t][r]), s[m][t][r + 1]);
            top[m] = attn_max4(top[m]) * p.scale2;
            grow |= top[m] > mx[m] + 8.f;
        }
        if (__any(grow)) {
#pragma unroll
            for (int m = 0; m < MQ; ++m) {
                const float mnew = fmaxf(mx[m], top[m]);
                const float fade = mnew == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx[m] - mnew);
                sum[m] *= fade;
                mx[m] = mnew;
#pragma unroll
                for (int d = 0; d < 2 * NS; ++d) acc[m][d] *= fade;
            }
        }
        frag b[MQ][2];
#pragma unroll
        for (int m = 0; m < MQ; ++m) {
            const float ref = mx[m] == -INFINITY ? 0.f : mx[m];    // (every score so far is -inf: their exponentials are 0, not NaN)
            float add[2] = {0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[m][t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m][t][r], p.scale2, -ref));
                    add[r & 1] += s[m][t][r];
                }
            sum[m] += add[0] + add[1];
            if (DROP)
#pragma unroll
                for (int t = 0; t < 4; ++t) attn_drop4(s[m][t], state[m], (uint32_t)(kt * kAttnTile + 16 * t + 4 * g), p.drop);
            // the probabilities are rounded to the operands' type for the second product; their sum is kept in 32 bits unrounded
            b[m][0] = attn_pack(s[m][0], s[m][1], (T)0.f);
            b[m][1] = attn_pack(s[m][2], s[m][3], (T)0.f);
        }
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) {
                const frag a = Tile::cols(vl0, blk, d, lane);
#pragma unroll
                for (int m = 0; m < MQ; ++m) acc[m][d] = attn_mma(a, b[m][blk], acc[m][d]);
            }
        if (more) {
            sk.store(kl(kt + 1), tid);
            sv.store(kl(kt + 1) + G::kTileBytes, tid);
        }
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < MQ; ++m) {
        const float total = attn_sum4(sum[m]);
        const int r = r0 + 16 * m;
        attn_write_rows<T, NS>(lds + wave * 16 * G::kRow, acc[m], (DROP ? p.keep_scale : 1.f) / total,
                               (T*)p.out + ((row0 + r - (lane & 15)) * p.heads + head) * p.dim, (int64_t)p.heads * p.dim, nrows - (r - (lane & 15)), p.dim, lane);
        if (p.lse && g == 0 && r < nrows) p.lse[(int64_t)head * p.total + row0 + r] = mx[m] + __builtin_amdgcn_logf(total);
    }
}

template <typename T, int NS, bool DROP>
__global__ __launch_bounds__(256) void attn_fwd_short_kernel(const AttnParams p) {
    constexpr int kBytes = (kAttnTile + (sizeof(T) == 2 ? 16 : 0)) * AttnGeom<T, NS>::kRow;
    __shared__ __attribute__((aligned(16))) char lds[4 * kBytes];
    const unsigned wave = threadIdx.x >> 6;
    attn_fwd_short<T, NS, DROP>(p, lds + wave * kBytes, (blockIdx.y * gridDim.x + blockIdx.x) * 4 + wave, (int)threadIdx.x & 63);
}

template <typename T, int NS, bool DROP>
__global__ __launch_bounds__(512, 4) void attn_fwd_mid_kernel(const AttnParams p) {
    __shared__ __attribute__((aligned(16))) char lds[4 * AttnGeom<T, NS>::kTileBytes];
    const int nm = p.nmids[0];
    const unsigned n = (unsigned)nm * (unsigned)p.heads;
    for (unsigned i = blockIdx.x; i < n; i += gridDim.x) {       // (heads innermost: they share a document's rows of memory)
        attn_fwd_mid<T, NS, DROP>(p, lds, p.mids[i / (unsigned)p.heads], (int)(i % (unsigned)p.heads));
        __syncthreads();
    }
}

template <typename T, int NS, int MQ, bool DROP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_fwd_kernel(const AttnParams p) {
    __shared__ __attribute__((aligned(16))) char lds[4 * AttnGeom<T, NS>::kTileBytes];
    const int nt = p.ntiles[0];
    const unsigned n = attn_items(nt, p.heads);
    for (unsigned i = blockIdx.x; i < n; i += gridDim.x) {
        int tile, head;
        if (!attn_place(i, nt, p.heads, tile, head)) continue;
        attn_fwd_tile<T, NS, MQ, DROP>(p, lds, p.tiles[tile], head);
        __syncthreads();
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------------
// With dropout, dX = 1 / (1 - p) P (kept dP - (1 - p) delta): the kernels hold delta times 1 - p, and the factor waits for the sums
template <bool DROP>
__device__ __forceinline__ float attn_grad_scale(const AttnParams& p) { return DROP ? p.scale * p.keep_scale : p.scale; }

// S and dP of 32 streamed rows (blk of a tile) against a wave's stationary rows
template <typename T, int NS, int MS>
__device__ __forceinline__ void attn_bwd_scores(const char* l1, const char* l2, int blk, const typename AttnType<T>::frag (&b1)[MS][NS],
                                                const typename AttnType<T>::frag (&b2)[MS][NS], f32x4 (&s)[MS][2], f32x4 (&dp)[MS][2], int lane) {
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int m = 0; m < MS; ++m) s[m][t] = dp[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        // (all reads of 16 rows go out before the first product: one read's latency for 2 NS products instead of one for two)
        frag a1[NS], a2[NS];
#pragma unroll
        for (int st = 0; st < NS; ++st) a1[st] = Tile::rows(l1, 2 * blk + t, st, lane), a2[st] = Tile::rows(l2, 2 * blk + t, st, lane);
        if (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int m = 0; m < MS; ++m) {
                s[m][t] = attn_mma(a1[st], b1[m][st], s[m][t]);
                dp[m][t] = attn_mma(a2[st], b2[m][st], dp[m][t]);
            }
    }
}

// Documents of up to 64 rows: a workgroup takes one document of one key head, Q, K, V and dO are read once and dQ, dK and dV leave from one
// launch.  First with queries stationary: a row's scores are all there, its statistics and delta need neither the forward pass's output nor
// its logarithm; then with keys.  Three workgroups per CU take turns at loading and computing (223 documents of 11 to 64 rows, 12 heads of 64,
// dropout: 30 us, 3.1 TB/s).
template <typename T, int NS, bool DROP>
__device__ __forceinline__ void attn_bwd_short(const AttnParams& p, char* lds, float* row_lse, float* row_delta, uint32_t* row_state, unsigned item) {
    typedef AttnGeom<T, NS> G;
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
    constexpr int E = (int)sizeof(T);
    const int seg = (int)(item / (unsigned)p.kv_heads), kvh = (int)(item % (unsigned)p.kv_heads), group = p.heads / p.kv_heads;
    if (seg >= p.nseg) return;
    const int start = p.bound[seg], len = p.bound[seg + 1] - start;
    if (len <= 0 || len > kAttnTile) return;
    if (seg == 0 || seg == p.nseg - 1) {
        for (int h = 0; h < group; ++h) attn_zero_rows((T*)p.dq, start, len, p.heads, kvh * group + h, p.dim, (int)threadIdx.x, 256);
        attn_zero_rows((T*)p.dk, start, len, p.kv_heads, kvh, p.dim, (int)threadIdx.x, 256);
        attn_zero_rows((T*)p.dv, start, len, p.kv_heads, kvh, p.dim, (int)threadIdx.x, 256);
        return;
    }
    const int tid = attn_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    char *const lk = lds, *const lv = lds + G::kTileBytes, *const lq = lds + 2 * G::kTileBytes, *const lg = lds + 3 * G::kTileBytes;
    const bool mine = 16 * wave < len;                 // this wave's 16 rows hold any
    const int row = 16 * wave + (lane & 15);
    const int64_t ost_q = (int64_t)p.heads * p.dim, ost_k = (int64_t)p.kv_heads * p.dim;
    int64_t seed = 0;
    if (DROP) seed = p.seed[0];
    AttnStage<T, NS> a, b, c, d;
    auto fetch = [&](int head) {
        a.load((const char*)p.q.p + ((int64_t)start * p.q.st + head * p.q.sh) * E, p.q.st * E, len, p.dim, tid);
        b.load((const char*)p.go.p + ((int64_t)start * p.go.st + head * p.go.sh) * E, p.go.st * E, len, p.dim, tid);
    };
    c.load((const char*)p.k.p + ((int64_t)start * p.k.st + kvh * p.k.sh) * E, p.k.st * E, len, p.dim, tid);
    d.load((const char*)p.v.p + ((int64_t)start * p.v.st + kvh * p.v.sh) * E, p.v.st * E, len, p.dim, tid);
    fetch(kvh * group);
    f32x4 dk[1][2 * NS], dv[1][2 * NS];
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d) dk[0][d] = dv[0][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float gain_k = kAttnGain<T>, unused_k = 0.f;
    c.store(lk, tid);
    d.store(lv, tid);
    for (int h = 0; h < group; ++h) {
        const int head = kvh * group + h;
        if (h) {
            fetch(head);
            __syncthreads();                           // (the head before is done with the tiles)
        }
        a.store(lq, tid);
        b.store(lg, tid);
        const uint32_t head_state = DROP ? attn_head_state(seed, head) : 0u;
        if (DROP && threadIdx.x < kAttnTile) row_state[threadIdx.x] = attn_row_state(head_state, seed, (int64_t)start + threadIdx.x);
        __syncthreads();
        frag b1[1][NS], b2[1][NS];
        if (mine) {
#pragma unroll
            for (int s = 0; s < NS; ++s) b1[0][s] = Tile::rows(lq, wave, s, lane), b2[0][s] = Tile::rows(lg, wave, s, lane);
            f32x4 s[2][1][2], dp[2][1][2];
            float top = -INFINITY;
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                if (32 * blk < len) attn_bwd_scores<T, NS, 1>(lk, lv, blk, b1, b2, s[blk], dp[blk], lane);
                else
#pragma unroll
                    for (int t = 0; t < 2; ++t) s[blk][0][t] = dp[blk][0][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (32 * blk + 16 * t + 4 * g + r >= len) s[blk][0][t][r] = -INFINITY;
                        top = fmaxf(top, s[blk][0][t][r]);
                    }
            }
            const float mx = attn_max4(top) * p.scale2, ref = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f;
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[blk][0][t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[blk][0][t][r], p.scale2, -ref));
                        sum += s[blk][0][t][r];
                    }
            sum = attn_sum4(sum);
            const float inv = 1.f / sum;
            float gain = kAttnGain<T>, unused = 0.f;
            const uint32_t state = DROP ? row_state[row] : 0u;
            float delta = 0.f;
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (DROP) attn_drop4(dp[blk][0][t], state, (uint32_t)(32 * blk + 16 * t + 4 * g), p.drop);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[blk][0][t][r] *= inv;
                        delta = __builtin_fmaf(s[blk][0][t][r], dp[blk][0][t][r], delta);
                    }
                }
            delta = attn_sum4(delta);
            if (g == 0) {
                row_lse[row] = row < len ? mx + __builtin_amdgcn_logf(sum) - kAttnLift<T> : INFINITY;
                row_delta[row] = row < len ? delta : 0.f;
            }
            f32x4 dq[2 * NS];
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) dq[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                if (32 * blk >= len) continue;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) dp[blk][0][t][r] = s[blk][0][t][r] * (dp[blk][0][t][r] - delta);
                attn_gain<T>(dp[blk][0][0], dp[blk][0][1], gain, unused, dq);
                const frag x = attn_pack(dp[blk][0][0], dp[blk][0][1], (T)0.f);
#pragma unroll
                for (int d = 0; d < 2 * NS; ++d) dq[d] = attn_mma(Tile::cols(lk, blk, d, lane), x, dq[d]);
            }
            attn_write_rows<T, NS>(lds + 4 * G::kTileBytes + wave * 16 * G::kRow, dq, attn_grad_scale<DROP>(p) / gain,
                                   (T*)p.dq + ((int64_t)start + 16 * wave) * ost_q + head * p.dim,
                                   ost_q, len - 16 * wave, p.dim, lane);
        } else if (g == 0) {
            row_lse[row] = INFINITY;                   // (probability 0)
            row_delta[row] = 0.f;
        }
        __syncthreads();
        if (mine) {
#pragma unroll
            for (int s = 0; s < NS; ++s) b1[0][s] = Tile::rows(lk, wave, s, lane), b2[0][s] = Tile::rows(lv, wave, s, lane);
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
                if (32 * blk >= len) continue;
                f32x4 s[1][2], dp[1][2];
                attn_bwd_scores<T, NS, 1>(lq, lg, blk, b1, b2, s, dp, lane);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int mr = 32 * blk + 16 * t + 4 * g;
                    const f32x4 lse4 = *(const f32x4*)&row_lse[mr], delta4 = *(const f32x4*)&row_delta[mr];
                    bool keep[4];
                    if (DROP) attn_keep4(row_state + mr, (uint32_t)row, p.drop, keep);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][t][r], p.scale2, -lse4[r]));
                        float kept = pr, d = dp[0][t][r];
                        if (DROP) {
                            kept = keep[r] ? pr : 0.f;
                            d = keep[r] ? d : 0.f;
                        }
                        s[0][t][r] = kept;
                        dp[0][t][r] = pr * (d - delta4[r]);
                    }
                }
                attn_gain<T>(dp[0][0], dp[0][1], gain_k, unused_k, dk[0]);
                const frag x1 = attn_pack(dp[0][0], dp[0][1], (T)0.f), x2 = attn_pack(s[0][0], s[0][1], (T)0.f);
#pragma unroll
                for (int d = 0; d < 2 * NS; ++d) {
                    dk[0][d] = attn_mma(Tile::cols(lq, blk, d, lane), x1, dk[0][d]);
                    dv[0][d] = attn_mma(Tile::cols(lg, blk, d, lane), x2, dv[0][d]);
                }
            }
        }
    }
    if (mine) {
        const int64_t at = ((int64_t)start + 16 * wave) * ost_k + kvh * p.dim;
        char* const scratch = lds + 4 * G::kTileBytes + wave * 16 * G::kRow;
        attn_write_rows<T, NS>(scratch, dk[0], attn_grad_scale<DROP>(p) * kAttnUnlift<T> / gain_k, (T*)p.dk + at, ost_k, len - 16 * wave, p.dim, lane);
        attn_write_rows<T, NS>(scratch, dv[0], (DROP ? p.keep_scale : 1.f) * kAttnUnlift<T>, (T*)p.dv + at, ost_k, len - 16 * wave, p.dim, lane);
    }
}

// Documents of 65 to 128 rows: eight waves share one document of one key head, all four operands in LDS; each wave first takes 16 rows of
// queries (dQ; delta from the forward pass's output, corrected as below), then 16 of keys.  Bound by vector instructions, which are busy for
// two thirds of the time, a third of them the dropout's (161 documents of 65 to 101 rows, 12 heads of 64: 52 us).
// (ONE: no query heads share a key head; dK and dV then need no registers while dQ is made)
template <typename T, int NS, bool DROP, bool ONE>
__device__ __forceinline__ void attn_bwd_mid(const AttnParams& p, char* lds, float* row_lse, float* row_delta, uint32_t* row_state, const int4 e, int kvh) {
    typedef AttnGeom<T, NS> G;
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
    constexpr int E = (int)sizeof(T);
    constexpr bool kFix = sizeof(T) == 2;
    const int start = e.x, len = e.y, group = ONE ? 1 : p.heads / p.kv_heads;
    if (e.w) {
        for (int h = 0; h < group; ++h) attn_zero_rows((T*)p.dq, start, len, p.heads, kvh * group + h, p.dim, (int)threadIdx.x, 512);
        attn_zero_rows((T*)p.dk, start, len, p.kv_heads, kvh, p.dim, (int)threadIdx.x, 512);
        attn_zero_rows((T*)p.dv, start, len, p.kv_heads, kvh, p.dim, (int)threadIdx.x, 512);
        return;
    }
    const int tid = attn_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    char *const lk = lds, *const lv = lds + 2 * G::kTileBytes, *const lq = lds + 4 * G::kTileBytes, *const lg = lds + 6 * G::kTileBytes;
    const bool mine = 16 * wave < len;
    char* const scratch = (ONE ? lk : lq) + wave * 16 * G::kRow;
    const int row = 16 * wave + (lane & 15);
    const int64_t ost_q = (int64_t)p.heads * p.dim, ost_k = (int64_t)p.kv_heads * p.dim;
    int64_t seed = 0;
    if (DROP) seed = p.seed[0];
    AttnStage<T, NS, 512> a, b, c, d;
    auto fetch = [&](int head) {
        a.load((const char*)p.q.p + ((int64_t)start * p.q.st + head * p.q.sh) * E, p.q.st * E, len, p.dim, tid);
        b.load((const char*)p.go.p + ((int64_t)start * p.go.st + head * p.go.sh) * E, p.go.st * E, len, p.dim, tid);
    };
    c.load((const char*)p.k.p + ((int64_t)start * p.k.st + kvh * p.k.sh) * E, p.k.st * E, len, p.dim, tid);
    d.load((const char*)p.v.p + ((int64_t)start * p.v.st + kvh * p.v.sh) * E, p.v.st * E, len, p.dim, tid);
    fetch(kvh * group);
    c.store(lk, tid);
    d.store(lv, tid);
    f32x4 dk[2 * NS], dv[2 * NS];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) dk[i] = dv[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    float gain_k = kAttnGain<T>, unused_k = 0.f;
    if (!ONE) clear();
    for (int h = 0; h < group; ++h) {
        const int head = kvh * group + h;
        if (h) {
            fetch(head);
            __syncthreads();                           // (the head before is done with the tiles)
        }
        a.store(lq, tid);
        b.store(lg, tid);
        frag o[NS];                                    // the forward pass's output, for delta
        attn_load_row<T, NS>(o, (const char*)p.o.p + (((int64_t)start + row) * p.o.st + head * p.o.sh) * E, row < len, p.dim, lane);
        const float my_lse = row < len ? p.lse[(int64_t)head * p.total + start + row] - kAttnLift<T> : INFINITY;      // (probability 0)
        const uint32_t state = DROP ? attn_row_state(attn_head_state(seed, head), seed, (int64_t)start + row) : 0u;
        if (g == 0) {
            row_lse[row] = my_lse;
            if (DROP) row_state[row] = state;
        }
        __syncthreads();
        frag b1[1][NS], b2[1][NS];
        f32x4 dq[2 * NS];
        float gain = kAttnGain<T>;
        if (mine) {
            f32x4 fix[2 * NS];
            float delta = 0.f, over = 0.f, total = 0.f;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                b1[0][s] = Tile::rows(lq, wave, s, lane), b2[0][s] = Tile::rows(lg, wave, s, lane);
#pragma unroll
                for (int j = 0; j < 8; ++j) delta = __builtin_fmaf((float)o[s][j], (float)b2[0][s][j], delta);
            }
            delta = attn_sum4(delta);
            if (DROP) delta /= p.keep_scale;
#pragma unroll
            for (int i = 0; i < 2 * NS; ++i) dq[i] = fix[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int blk = 0; 32 * blk < len; ++blk) {
                f32x4 s[1][2], dp[1][2];
                attn_bwd_scores<T, NS, 1>(lk, lv, blk, b1, b2, s, dp, lane);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int key = 32 * blk + 16 * t + 4 * g;
                    if (DROP) attn_drop4(dp[0][t], state, (uint32_t)key, p.drop);
                    if (32 * (blk + 1) > len)                     // (keys past the last one)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (key + r >= len) s[0][t][r] = -INFINITY;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][t][r], p.scale2, -my_lse));
                        s[0][t][r] = pr;
                        dp[0][t][r] = pr * (dp[0][t][r] - delta);
                        over += dp[0][t][r];
                    }
                }
                attn_gain<T>(dp[0][0], dp[0][1], gain, total, dq);
                const frag x1 = attn_pack(dp[0][0], dp[0][1], (T)0.f), x2 = attn_pack(s[0][0], s[0][1], (T)0.f);
                if (kFix) total = attn_total(x1, total);
#pragma unroll
                for (int i = 0; i < 2 * NS; ++i) {
                    const frag k = Tile::cols(lk, blk, i, lane);
                    dq[i] = attn_mma(k, x1, dq[i]);
                    if (kFix) fix[i] = attn_mma(k, x2, fix[i]);
                }
            }
            if (kFix) {
                const float by = attn_sum4(total) * kAttnUnlift<T>;
                delta += attn_sum4(over) * kAttnUnlift<T>;
#pragma unroll
                for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) dq[i][j] = __builtin_fmaf(-by, fix[i][j], dq[i][j]);
            }
            if (g == 0) row_delta[row] = delta;
        } else if (g == 0) {
            row_delta[row] = 0.f;
        }
        __syncthreads();
        if (mine) {
#pragma unroll
            for (int s = 0; s < NS; ++s) b1[0][s] = Tile::rows(lk, wave, s, lane), b2[0][s] = Tile::rows(lv, wave, s, lane);
        }
        if (ONE) {                                     // (the keys and values are in registers now: the rows leave through their place)
            __syncthreads();
            if (mine)
                attn_write_rows<T, NS>(scratch, dq, attn_grad_scale<DROP>(p) * kAttnUnlift<T> / gain,
                                       (T*)p.dq + ((int64_t)start + 16 * wave) * ost_q + head * p.dim, ost_q, len - 16 * wave, p.dim, lane);
            clear();
        }
        if (mine) {
#pragma unroll 1
            for (int blk = 0; 32 * blk < len; ++blk) {
                f32x4 s[1][2], dp[1][2];
                attn_bwd_scores<T, NS, 1>(lq, lg, blk, b1, b2, s, dp, lane);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int mr = 32 * blk + 16 * t + 4 * g;
                    const f32x4 lse4 = *(const f32x4*)&row_lse[mr], delta4 = *(const f32x4*)&row_delta[mr];
                    bool keep[4];
                    if (DROP) attn_keep4(row_state + mr, (uint32_t)row, p.drop, keep);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][t][r], p.scale2, -lse4[r]));
                        float kept = pr, dd = dp[0][t][r];
                        if (DROP) {
                            kept = keep[r] ? pr : 0.f;
                            dd = keep[r] ? dd : 0.f;
                        }
                        s[0][t][r] = kept;
                        dp[0][t][r] = pr * (dd - delta4[r]);
                    }
                }
                attn_gain<T>(dp[0][0], dp[0][1], gain_k, unused_k, dk);
                const frag x1 = attn_pack(dp[0][0], dp[0][1], (T)0.f), x2 = attn_pack(s[0][0], s[0][1], (T)0.f);
#pragma unroll
                for (int i = 0; i < 2 * NS; ++i) {
                    dk[i] = attn_mma(Tile::cols(lq, blk, i, lane), x1, dk[i]);
                    dv[i] = attn_mma(Tile::cols(lg, blk, i, lane), x2, dv[i]);
                }
            }
        }
        if (ONE) break;
        __syncthreads();                               // (the rows leave through the queries' place)
        if (mine)
            attn_write_rows<T, NS>(scratch, dq, attn_grad_scale<DROP>(p) * kAttnUnlift<T> / gain, (T*)p.dq + ((int64_t)start + 16 * wave) * ost_q + head * p.dim, ost_q,
                                   len - 16 * wave, p.dim, lane);
    }
    if (mine) {
        const int64_t at = ((int64_t)start + 16 * wave) * ost_k + kvh * p.dim;
        attn_write_rows<T, NS>(scratch, dk, attn_grad_scale<DROP>(p) * kAttnUnlift<T> / gain_k, (T*)p.dk + at, ost_k, len - 16 * wave, p.dim, lane);
        attn_write_rows<T, NS>(scratch, dv, (DROP ? p.keep_scale : 1.f) * kAttnUnlift<T>, (T*)p.dv + at, ost_k, len - 16 * wave, p.dim, lane);
    }
}

// Longer ones.  KEYS: dK and dV of a tile of keys (the document's queries are streamed, for every query head that shares the key head);
// else: dQ of a tile of queries (its keys are streamed), and delta, which the KEYS launch behind it reads.
// delta from the forward pass's output is off by that output's rounding, the same for a whole row.  The error comes out of the pass itself:
// sum_j dX_ij is 0 by definition, so what the sums leave over is what delta lacks: the KEYS launch reads the corrected one.  dQ is corrected
// by the sum of the dX as rounded for the product, times sum_j P_ij K_j, an accumulator more: that takes delta's error out and of the
// roundings what acts along the mean of the keys (16-wide heads, whose keys of large P lie close: error 1.54 -> 1.43 of dQ's own rounding).
// Two launches: one that made all three gradients would add up dQ over workgroups by atomics, in an order that changes the result.  Bound by the
// matrix pipe and the vector instructions beside it (16 heads of 128, 4 key heads, 5 documents of 1900 to 8192 rows: dQ 1.47 ms, dK and dV 1.78 ms,
// 980 and 810 TFLOP/s of executed products).
template <typename T, int NS, int MS, bool DROP, bool KEYS>
__device__ __forceinline__ void attn_bwd_tile(const AttnParams& p, char* lds, float (*row_lse)[kAttnTile], float (*row_delta)[kAttnTile],
                                              uint32_t (*row_state)[kAttnTile], const int4 e, int head) {
    typedef AttnGeom<T, NS> G;
    typedef AttnTile<T, NS> Tile;
    typedef typename AttnType<T>::frag frag;
    const int heads = KEYS ? p.kv_heads : p.heads;
    const int64_t row0 = (int64_t)e.x + (int64_t)e.z * (kAttnTile * MS);
    const int nrows = min(kAttnTile * MS, e.y - e.z * (kAttnTile * MS));
    if (nrows <= 0) return;
    if (e.w) {
        attn_zero_rows((T*)(KEYS ? p.dk : p.dq), row0, nrows, heads, head, p.dim, (int)threadIdx.x, 256);
        if (KEYS) attn_zero_rows((T*)p.dv, row0, nrows, heads, head, p.dim, (int)threadIdx.x, 256);
        return;
    }
    constexpr int E = (int)sizeof(T);
    constexpr bool kTwo = KEYS || sizeof(T) == 2;      // (an fp32 output's rounding is none that its gradients would notice)
    const int tid = attn_thread(), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const int group = p.heads / p.kv_heads;
    const int head_q0 = KEYS ? head * group : head, head_kv = KEYS ? head : head / group;
    const int nt = (e.y - 1) / kAttnTile + 1;
    const int steps = KEYS ? nt * group : nt;
    auto tile1 = [&](int i) { return lds + (i & 1) * 2 * G::kTileBytes; };

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
        s1.load((const char*)t1.p + (((int64_t)e.x + at) * t1.st + hq * t1.sh) * E, st1, left, p.dim, tid);
        s2.load((const char*)t2.p + (((int64_t)e.x + at) * t2.st + hq * t2.sh) * E, st2, left, p.dim, tid);
        if (KEYS && threadIdx.x < kAttnTile) {
            const int64_t r = (int64_t)e.x + at + threadIdx.x;
            const bool in = (int)threadIdx.x < left;
            next_lse = in ? p.lse[(int64_t)hq * p.total + r] - kAttnLift<T> : INFINITY;      // (probability 0)
            next_delta = in ? p.delta[(int64_t)hq * p.total + r] : 0.f;
            if (DROP) next_state = attn_row_state(attn_head_state(seed, hq), seed, r);
        }
    };
    auto put = [&](int buf) {
        s1.store(tile1(buf), tid);
        s2.store(tile1(buf) + G::kTileBytes, tid);
        if (KEYS && threadIdx.x < kAttnTile) {
            row_lse[buf][threadIdx.x] = next_lse;
            row_delta[buf][threadIdx.x] = next_delta;
            if (DROP) row_state[buf][threadIdx.x] = next_state;
        }
    };
    fetch(0);
    frag b1[MS][NS], b2[MS][NS];
    float my_lse[MS], my_delta[MS], over[MS], total[MS], gain[MS];
    uint32_t my_state[MS];
    const int r0 = wave * 16 * MS + (lane & 15);
    const AttnTensor u1 = KEYS ? p.k : p.q, u2 = KEYS ? p.v : p.go;
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int r = r0 + 16 * m;
        const bool in = r < nrows;
        gain[m] = kAttnGain<T>;
        total[m] = 0.f;
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
            if (DROP) my_delta[m] /= p.keep_scale;
            my_lse[m] = in ? p.lse[(int64_t)head * p.total + row0 + r] - kAttnLift<T> : INFINITY;
            over[m] = 0.f;
            if (DROP) my_state[m] = attn_row_state(attn_head_state(seed, head), seed, row0 + r);
        }
    }
    put(0);
    __syncthreads();

    f32x4 acc1[MS][2 * NS], acc2[MS][2 * NS];
#pragma unroll
    for (int m = 0; m < MS; ++m)
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) acc1[m][d] = acc2[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int step = 0; step < steps; ++step) {
        const bool more = step + 1 < steps;
        if (more) fetch(step + 1);
        const int buf = step & 1;
        const int at = (KEYS ? step % nt : step) * kAttnTile, left = e.y - at;
        const char *const l1 = tile1(buf), *const l2 = l1 + G::kTileBytes;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            if (wave * 16 * MS >= nrows || 32 * blk >= left) continue;            // (nothing of this wave's, or of these 32 rows)
            f32x4 s[MS][2], dp[MS][2];
            attn_bwd_scores<T, NS, MS>(l1, l2, blk, b1, b2, s, dp, lane);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int mr = 16 * (2 * blk + t) + 4 * g;        // this lane's first streamed row of the tile
                f32x4 lse4, delta4;
                if (KEYS) {
                    lse4 = *(const f32x4*)&row_lse[buf][mr];
                    delta4 = *(const f32x4*)&row_delta[buf][mr];
                }
#pragma unroll
                for (int m = 0; m < MS; ++m) {
                    bool keep[4];
                    if (DROP && KEYS) attn_keep4(row_state[buf] + mr, (uint32_t)(e.z * (kAttnTile * MS) + r0 + 16 * m), p.drop, keep);
                    if (DROP && !KEYS) attn_drop4(dp[m][t], my_state[m], (uint32_t)(at + mr), p.drop);
                    if (!KEYS && left < kAttnTile)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (mr + r >= left) s[m][t][r] = -INFINITY;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[m][t][r], p.scale2, -(KEYS ? lse4[r] : my_lse[m])));
                        float kept = pr, d = dp[m][t][r];
                        if (DROP && KEYS) {
                            kept = keep[r] ? pr : 0.f;
                            d = keep[r] ? d : 0.f;
                        }
                        s[m][t][r] = kept;
                        dp[m][t][r] = pr * (d - (KEYS ? delta4[r] : my_delta[m]));
                        if (!KEYS) over[m] += dp[m][t][r];
                    }
                }
            }
            // probabilities and score gradients are rounded to the operands' type for the second products (32-bit sums)
            frag x1[MS], x2[MS];
#pragma unroll
            for (int m = 0; m < MS; ++m) {
                attn_gain<T>(dp[m][0], dp[m][1], gain[m], total[m], acc1[m]);
                x1[m] = attn_pack(dp[m][0], dp[m][1], (T)0.f);
                if (!KEYS) total[m] = attn_total(x1[m], total[m]);
                x2[m] = attn_pack(s[m][0], s[m][1], (T)0.f);
            }
            constexpr int kAhead = NS == 3 ? 3 : 4 < 2 * NS ? 4 : 2 * NS;         // (reads in flight together, as above)
#pragma unroll
            for (int d0 = 0; d0 < 2 * NS; d0 += kAhead) {
                frag a1[kAhead], a2[kAhead];
#pragma unroll
                for (int d = 0; d < kAhead; ++d) {
                    a1[d] = Tile::cols(l1, blk, d0 + d, lane);
                    a2[d] = KEYS ? Tile::cols(l2, blk, d0 + d, lane) : a1[d];
                }
                if (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < kAhead; ++d)
#pragma unroll
                    for (int m = 0; m < MS; ++m) {
                        acc1[m][d0 + d] = attn_mma(a1[d], x1[m], acc1[m][d0 + d]);
                        if (kTwo) acc2[m][d0 + d] = attn_mma(a2[d], x2[m], acc2[m][d0 + d]);
                    }
            }
        }
        if (more) put(buf ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < MS; ++m) {
        const int r = r0 + 16 * m, first = r - (lane & 15);
        const int64_t o = ((row0 + first) * heads + head) * p.dim, ost = (int64_t)heads * p.dim;
        char* const scratch = lds + wave * 16 * G::kRow;
        if (!KEYS) {
            const float lacks = kTwo ? attn_sum4(over[m]) * kAttnUnlift<T> : 0.f, by = kTwo ? attn_sum4(total[m]) * kAttnUnlift<T> : 0.f;
            if (r < nrows && g == 0) p.delta[(int64_t)head * p.total + row0 + r] = my_delta[m] + lacks;
            if (kTwo)
#pragma unroll
                for (int d = 0; d < 2 * NS; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc1[m][d][j] = __builtin_fmaf(-by, acc2[m][d][j], acc1[m][d][j]);
        }
        attn_write_rows<T, NS>(scratch, acc1[m], attn_grad_scale<DROP>(p) * kAttnUnlift<T> / gain[m], (T*)(KEYS ? p.dk : p.dq) + o, ost, nrows - first, p.dim, lane);
        if (KEYS) attn_write_rows<T, NS>(scratch, acc2[m], (DROP ? p.keep_scale : 1.f) * kAttnUnlift<T>, (T*)p.dv + o, ost, nrows - first, p.dim, lane);
    }
}

template <typename T, int NS, bool DROP>
__global__ __launch_bounds__(256, sizeof(T) == 2 && NS <= 2 ? 3 : 1) void attn_bwd_short_kernel(const AttnParams p) {
    __shared__ __attribute__((aligned(16))) char lds[(4 * kAttnTile + (sizeof(T) == 2 ? 64 : 0)) * AttnGeom<T, NS>::kRow];
    __shared__ __attribute__((aligned(16))) float row_lse[kAttnTile], row_delta[kAttnTile];
    __shared__ __attribute__((aligned(16))) uint32_t row_state[kAttnTile];
    attn_bwd_short<T, NS, DROP>(p, lds, row_lse, row_delta, row_state, blockIdx.y * gridDim.x + blockIdx.x);
}

template <typename T, int NS, bool DROP, bool ONE>
__global__ __launch_bounds__(512, ONE ? 4 : 2) void attn_bwd_mid_kernel(const AttnParams p) {
    __shared__ __attribute__((aligned(16))) char lds[8 * AttnGeom<T, NS>::kTileBytes];
    __shared__ __attribute__((aligned(16))) float row_lse[2 * kAttnTile], row_delta[2 * kAttnTile];
    __shared__ __attribute__((aligned(16))) uint32_t row_state[2 * kAttnTile];
    const int nm = p.nmids[0];
    const unsigned n = (unsigned)nm * (unsigned)p.kv_heads;
    for (unsigned i = blockIdx.x; i < n; i += gridDim.x) {
        attn_bwd_mid<T, NS, DROP, ONE>(p, lds, row_lse, row_delta, row_state, p.mids[i / (unsigned)p.kv_heads], (int)(i % (unsigned)p.kv_heads));
        __syncthreads();
    }
}

template <typename T, int NS, int MS, bool DROP, bool KEYS>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_bwd_kernel(const AttnParams p) {
    __shared__ __attribute__((aligned(16))) char lds[4 * AttnGeom<T, NS>::kTileBytes];
    __shared__ __attribute__((aligned(16))) float row_lse[2][kAttnTile], row_delta[2][kAttnTile];
    __shared__ __attribute__((aligned(16))) uint32_t row_state[2][kAttnTile];
    const int nt = p.ntiles[0], heads = KEYS ? p.kv_heads : p.heads;
    const unsigned n = attn_items(nt, heads);
    for (unsigned i = blockIdx.x; i < n; i += gridDim.x) {
        int tile, head;
        if (!attn_place(i, nt, heads, tile, head)) continue;
        attn_bwd_tile<T, NS, MS, DROP, KEYS>(p, lds, row_lse, row_delta, row_state, p.tiles[tile], head);
        __syncthreads();
    }
}

// launches for one element type (one source file each: they compile in parallel); mq: 16-row groups of a wave (the tiles are 64 * mq rows);
// most, most_mid: upper bounds of the numbers of tiles and of documents of 65 to 128 rows
template <typename T>
int attn_launch(const AttnParams& p, bool backward, int mq, int64_t most, int64_t most_mid, hipStream_t st);
extern template int attn_launch<__bf16>(const AttnParams&, bool, int, int64_t, int64_t, hipStream_t);
extern template int attn_launch<_Float16>(const AttnParams&, bool, int, int64_t, int64_t, hipStream_t);
extern template int attn_launch<float>(const AttnParams&, bool, int, int64_t, int64_t, hipStream_t);

template <typename T, int NS, int MQ, bool DROP>
int attn_launch_as(const AttnParams& p, bool backward, int64_t most, int64_t most_mid, hipStream_t st) {
    // The number of tiles is known to the device alone: up to 4096 workgroups (16 per CU) share them, a multiple of 8 (one XCD's items stay
    // its own), 1024 where the average document is no tile (idle, they cost a launch, 4 us).  With fewer possible tiles every one has its
    // workgroup.
    const int64_t share = p.total / p.nseg > 2 * kAttnTile ? 4096 : 1024;
    auto groups = [&](int heads) { return dim3((unsigned)std::min<int64_t>(round_up(most, 8) * heads, share)); };
    // (a launch has fewer than 2^32 threads in x: millions of documents go on in y)
    auto shorts = [](int64_t n) { return dim3((unsigned)std::min<int64_t>(n, 1 << 23), (unsigned)((n + (1 << 23) - 1) >> 23)); };
    auto mids = [&](int heads) { return dim3((unsigned)std::min<int64_t>(most_mid * heads, 2048)); };
    const dim3 wg(256);
    constexpr bool kMid = attn_has_mid(NS, sizeof(T));
    if (!backward) {
        if (p.shorts) hipLaunchKernelGGL((attn_fwd_short_kernel<T, NS, DROP>), shorts(((int64_t)p.nseg * p.heads + 3) / 4), wg, 0, st, p);
        LDOT_HIP_CHECK(hipGetLastError());
        if constexpr (kMid)
            if (most_mid) hipLaunchKernelGGL((attn_fwd_mid_kernel<T, NS, DROP>), mids(p.heads), dim3(512), 0, st, p);
        LDOT_HIP_CHECK(hipGetLastError());
        if (most) hipLaunchKernelGGL((attn_fwd_kernel<T, NS, MQ, DROP>), groups(p.heads), wg, 0, st, p);
        LDOT_HIP_CHECK(hipGetLastError());
        return LDOT_OK;
    }
    if (p.shorts) hipLaunchKernelGGL((attn_bwd_short_kernel<T, NS, DROP>), shorts((int64_t)p.nseg * p.kv_heads), wg, 0, st, p);
    LDOT_HIP_CHECK(hipGetLastError());
    if constexpr (kMid) {
        if (most_mid && p.heads == p.kv_heads) hipLaunchKernelGGL((attn_bwd_mid_kernel<T, NS, DROP, true>), mids(p.kv_heads), dim3(512), 0, st, p);
        else if (most_mid) hipLaunchKernelGGL((attn_bwd_mid_kernel<T, NS, DROP, false>), mids(p.kv_heads), dim3(512), 0, st, p);
        LDOT_HIP_CHECK(hipGetLastError());
    }
    if (!most) return LDOT_OK;
    constexpr int MS = attn_bwd_groups(NS, MQ);
    hipLaunchKernelGGL((attn_bwd_kernel<T, NS, MS, DROP, false>), groups(p.heads), wg, 0, st, p);
    LDOT_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((attn_bwd_kernel<T, NS, MS, DROP, true>), groups(p.kv_heads), wg, 0, st, p);
    LDOT_HIP_CHECK(hipGetLastError());
    return LDOT_OK;
}

template <typename T, int NS>
int attn_launch_ns(const AttnParams& p, bool backward, int mq, int64_t most, int64_t most_mid, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (mq == 2) return p.drop ? attn_launch_as<T, NS, 2, true>(p, backward, most, most_mid, st) : attn_launch_as<T, NS, 2, false>(p, backward, most, most_mid, st);
    }
    return p.drop ? attn_launch_as<T, NS, 1, true>(p, backward, most, most_mid, st) : attn_launch_as<T, NS, 1, false>(p, backward, most, most_mid, st);
}

template <typename T>
int attn_launch(const AttnParams& p, bool backward, int mq, int64_t most, int64_t most_mid, hipStream_t st) {
    switch ((p.dim + 31) / 32) {
        case 1: return attn_launch_ns<T, 1>(p, backward, mq, most, most_mid, st);
        case 2: return attn_launch_ns<T, 2>(p, backward, mq, most, most_mid, st);
        case 3: return attn_launch_ns<T, 3>(p, backward, mq, most, most_mid, st);
        default: return attn_launch_ns<T, 4>(p, backward, mq, most, most_mid, st);
    }
}

}  // namespace ldot
