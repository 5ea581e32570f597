// Global gradient norm over many tensors, and clipping (torch.nn.utils.clip_grad_norm_ of train_itm.py:262):
//     norm = sqrt(sum_t sum_i x_ti^2)  or  max |x_ti|,     coef = min(1, max_norm / (norm + 1e-6)),     y = coef x
// Two passes over the gradients: the norm has to be known before the first element can be scaled, and the gradients of real towers
// (0.9 GB) do not fit a cache.  Bound by memory (two towers of 768, fp32, 886 MB read twice and written once: 569 us, 4.7 TB/s).  Few
// launches: the table of tensors rides in the kernel's arguments (no upload, nothing to keep alive, and a captured graph keeps its own copy),
// and where there are few partial sums every workgroup of the second pass joins them itself, in one fixed order.
#include <algorithm>
#include <cmath>
#include <vector>

#include "ldot_common.h"

namespace ldot {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipEntries = 160;        // tensors per launch: 160 * 24 bytes + the rest < 4 KB of arguments
constexpr int64_t kClipChunk = 32768;    // share of a workgroup, in elements: 8 * 4 loads of 16 bytes per thread, thousands of workgroups
constexpr int kClipInline = 512;         // partial sums that the second pass joins by itself (two loads per thread)

struct ClipEntry {
    const void* src;
    void* dst;
    uint32_t n;          // elements
    uint32_t first;      // first workgroup of this tensor in its launch * 4 + dtype
};
struct ClipTable {
    ClipEntry e[kClipEntries];
    int n, base;         // base: workgroups of the launches before
};
static_assert(sizeof(ClipTable) + 48 <= 4096, "kernel arguments");

__device__ __forceinline__ double clip_nan_max(double a, double b) { return (b > a || b != b) ? b : a; }

// 16 bytes of one element type <-> fp32
template <int DT>
struct ClipVec {
    static constexpr int N = DT == LDOT_F32 ? 4 : 8;
    static constexpr int E = DT == LDOT_F32 ? 4 : 2;
    static __device__ __forceinline__ float one(const char* p) {
        if (DT == LDOT_F32) return *(const float*)p;
        if (DT == LDOT_BF16) return (float)*(const __bf16*)p;
        return (float)*(const _Float16*)p;
    }
    static __device__ __forceinline__ void put(char* p, float v) {
        if (DT == LDOT_F32) *(float*)p = v;
        else if (DT == LDOT_BF16) *(__bf16*)p = (__bf16)v;
        else *(_Float16*)p = (_Float16)v;
    }
    union Vec {
        uint4 u;
        float f[4];
        __bf16 b[8];
        _Float16 h[8];
    };
    static __device__ __forceinline__ float get(const Vec& v, int i) { return DT == LDOT_F32 ? v.f[i & 3] : DT == LDOT_BF16 ? (float)v.b[i] : (float)v.h[i]; }
    static __device__ __forceinline__ void set(Vec& v, int i, float x) {
        if (DT == LDOT_F32) v.f[i & 3] = x;
        else if (DT == LDOT_BF16) v.b[i] = (__bf16)x;
        else v.h[i] = (_Float16)x;
    }
};

// the tensor that a workgroup works on, and its share of it
__device__ __forceinline__ const ClipEntry& clip_find(const ClipTable& t, int64_t& from, int64_t& to, int& dtype) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].first >> 2 <= blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const ClipEntry& e = t.e[lo];
    dtype = (int)(e.first & 3);
    from = ((int64_t)blockIdx.x - (e.first >> 2)) * kClipChunk;
    to = min((int64_t)e.n, from + kClipChunk);
    return e;
}

template <bool INF, int DT>
__device__ __forceinline__ double clip_part(const char* src, int64_t n) {
    typedef ClipVec<DT> V;
    // squares and their sums in 64 bits: no gradient overflows or vanishes in them, and a long sum loses nothing
    double acc[4] = {0., 0., 0., 0.};
    const int64_t head = min(n, (int64_t)((16 - ((uintptr_t)src & 15)) & 15) / V::E);
    const int64_t nv = (n - head) / V::N;
    auto take = [&](float x, int i) {
        if (INF) acc[i & 3] = clip_nan_max(acc[i & 3], (double)fabsf(x));
        else acc[i & 3] = __builtin_fma((double)x, (double)x, acc[i & 3]);
    };
    const uint4* v = (const uint4*)(src + head * V::E);
    int64_t i = threadIdx.x;
    for (; i + 3 * kClipThreads < nv; i += 4 * kClipThreads) {
        typename V::Vec a[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j].u = v[i + j * kClipThreads];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < V::N; ++k) take(V::get(a[j], k), k);
    }
    for (; i < nv; i += kClipThreads) {
        typename V::Vec a;
        a.u = v[i];
#pragma unroll
        for (int k = 0; k < V::N; ++k) take(V::get(a, k), k);
    }
    // elements before the first and behind the last 16 bytes
    if ((int64_t)threadIdx.x < head) take(V::one(src + threadIdx.x * V::E), 0);
    const int64_t tail = head + nv * V::N + threadIdx.x;
    if (tail < n) take(V::one(src + tail * V::E), 1);
    if (INF) return clip_nan_max(clip_nan_max(acc[0], acc[1]), clip_nan_max(acc[2], acc[3]));
    return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

// over the workgroup, in one fixed order
template <bool INF, int THREADS = kClipThreads>
__device__ __forceinline__ double clip_join(double x) {
    __shared__ double sh[THREADS / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const double y = __shfl_xor(x, o);
        x = INF ? clip_nan_max(x, y) : x + y;
    }
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    x = sh[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) x = INF ? clip_nan_max(x, sh[i]) : x + sh[i];
    return x;
}

template <bool INF>
__global__ __launch_bounds__(kClipThreads) void clip_norm_kernel(const ClipTable t, double* __restrict__ partial) {
    int64_t from, to;
    int dtype;
    const ClipEntry& e = clip_find(t, from, to, dtype);
    double x;
    if (dtype == LDOT_F32) x = clip_part<INF, LDOT_F32>((const char*)e.src + from * 4, to - from);
    else if (dtype == LDOT_BF16) x = clip_part<INF, LDOT_BF16>((const char*)e.src + from * 2, to - from);
    else x = clip_part<INF, LDOT_F16>((const char*)e.src + from * 2, to - from);
    x = clip_join<INF>(x);
    if (threadIdx.x == 0) partial[t.base + blockIdx.x] = x;
}

// the total out of the partial results: whoever adds them does it in the same order
template <bool INF, int THREADS>
__device__ __forceinline__ double clip_total(const double* __restrict__ partial, int n) {
    double x = 0.;
    for (int i = threadIdx.x; i < n; i += THREADS) x = INF ? clip_nan_max(x, partial[i]) : x + partial[i];
    x = clip_join<INF, THREADS>(x);
    return INF ? x : sqrt(x);
}

__device__ __forceinline__ float clip_coef(double total, double max_norm) {
    const double c = max_norm / (total + 1e-6);
    return c > 1. ? 1.f : (float)c;                        // (NaN stays NaN)
}

template <int DT>
__device__ __forceinline__ void clip_scale(const char* src, char* dst, int64_t n, float coef) {
    typedef ClipVec<DT> V;
    const int64_t head = min(n, (int64_t)((16 - ((uintptr_t)src & 15)) & 15) / V::E);
    const bool wide = (((uintptr_t)dst + head * V::E) & 15) == 0;
    const int64_t nv = (n - head) / V::N;
    const uint4* v = (const uint4*)(src + head * V::E);
    char* d = dst + head * V::E;
    auto store = [&](int64_t at, typename V::Vec& a) {
#pragma unroll
        for (int k = 0; k < V::N; ++k) V::set(a, k, V::get(a, k) * coef);
        if (wide) {
            *((uint4*)d + at) = a.u;
        } else {
#pragma unroll
            for (int k = 0; k < V::N; ++k) V::put(d + (at * V::N + k) * V::E, V::get(a, k));
        }
    };
    int64_t i = threadIdx.x;
    for (; i + 3 * kClipThreads < nv; i += 4 * kClipThreads) {
        typename V::Vec a[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j].u = v[i + j * kClipThreads];
#pragma unroll
        for (int j = 0; j < 4; ++j) store(i + j * kClipThreads, a[j]);
    }
    for (; i < nv; i += kClipThreads) {
        typename V::Vec a;
        a.u = v[i];
        store(i, a);
    }
    if ((int64_t)threadIdx.x < head) V::put(dst + threadIdx.x * V::E, V::one(src + threadIdx.x * V::E) * coef);
    const int64_t tail = head + nv * V::N + threadIdx.x;
    if (tail < n) V::put(dst + tail * V::E, V::one(src + tail * V::E) * coef);
}

// npartial 0: the coefficient is there already
template <bool INF>
__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(const ClipTable t, const double* __restrict__ partial, int npartial, double max_norm,
                                                                  const float* __restrict__ ready, float* __restrict__ norm) {
    float coef;
    if (npartial) {
        const double total = clip_total<INF, kClipThreads>(partial, npartial);
        if (t.base == 0 && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)total;
        coef = clip_coef(total, max_norm);
    } else {
        coef = ready[0];
    }
    int64_t from, to;
    int dtype;
    const ClipEntry& e = clip_find(t, from, to, dtype);
    if (coef == 1.f && e.src == e.dst) return;             // nothing changes
    const int es = dtype == LDOT_F32 ? 4 : 2;
    const char* s = (const char*)e.src + from * es;
    char* d = (char*)e.dst + from * es;
    if (dtype == LDOT_F32) clip_scale<LDOT_F32>(s, d, to - from, coef);
    else if (dtype == LDOT_BF16) clip_scale<LDOT_BF16>(s, d, to - from, coef);
    else clip_scale<LDOT_F16>(s, d, to - from, coef);
}

template <bool INF>
__global__ __launch_bounds__(1024) void clip_total_kernel(const double* __restrict__ partial, int npartial, double max_norm, float* __restrict__ coef,
                                                          float* __restrict__ norm) {
    const double total = clip_total<INF, 1024>(partial, npartial);
    if (threadIdx.x == 0) {
        norm[0] = (float)total;
        coef[0] = clip_coef(total, max_norm);
    }
}

struct Span {
    uintptr_t from, to;
    bool dst;
};

}  // namespace
}  // namespace ldot

using namespace ldot;

extern "C" {

// (one more than there are partial sums: the coefficient lies behind them)
int64_t ldot_clip_grad_partials(const int64_t* numel, int n) {
    if (n < 0 || (n > 0 && !numel)) return -1;
    int64_t all = 1;
    for (int i = 0; i < n; ++i) all += (std::max<int64_t>(numel[i], 0) + kClipChunk - 1) / kClipChunk;
    return all;
}

int ldot_clip_grad(const void* const* src, void* const* dst, const int64_t* numel, const int* dtype, int n, double max_norm, int norm_inf,
                   double* partial, float* norm, void* stream) {
    LDOT_REQUIRE(n >= 0 && partial && norm, LDOT_EINVAL, "NULL buffer");
    LDOT_REQUIRE(n == 0 || (src && numel && dtype), LDOT_EINVAL, "NULL list");
    LDOT_REQUIRE(!(max_norm < 0) && max_norm == max_norm, LDOT_EINVAL, "max_norm has to be >= 0");
    for (int i = 0; i < n; ++i) {
        LDOT_REQUIRE(dtype[i] == LDOT_F32 || dtype[i] == LDOT_BF16 || dtype[i] == LDOT_F16, LDOT_EINVAL, "tensor %d: bad dtype %d", i, dtype[i]);
        LDOT_REQUIRE(numel[i] >= 0 && (numel[i] == 0 || (src[i] && (!dst || dst[i]))), LDOT_EINVAL, "tensor %d: NULL address or bad size", i);
        const uintptr_t es = dtype[i] == LDOT_F32 ? 4 : 2;
        LDOT_REQUIRE(numel[i] == 0 || ((uintptr_t)src[i] % es == 0 && (!dst || (uintptr_t)dst[i] % es == 0)), LDOT_EINVAL, "tensor %d: address is not aligned to its elements", i);
    }
    if (dst) {
        // a destination that overlaps anything but its own source would be read or written by two workgroups in any order
        try {
            std::vector<Span> s;
            s.reserve(2 * (size_t)n);
            for (int i = 0; i < n; ++i) {
                if (!numel[i]) continue;
                const uintptr_t b = (uintptr_t)numel[i] * (dtype[i] == LDOT_F32 ? 4 : 2);
                s.push_back(Span{(uintptr_t)dst[i], (uintptr_t)dst[i] + b, true});
                if (dst[i] != src[i]) s.push_back(Span{(uintptr_t)src[i], (uintptr_t)src[i] + b, false});
            }
            std::sort(s.begin(), s.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
            uintptr_t end_dst = 0, end_any = 0;
            for (const Span& x : s) {
                LDOT_REQUIRE(x.from >= end_dst && (!x.dst || x.from >= end_any), LDOT_EINVAL, "a destination overlaps another tensor of the list");
                end_any = std::max(end_any, x.to);
                if (x.dst) end_dst = std::max(end_dst, x.to);
            }
        } catch (...) {
            LDOT_REQUIRE(false, LDOT_ENOMEM, "out of host memory");
        }
    }
    hipStream_t st = (hipStream_t)stream;
    const int64_t all = ldot_clip_grad_partials(numel, n) - 1;
    LDOT_REQUIRE(all < (1ll << 29), LDOT_EINVAL, "too many elements");
    const int npartial = (int)all;
    float* const coef = (float*)(partial + npartial);
    // (the partial sums' order goes by their number: by one workgroup of 1024, or by every workgroup of the second pass, of 256)
    const bool inline_join = dst && npartial && npartial <= kClipInline;
    constexpr int64_t kMost = 1ll << 31;                   // elements of an entry: a multiple of the share
    // pass 0: partial norms, pass 1: scaling
    for (int pass = 0; pass < (dst && npartial ? 2 : 1); ++pass) {
        int i = 0, base = 0;
        int64_t done = 0;                                  // elements of tensor i in the launches before
        while (i < n) {
            ClipTable t;
            t.n = 0;
            t.base = base;
            int64_t blocks = 0;
            while (i < n && t.n < kClipEntries) {
                const int64_t es = dtype[i] == LDOT_F32 ? 4 : 2, len = std::min(numel[i] - done, kMost);
                if (len > 0) {
                    t.e[t.n++] = ClipEntry{(const char*)src[i] + done * es, dst ? (char*)dst[i] + done * es : nullptr, (uint32_t)len, (uint32_t)blocks * 4 + (uint32_t)dtype[i]};
                    blocks += (len + kClipChunk - 1) / kClipChunk;
                }
                done += len;
                if (done >= numel[i]) ++i, done = 0;
            }
            if (!t.n) break;
            const dim3 grid((unsigned)blocks), wg(kClipThreads);
            if (pass == 0) {
                if (norm_inf) hipLaunchKernelGGL(clip_norm_kernel<true>, grid, wg, 0, st, t, partial);
                else hipLaunchKernelGGL(clip_norm_kernel<false>, grid, wg, 0, st, t, partial);
            } else {
                const int join = inline_join ? npartial : 0;
                if (norm_inf) hipLaunchKernelGGL(clip_scale_kernel<true>, grid, wg, 0, st, t, partial, join, max_norm, coef, norm);
                else hipLaunchKernelGGL(clip_scale_kernel<false>, grid, wg, 0, st, t, partial, join, max_norm, coef, norm);
            }
            LDOT_HIP_CHECK(hipGetLastError());
            base += (int)blocks;
        }
        if (pass == 0 && !inline_join) {                   // (the norm of an empty list: 0)
            if (norm_inf) hipLaunchKernelGGL(clip_total_kernel<true>, dim3(1), dim3(1024), 0, st, partial, npartial, max_norm, coef, norm);
            else hipLaunchKernelGGL(clip_total_kernel<false>, dim3(1), dim3(1024), 0, st, partial, npartial, max_norm, coef, norm);
            LDOT_HIP_CHECK(hipGetLastError());
        }
    }
    return LDOT_OK;
}

}  // extern "C"
