// Attention over packed documents: the plan (which tiles there are) and the C entry points.
#include <algorithm>
#include <cmath>

#include "packed_attention.h"

namespace ldot {
namespace {

// Segments of the packed batch: [0, offsets[0]) and [offsets[n], total), which no document holds, around the n documents.  Offsets come
// from the device and are not read by the host: each is clamped to [largest one before it, total], so that no segment leaves the tensor
// and none overlaps another, whatever they are.  Lists: 0 and 1 hold the tiles, of 64 and of 128 rows, of segments of more than 128 rows, 2
// and 3 the same of more than 64 (for rows too wide for the kernels of 65 to 128 rows), 4 the segments of 65 to 128 rows, whole.  The
// kernels find shorter ones by their number.
constexpr int kLists = 5;
struct PlanView {
    int4* list[kLists];
    int64_t cap[kLists];
    int* kinds;          // [3]: 0 if no segment has 1 to 64 rows, 65 to 128, more
    int* count;          // [kLists]: how many there are
    int* bound;          // [nseg + 1]
    int* first[kLists];  // [nseg]: the place of a segment's first entry
    int nseg;
};

__device__ __forceinline__ int plan_entries(int list, int n) {
    if (list == 4) return n > kAttnTile && n <= 2 * kAttnTile;
    const int rows = kAttnTile << (list & 1);
    return n > (list < 2 ? 2 * kAttnTile : kAttnTile) ? (n - 1) / rows + 1 : 0;
}

// a segment of r rows has at most r / 64 + 1 tiles, and at most total / 65 segments have more than 64 rows (total / 129 more than 128)
int64_t plan_cap(int64_t ndocs, int64_t total, int list) {
    const int64_t some = std::min(ndocs + 2, total / (list < 2 ? 2 * kAttnTile + 1 : kAttnTile + 1));
    return some == 0 ? 0 : (list == 4 ? 0 : total / (kAttnTile << (list & 1))) + some;
}

PlanView plan_view(int32_t* buf, int64_t ndocs, int64_t total) {
    PlanView v;
    v.kinds = buf;
    char* p = (char*)(buf + 4);
    for (int w = 0; w < kLists; ++w) {
        v.cap[w] = plan_cap(ndocs, total, w);
        v.list[w] = (int4*)p;
        p += (size_t)v.cap[w] * sizeof(int4);
    }
    v.nseg = (int)ndocs + 2;
    v.count = (int*)p;
    v.bound = v.count + 8;
    for (int w = 0; w < kLists; ++w) v.first[w] = v.bound + (w + 1) * (int64_t)(v.nseg + 1);
    return v;
}

// running maximum over a workgroup of 1024
__device__ __forceinline__ int plan_max_scan(int* sh, int x) {
    const int t = (int)threadIdx.x, lane = t & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x = max(x, y);
    }
    if (lane == 63) sh[t >> 6] = x;
    __syncthreads();
    for (int w = 0; w < (t >> 6); ++w) x = max(x, sh[w]);
    return x;
}

// One workgroup: clamped bounds (running maximum, 1024 segments at a time), then the places of the segments' entries, long segments first:
// a place within a class of lengths goes by the order of arrival, which decides when a tile is worked on and nothing else.
constexpr int kClasses = 64;             // rows / 64, the last one open
template <typename I>
__global__ __launch_bounds__(1024) void plan_scan_kernel(const I* __restrict__ offsets, int64_t total, PlanView v) {
    __shared__ int sh[16], last, shorts, next[kLists][kClasses];
    const int t = (int)threadIdx.x;
    if (t == 0) shorts = 0;
    for (int i = t; i < kLists * kClasses; i += 1024) next[i / kClasses][i % kClasses] = 0;
    int top = 0;                                       // the largest offset of the blocks before
    for (int base = 0; base <= v.nseg; base += 1024) {
        const int i = base + t;                        // bound i: 0 -> 0, 1 .. n + 1 -> offsets[i - 1], n + 2 -> total
        int64_t b = 0;
        if (i >= 1 && i < v.nseg) b = (int64_t)offsets[i - 1];
        if (i >= v.nseg) b = total;
        b = b < 0 ? 0 : (b > total ? total : b);
        const int r = max(top, plan_max_scan(sh, (int)b));
        if (i <= v.nseg) v.bound[i] = r;
        if (t == 1023) last = r;
        __syncthreads();
        top = last;
        __syncthreads();
    }
    for (int i = t; i < v.nseg; i += 1024) {
        const int n = v.bound[i + 1] - v.bound[i], c = min(n / kAttnTile, kClasses - 1);
        for (int w = 0; w < kLists; ++w)
            if (const int k = plan_entries(w, n)) atomicAdd(&next[w][c], k);
        if (n > 0 && n <= kAttnTile) shorts = 1;       // (whoever writes it)
    }
    __syncthreads();
    if (t < kLists) {
        int before = 0;
        for (int c = kClasses - 1; c >= 0; --c) {
            const int k = next[t][c];
            next[t][c] = before;
            before += k;
        }
        v.count[t] = before;
        if (t == 0) v.kinds[0] = shorts, v.kinds[2] = before;
        if (t == 4) v.kinds[1] = before;
    }
    __syncthreads();
    for (int i = t; i < v.nseg; i += 1024) {
        const int n = v.bound[i + 1] - v.bound[i], c = min(n / kAttnTile, kClasses - 1);
        for (int w = 0; w < kLists; ++w) {
            const int k = plan_entries(w, n);
            v.first[w][i] = k ? atomicAdd(&next[w][c], k) : 0;
        }
    }
}

// a wave per segment writes its entries
__global__ __launch_bounds__(256) void plan_fill_kernel(PlanView v) {
    const int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (i >= v.nseg) return;
    const int start = v.bound[i], n = v.bound[i + 1] - start;
    for (int w = 0; w < kLists; ++w) {
        const int k = plan_entries(w, n);
        const int64_t first = v.first[w][i];
        for (int64_t j = lane; j < k && first + j < v.cap[w]; j += 64) v.list[w][first + j] = make_int4(start, n, (int)j, i == 0 || i == v.nseg - 1);
    }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_tensor(const void* p, int64_t st, int64_t sh, int esize, const char* name) {
    LDOT_REQUIRE(p != nullptr, LDOT_EINVAL, "%s is NULL", name);
    LDOT_REQUIRE(aligned16(p) && st * esize % 16 == 0 && sh * esize % 16 == 0, LDOT_EINVAL,
                 "%s: address and strides have to be multiples of 16 bytes", name);
    return LDOT_OK;
}

int attn_entry(const ldot_packed_attn* a, bool backward, void* stream) {
    LDOT_REQUIRE(a != nullptr, LDOT_EINVAL, "args is NULL");
    LDOT_REQUIRE(a->dtype == LDOT_F32 || a->dtype == LDOT_BF16 || a->dtype == LDOT_F16, LDOT_EINVAL, "bad dtype %d", a->dtype);
    LDOT_REQUIRE(a->ndocs >= 0 && a->total >= 0 && a->total < (1ll << 31) && a->ndocs < (1ll << 30), LDOT_EINVAL, "bad sizes: %lld documents, %lld tokens",
                 (long long)a->ndocs, (long long)a->total);
    LDOT_REQUIRE(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0, LDOT_EINVAL, "%d heads are no multiple of %d key heads", a->heads, a->kv_heads);
    LDOT_REQUIRE(a->dim > 0 && a->dim <= 128 && a->dim % 8 == 0, LDOT_EINVAL, "head size %d: a multiple of 8 up to 128 is needed", a->dim);
    const float scale2 = (float)((double)a->scale * 1.4426950408889634);
    LDOT_REQUIRE(std::isfinite(scale2) && a->scale > 0.f, LDOT_EINVAL, "scale has to be positive and finite, in base 2 too");
    LDOT_REQUIRE(a->dropout >= 0.f && a->dropout < 1.f, LDOT_EINVAL, "dropout has to be in [0, 1)");
    const uint32_t drop = (uint32_t)(a->dropout * 65536.0 + 0.5);
    LDOT_REQUIRE(drop < 65536u, LDOT_EINVAL, "dropout %g leaves nothing", (double)a->dropout);
    LDOT_REQUIRE(drop == 0 || a->seed != nullptr, LDOT_EINVAL, "dropout needs a seed");
    if (a->total == 0) return LDOT_OK;
    LDOT_REQUIRE(a->plan != nullptr, LDOT_EINVAL, "plan is NULL");
    const int es = a->dtype == LDOT_F32 ? 4 : 2;
    int rc;
    if ((rc = check_tensor(a->q, a->q_st, a->q_sh, es, "q"))) return rc;
    if ((rc = check_tensor(a->k, a->k_st, a->k_sh, es, "k"))) return rc;
    if ((rc = check_tensor(a->v, a->v_st, a->v_sh, es, "v"))) return rc;
    if ((rc = check_tensor(a->out, 0, 0, es, "out"))) return rc;
    if (backward) {
        if ((rc = check_tensor(a->grad, a->g_st, a->g_sh, es, "grad"))) return rc;
        LDOT_REQUIRE(a->lse && a->delta && a->dq && a->dk && a->dv, LDOT_EINVAL, "NULL buffer");
        LDOT_REQUIRE(aligned16(a->dq) && aligned16(a->dk) && aligned16(a->dv), LDOT_EINVAL, "gradients have to be aligned to 16 bytes");
    }
    // rows of a workgroup: a wave of 32 rows reads the streamed tiles from LDS half as often for the same products, but leaves short
    // documents' waves idle (12 heads of 64, forward / backward: 8 documents of 4096 rows 0.58 / 1.67 ms against 0.69 / 1.94 with waves of 16
    // rows; 100 documents of 129 to 200 rows 42 / 108 us against 39 / 94)
    const int mq = es == 2 && a->ndocs > 0 && a->total / a->ndocs >= 256 ? 2 : 1;
    const PlanView v = plan_view((int32_t*)a->plan, a->ndocs, a->total);
    AttnParams p{};
    p.q = AttnTensor{a->q, a->q_st, a->q_sh};
    p.k = AttnTensor{a->k, a->k_st, a->k_sh};
    p.v = AttnTensor{a->v, a->v_st, a->v_sh};
    p.o = AttnTensor{a->out, (int64_t)a->heads * a->dim, a->dim};
    p.go = AttnTensor{a->grad, a->g_st, a->g_sh};
    p.out = a->out;
    p.dq = a->dq;
    p.dk = a->dk;
    p.dv = a->dv;
    p.lse = a->lse;
    p.delta = a->delta;
    const int ns = (a->dim + 31) / 32;
    const bool mid = attn_has_mid(ns, (size_t)es);
    const int list = (backward ? attn_bwd_groups(ns, mq) : mq) - 1 + (mid ? 0 : 2);
    p.tiles = v.list[list];
    p.ntiles = v.count + list;
    p.mids = v.list[4];
    p.nmids = v.count + 4;
    p.bound = v.bound;
    p.nseg = v.nseg;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.dim = a->dim;
    p.total = a->total;
    p.scale = a->scale;
    p.scale2 = scale2;
    p.drop = drop;
    p.keep_scale = (float)(65536.0 / (65536.0 - drop));
    p.seed = a->seed;
    const int long_kinds = mid ? 4 : 6;
    const int64_t most = (a->absent & long_kinds) == long_kinds ? 0 : v.cap[list], most_mid = mid && !(a->absent & 2) ? v.cap[4] : 0;
    p.shorts = !(a->absent & 1);
    LDOT_REQUIRE((most + v.nseg) * p.heads < (1ll << 31) - 8192, LDOT_EINVAL, "too many tiles: %lld x %d heads", (long long)(most + v.nseg), p.heads);
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == LDOT_F32) return attn_launch<float>(p, backward, mq, most, most_mid, st);
    if (a->dtype == LDOT_BF16) return attn_launch<__bf16>(p, backward, mq, most, most_mid, st);
    return attn_launch<_Float16>(p, backward, mq, most, most_mid, st);
}

}  // namespace
}  // namespace ldot

using namespace ldot;

extern "C" {

int64_t ldot_packed_plan_ints(int64_t ndocs, int64_t total) {
    if (ndocs < 0 || total < 0 || total >= (1ll << 31) || ndocs >= (1ll << 30)) return -1;
    int64_t all = 4 + 8 + (kLists + 1) * (ndocs + 3);
    for (int w = 0; w < kLists; ++w) all += 4 * plan_cap(ndocs, total, w);
    return all;
}

int ldot_packed_plan(const void* offsets, int wide, int64_t ndocs, int64_t total, int32_t* plan, void* stream) {
    LDOT_REQUIRE(plan != nullptr && (offsets != nullptr), LDOT_EINVAL, "NULL buffer");
    LDOT_REQUIRE(ldot_packed_plan_ints(ndocs, total) >= 0, LDOT_EINVAL, "bad sizes: %lld documents, %lld tokens", (long long)ndocs, (long long)total);
    LDOT_REQUIRE(aligned16(plan), LDOT_EINVAL, "the plan has to be aligned to 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    const PlanView v = plan_view(plan, ndocs, total);
    if (wide)
        hipLaunchKernelGGL(plan_scan_kernel<int64_t>, dim3(1), dim3(1024), 0, st, (const int64_t*)offsets, total, v);
    else
        hipLaunchKernelGGL(plan_scan_kernel<int32_t>, dim3(1), dim3(1024), 0, st, (const int32_t*)offsets, total, v);
    LDOT_HIP_CHECK(hipGetLastError());
    if (v.cap[4] || v.cap[2]) {
        hipLaunchKernelGGL(plan_fill_kernel, dim3((unsigned)std::min((v.nseg + 3) / 4, 1 << 23), (unsigned)((v.nseg / 4 >> 23) + 1)), dim3(256), 0, st, v);
        LDOT_HIP_CHECK(hipGetLastError());
    }
    return LDOT_OK;
}

int ldot_packed_attn_fwd(const ldot_packed_attn* args, void* stream) { return attn_entry(args, false, stream); }
int ldot_packed_attn_bwd(const ldot_packed_attn* args, void* stream) { return attn_entry(args, true, stream); }

}  // extern "C"
