// grad_norm.hip -- the norm of many gradient tensors at once, and clipping by it
// (second/pytorch/train.py:342: clip_grad_norm_(parameters, 10) in every training step).
//
//   norm = (sum over all tensors and elements of |g|^p)^(1/p),   out = g * min(1, m / (norm + 1e-6))
//
// Bound by memory: the sum has to be known before the first output, so every gradient is read
// twice and written once.  The tensors' addresses travel as kernel arguments (GN_TENSORS of them in
// a launch: 4 KB is what a kernel's arguments may take), so nothing has to be uploaded, kept or
// freed, and a captured graph holds its own copy.  A launch cuts its tensors into chunks of
// GN_CHUNK elements; a workgroup finds a chunk's tensor by bisection over the first chunk numbers.
// Measured: 57 M bf16 elements to fp32 in one launch, sums 35 us (3.3 TB/s; neither fp32 squares nor
// other chunk and grid sizes are faster, and what bounds them is not shown), scaling 69 us (5.0 TB/s,
// what a large copy reaches); 400 tensors of 200 M elements 379 us a call; 1.85 M fp32 elements in 78
// tensors 5.2 + 7.5 us.
#include "rows.h"

#define GN_TENSORS 120
#define GN_CHUNK 8192 // elements: 256 threads x 8 elements x 4
#define GN_BLOCKS 2048 // workgroups of a summing launch, i.e. its parts

struct GnList {
    const void *g[GN_TENSORS];
    void *out[GN_TENSORS];
    long long n[GN_TENSORS];
    int chunk0[GN_TENSORS + 1]; // first chunk of each tensor; [count] = chunks of the launch
    int count;
};
static_assert(sizeof(GnList) <= 3840, "kernel arguments");

__device__ __forceinline__ int gn_find(const GnList &l, int chunk)
{
    int lo = 0, hi = l.count - 1; // the last tensor whose first chunk is <= chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.chunk0[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// one term of the sum; P 0: the largest magnitude, NaN winning
template <int P> __device__ __forceinline__ void gn_add(double &acc, float v)
{
    if constexpr (P == 2) {
        const double d = (double)v;
        acc = fma(d, d, acc);
    } else if constexpr (P == 1) {
        acc += (double)__builtin_fabsf(v);
    } else {
        const double d = (double)__builtin_fabsf(v);
        acc = (d > acc || d != d) ? d : acc;
    }
}
template <int P> __device__ __forceinline__ double gn_join(double a, double b)
{
    if constexpr (P == 0) return (b > a || b != b) ? b : a;
    else return a + b;
}

// sum over a workgroup in a fixed order; the result is valid in thread 0
template <int P> __device__ __forceinline__ double gn_block_sum(double v, double *lds)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = gn_join<P>(v, __shfl_down(v, d, 64));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = gn_join<P>(v, lds[w]);
    return v;
}

template <typename T, int P>
__global__ void __launch_bounds__(256) gn_sum_kernel(GnList l, double *__restrict__ parts)
{
    __shared__ double lds[4];
    double acc[2] = {0.0, 0.0};
    const int chunks = l.chunk0[l.count];
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int t = gn_find(l, chunk);
        const long long off = (long long)(chunk - l.chunk0[t]) * GN_CHUNK;
        const T *g = (const T *)l.g[t] + off;
        const long long left = l.n[t] - off;
        if (left >= GN_CHUNK) {
            float v[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i) lcf_ld8(g + (i * 256 + threadIdx.x) * 8, v[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) gn_add<P>(acc[j & 1], v[i][j]);
        } else {
            for (int i = threadIdx.x * 8; i < (int)left; i += 2048) {
                float v[8];
                lcf_ld8_tail(g, i, (int)left, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) gn_add<P>(acc[j & 1], v[j]);
            }
        }
    }
    const double s = gn_block_sum<P>(gn_join<P>(acc[0], acc[1]), lds);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

__device__ __forceinline__ float gn_coef(float total, float max_norm)
{
    const float c = max_norm / (total + 1e-6f);
    return c > 1.f ? 1.f : c; // a NaN stays one
}

// the norm out of the parts of all launches, in a fixed order; valid in thread 0
__device__ __forceinline__ float gn_total(const double *__restrict__ parts, int nparts, int p, double *lds)
{
    double acc = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < nparts; i += blockDim.x) acc = p ? acc + parts[i] : gn_join<0>(acc, parts[i]);
    acc = p ? gn_block_sum<2>(acc, lds) : gn_block_sum<0>(acc, lds);
    return (float)(p == 2 ? sqrt(acc) : acc);
}

// norm, and the factor that the clip multiplies by
__global__ void __launch_bounds__(1024) gn_final_kernel(const double *__restrict__ parts, int nparts, int p, float max_norm,
                                                       float *__restrict__ norm, float *__restrict__ coef)
{
    __shared__ double lds[16];
    const float total = gn_total(parts, nparts, p, lds);
    if (threadIdx.x == 0) {
        *norm = total;
        *coef = gn_coef(total, max_norm);
    }
}

// nparts > 0: every workgroup joins the parts itself (a few loads out of L2), which saves the launch
// of gn_final_kernel; the first one writes the norm
template <typename T, typename O>
__global__ void __launch_bounds__(256) gn_scale_kernel(GnList l, const double *__restrict__ parts, int nparts, int p,
                                                       float max_norm, float *__restrict__ norm,
                                                       const float *__restrict__ coef)
{
    __shared__ double lds[4];
    __shared__ float shared;
    float c;
    if (nparts > 0) {
        const float total = gn_total(parts, nparts, p, lds);
        if (threadIdx.x == 0) {
            shared = gn_coef(total, max_norm);
            if (blockIdx.x == 0) *norm = total;
        }
        __syncthreads();
        c = shared;
    } else {
        c = *coef;
    }
    const int chunks = l.chunk0[l.count];
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int t = gn_find(l, chunk);
        const long long off = (long long)(chunk - l.chunk0[t]) * GN_CHUNK;
        const T *g = (const T *)l.g[t] + off;
        O *out = (O *)l.out[t] + off;
        const long long left = l.n[t] - off;
        if (left >= GN_CHUNK) {
            float v[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i) lcf_ld8(g + (i * 256 + threadIdx.x) * 8, v[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] *= c;
                lcf_st8(out + (i * 256 + threadIdx.x) * 8, v[i]);
            }
        } else {
            for (int i = threadIdx.x * 8; i < (int)left; i += 2048) {
                float v[8];
                lcf_ld8_tail(g, i, (int)left, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= c;
                lcf_st8_tail(out, i, (int)left, v);
            }
        }
    }
}

// All of it in one workgroup, for a few thousand elements, where launches are all the time there is:
// a wave takes a chunk, the sums meet in LDS, and the second reading comes out of the cache.
template <typename T, typename O, int P>
__global__ void __launch_bounds__(1024) gn_one_kernel(GnList l, float max_norm, float *__restrict__ norm)
{
    __shared__ double lds[16];
    __shared__ float shared;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, chunks = l.chunk0[l.count];
    double acc = 0.0;
    for (int chunk = wave; chunk < chunks; chunk += 16) {
        const int t = gn_find(l, chunk);
        const long long off = (long long)(chunk - l.chunk0[t]) * GN_CHUNK;
        const T *g = (const T *)l.g[t] + off;
        const int left = (int)(l.n[t] - off < GN_CHUNK ? l.n[t] - off : GN_CHUNK);
#pragma unroll 4
        for (int i = lane * 8; i < left; i += 512) {
            float v[8];
            lcf_ld8_tail(g, i, left, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) gn_add<P>(acc, v[j]);
        }
    }
    const double s = gn_block_sum<P>(acc, lds);
    if (threadIdx.x == 0) {
        const float total = (float)(P == 2 ? sqrt(s) : s);
        *norm = total;
        shared = gn_coef(total, max_norm);
    }
    __syncthreads();
    const float c = shared;
    for (int chunk = wave; chunk < chunks; chunk += 16) {
        const int t = gn_find(l, chunk);
        const long long off = (long long)(chunk - l.chunk0[t]) * GN_CHUNK;
        const T *g = (const T *)l.g[t] + off;
        O *out = (O *)l.out[t] + off;
        const int left = (int)(l.n[t] - off < GN_CHUNK ? l.n[t] - off : GN_CHUNK);
#pragma unroll 4
        for (int i = lane * 8; i < left; i += 512) {
            float v[8];
            lcf_ld8_tail(g, i, left, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= c;
            lcf_st8_tail(out, i, left, v);
        }
    }
}

// ---------------------------------------------------------------- host
#include <algorithm>
#include <new>

static bool gn_table_ok(const lcf_grad *t, int count, int p, bool clip)
{
    if (count < 0 || (count > 0 && !t) || (p != 0 && p != 1 && p != 2)) return false;
    for (int i = 0; i < count; ++i) {
        if (t[i].n < 0 || t[i].n > (1ll << 40) || !lcf_is_type(t[i].dtype)) return false;
        if (t[i].n > 0 && !t[i].g) return false;
        if (clip && (!lcf_is_type(t[i].out_dtype) || (t[i].n > 0 && !t[i].out))) return false;
    }
    return true;
}

// Two workgroups may not write the same bytes, and none may write what another still reads: sorts
// the ranges by address and looks at neighbours.  0 = apart, 1 = they overlap, -1 = no host memory.
static int gn_overlap(const lcf_grad *t, int count)
{
    struct Range {
        uintptr_t a, b;
        int i, kind; // 0: read, 1: written, 2: both (clipped in place)
    };
    Range *r = new (std::nothrow) Range[2 * (size_t)count];
    if (!r) return -1;
    int n = 0;
    for (int i = 0; i < count; ++i) {
        if (t[i].n == 0) continue;
        const uintptr_t g = (uintptr_t)t[i].g, o = (uintptr_t)t[i].out;
        const uintptr_t gb = (uintptr_t)t[i].n * lcf_type_size(t[i].dtype);
        const uintptr_t ob = (uintptr_t)t[i].n * lcf_type_size(t[i].out_dtype);
        if (g == o && t[i].dtype == t[i].out_dtype) {
            r[n++] = {g, g + gb, i, 2};
        } else {
            r[n++] = {g, g + gb, i, 0};
            r[n++] = {o, o + ob, i, 1};
        }
    }
    std::sort(r, r + n, [](const Range &x, const Range &y) { return x.a < y.a; });
    uintptr_t read_end = 0, write_end = 0; // furthest ends of what came before
    int bad = 0;
    for (int i = 0; i < n && !bad; ++i) {
        if (r[i].a < write_end) bad = 1;
        if (r[i].kind != 0 && r[i].a < read_end) bad = 1;
        if (r[i].kind != 1) read_end = std::max(read_end, r[i].b);
        if (r[i].kind != 0) write_end = std::max(write_end, r[i].b);
    }
    delete[] r;
    return bad;
}

// Calls fn(list, dtype, out_dtype) for runs of at most GN_TENSORS tensors of one pair of types and at
// most 2^30 chunks.  (Scaling from the last tensor to the first, for what the caches still hold of the
// sums' reading, measured slower: 75 us against 68 for 57 M bf16 elements.)
template <typename F> static int gn_launches(const lcf_grad *t, int count, bool clip, F fn)
{
    for (int ab = 0; ab < (clip ? 9 : 3); ++ab) {
        const int a = ab % 3, b = ab / 3;
        GnList l;
        l.count = 0;
        long long chunks = 0;
        for (int i = 0; i <= count; ++i) {
            const bool take = i < count && t[i].n > 0 && t[i].dtype == a && (!clip || t[i].out_dtype == b);
            const long long c = take ? (t[i].n + GN_CHUNK - 1) / GN_CHUNK : 0;
            if (l.count && (i == count || (take && (l.count == GN_TENSORS || chunks + c > (1ll << 30))))) {
                l.chunk0[l.count] = (int)chunks;
                const int rc = fn(l, a, b);
                if (rc != LCF_OK) return rc;
                l.count = 0;
                chunks = 0;
            }
            if (take) {
                l.g[l.count] = t[i].g;
                l.out[l.count] = t[i].out;
                l.n[l.count] = t[i].n;
                l.chunk0[l.count++] = (int)chunks;
                chunks += c;
            }
        }
    }
    return LCF_OK;
}

template <int P> static void gn_sum_launch(const GnList &l, int dtype, int grid, double *parts, hipStream_t st)
{
    if (dtype == LCF_F32) gn_sum_kernel<float, P><<<grid, 256, 0, st>>>(l, parts);
    else if (dtype == LCF_BF16) gn_sum_kernel<lcf_b, P><<<grid, 256, 0, st>>>(l, parts);
    else gn_sum_kernel<lcf_h, P><<<grid, 256, 0, st>>>(l, parts);
}

struct GnScale { // what a scale launch needs besides its list
    const double *parts;
    int nparts, p;
    float max_norm, *norm;
    const float *coef;
};
template <typename T> static void gn_scale_launch(const GnList &l, int od, int grid, const GnScale &s, hipStream_t st)
{
#define GN_SCALE(O) \
    gn_scale_kernel<T, O><<<grid, 256, 0, st>>>(l, s.parts, s.nparts, s.p, s.max_norm, s.norm, s.coef)
    if (od == LCF_F32) GN_SCALE(float);
    else if (od == LCF_BF16) GN_SCALE(lcf_b);
    else GN_SCALE(lcf_h);
#undef GN_SCALE
}

template <typename T> static void gn_one_launch(const GnList &l, int od, int p, float max_norm, float *norm, hipStream_t st)
{
#define GN_ONE(O)                                                                     \
    if (p == 2) gn_one_kernel<T, O, 2><<<1, 1024, 0, st>>>(l, max_norm, norm);        \
    else if (p == 1) gn_one_kernel<T, O, 1><<<1, 1024, 0, st>>>(l, max_norm, norm);   \
    else gn_one_kernel<T, O, 0><<<1, 1024, 0, st>>>(l, max_norm, norm)
    if (od == LCF_F32) { GN_ONE(float); }
    else if (od == LCF_BF16) { GN_ONE(lcf_b); }
    else { GN_ONE(lcf_h); }
#undef GN_ONE
}

// runs of tensors that gn_launches can make of `count`: full ones, plus one begun run per type
static size_t gn_runs(int count) { return (size_t)(count > 0 ? count : 0) / GN_TENSORS + 4; }

extern "C" size_t lcf_grad_norm_workspace_bytes(int count)
{
    return 256 + gn_runs(count) * GN_BLOCKS * sizeof(double);
}

// the sums; *nparts of them
static int gn_sums(const lcf_grad *t, int count, int p, double *parts, size_t room, int *nparts, hipStream_t st)
{
    *nparts = 0;
    return gn_launches(t, count, false, [&](const GnList &l, int dtype, int) -> int {
        const int chunks = l.chunk0[l.count];
        const int grid = chunks < GN_BLOCKS ? chunks : GN_BLOCKS;
        if ((size_t)*nparts + grid > room) return LCF_ERR_WORKSPACE;
        if (p == 2) gn_sum_launch<2>(l, dtype, grid, parts + *nparts, st);
        else if (p == 1) gn_sum_launch<1>(l, dtype, grid, parts + *nparts, st);
        else gn_sum_launch<0>(l, dtype, grid, parts + *nparts, st);
        *nparts += grid;
        LCF_CHECK_LAUNCH();
        return LCF_OK;
    });
}

extern "C" int lcf_grad_norm(const lcf_grad *grads, int count, int p, float *norm, void *ws, size_t ws_bytes,
                             void *stream)
{
    if (!gn_table_ok(grads, count, p, false) || !norm || !ws) return LCF_ERR_ARG;
    if (ws_bytes < lcf_grad_norm_workspace_bytes(count)) return LCF_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    double *parts = (double *)((char *)ws + 256);
    int nparts;
    const int rc = gn_sums(grads, count, p, parts, (ws_bytes - 256) / sizeof(double), &nparts, st);
    if (rc != LCF_OK) return rc;
    gn_final_kernel<<<1, 1024, 0, st>>>(parts, nparts, p, 1.f, norm, (float *)ws);
    LCF_CHECK_LAUNCH();
    return LCF_OK;
}

extern "C" int lcf_grad_clip(const lcf_grad *grads, int count, int p, float max_norm, float *norm, void *ws,
                             size_t ws_bytes, void *stream)
{
    if (!gn_table_ok(grads, count, p, true) || !norm || !ws || !(max_norm >= 0.f)) return LCF_ERR_ARG;
    if (ws_bytes < lcf_grad_norm_workspace_bytes(count)) return LCF_ERR_WORKSPACE;
    const int over = gn_overlap(grads, count);
    if (over) return LCF_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    // Few elements in few chunks of one pair of types: one launch.  (4102 elements in 6 tensors: 11.3 us
    // a call in three launches; a wave walks a chunk by itself, so more than two chunks for each of the
    // 16 waves would take longer than the launches.)
    long long total = 0, chunks = 0;
    bool same = count > 0 && count <= GN_TENSORS;
    for (int i = 0; i < count; ++i) {
        total += grads[i].n;
        chunks += (grads[i].n + GN_CHUNK - 1) / GN_CHUNK;
        same = same && grads[i].dtype == grads[0].dtype && grads[i].out_dtype == grads[0].out_dtype;
    }
    if (same && total > 0 && chunks <= 32 && total <= 65536)
        return gn_launches(grads, count, true, [&](const GnList &l, int dtype, int od) -> int {
            if (dtype == LCF_F32) gn_one_launch<float>(l, od, p, max_norm, norm, st);
            else if (dtype == LCF_BF16) gn_one_launch<lcf_b>(l, od, p, max_norm, norm, st);
            else gn_one_launch<lcf_h>(l, od, p, max_norm, norm, st);
            LCF_CHECK_LAUNCH();
            return LCF_OK;
        });
    double *parts = (double *)((char *)ws + 256);
    int nparts;
    int rc = gn_sums(grads, count, p, parts, (ws_bytes - 256) / sizeof(double), &nparts, st);
    if (rc != LCF_OK) return rc;
    // up to 1024 parts each workgroup of the scaling joins them itself (four loads a thread); more are
    // joined once, by a launch of their own
    GnScale s{parts, nparts, p, max_norm, norm, (const float *)ws};
    if (nparts > 1024 || nparts == 0) {
        gn_final_kernel<<<1, 1024, 0, st>>>(parts, nparts, p, max_norm, norm, (float *)ws);
        LCF_CHECK_LAUNCH();
        s.nparts = 0;
    }
    return gn_launches(grads, count, true, [&](const GnList &l, int dtype, int od) -> int {
        const int chunks = l.chunk0[l.count];
        const int grid = chunks < 2048 ? chunks : 2048;
        if (dtype == LCF_F32) gn_scale_launch<float>(l, od, grid, s, st);
        else if (dtype == LCF_BF16) gn_scale_launch<lcf_b>(l, od, grid, s, st);
        else gn_scale_launch<lcf_h>(l, od, grid, s, st);
        LCF_CHECK_LAUNCH();
        return LCF_OK;
    });
}
