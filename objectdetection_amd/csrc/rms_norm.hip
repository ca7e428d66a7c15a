// rms_norm.hip -- root-mean-square norm of rows with the residual's addition, forward (optionally
// to 8-bit rows with block scales) and backward.
//
//   h = round(x + r),  inv = 1 / sqrt(mean(h^2) + eps),  y = h inv w
//   g = dy w,  dx = inv (g - h inv^2 mean(g h)) + dh,  dw = sum over rows of dy h inv
//
// Bound by memory: a row is read once, held in registers between its sum and its use, and written
// once.  A lane holds CH pieces of eight consecutive columns (16 bytes of a 16-bit type, 32 of
// fp32); LPR lanes share a row, so a wave works on 64 / LPR narrow rows at once, and 16 lanes hold
// exactly one 128-column scale block of the 8-bit form: its largest magnitude is four lane swaps.
// Rows wider than a wave's registers take a workgroup (LPR = 256 or 1024).
// Measured with residual: 16384 x 4096 bf16 forward 95 us (5.6 TB/s), backward 109 us (4.9 TB/s) and
// 8 us for the weight's gradient; 136000 x 64 fp32 28 + 25 + 4 us; 40000 x 256 bf16 to 8-bit rows 16 us
// (4.5 TB/s); one row of 4096 3.5 us, the smallest kernel's duration.
#include "rows.h"

#define RN_MAX_WIDTH 16384
#define RN_PARTS 1024 // workgroups of the backward pass, i.e. partial sums of dweight

template <int LPR> __device__ __forceinline__ float rn_row_sum(float v, float *lds, int &flip)
{
#pragma unroll
    for (int d = (LPR < 64 ? LPR : 64) / 2; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    if constexpr (LPR > 64) {
        // two halves used in turn: one barrier a row is enough
        constexpr int W = LPR / 64;
        float *l = lds + (flip ? W : 0);
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) l[threadIdx.x >> 6] = v;
        __syncthreads();
        v = l[0];
#pragma unroll
        for (int w = 1; w < W; ++w) v += l[w];
    }
    return v;
}

struct RnFwd {
    const void *x, *r, *w;
    void *y, *h;
    float *inv;
    unsigned char *q8, *scale;
    long long ldx, ldr, ldq;
    int rows, width, wcode, lds, fmt;
    float eps;
};

template <typename T, int LPR, int CH>
__global__ void __launch_bounds__(LPR > 256 ? LPR : 256) rn_fwd_kernel(RnFwd p)
{
    constexpr int NT = LPR > 256 ? LPR : 256;
    constexpr int RPB = NT / LPR; // rows of a workgroup
    __shared__ float lds[LPR > 64 ? 2 * LPR / 64 : 1];
    const int lane = threadIdx.x % LPR;
    int flip = 0;
    float w[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * LPR + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[c][i] = 1.f;
        if (p.w && col < p.width) lcf_ld8_code(p.w, p.wcode, col, p.width, w[c]);
    }
    for (long long row0 = (long long)blockIdx.x * RPB; row0 < p.rows; row0 += (long long)gridDim.x * RPB) {
        const long long row = row0 + threadIdx.x / LPR;
        const bool live = row < p.rows; // uniform over the LPR lanes of a row
        const T *x = (const T *)p.x + row * p.ldx;
        const T *r = (const T *)p.r + row * p.ldr;
        float h[CH][8];
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LPR + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = 0.f;
            if (live && col < p.width) {
                lcf_ld8_tail(x, col, p.width, h[c]);
                if (p.r) {
                    float a[8];
                    lcf_ld8_tail(r, col, p.width, a);
                    // the sum is rounded to the rows' type before it is normed: the stored stream
                    // and the norm (and the backward pass, which reads the stream) agree
#pragma unroll
                    for (int i = 0; i < 8; ++i) h[c][i] = lcf_to_f32(lcf_from_f32<T>(h[c][i] + a[i]));
                }
            }
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LPR + lane) * 8;
            if (live && p.h && col < p.width) lcf_st8_tail((T *)p.h + row * p.width, col, p.width, h[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(h[c][i], h[c][i], sum);
        }
        sum = rn_row_sum<LPR>(sum, lds, flip);
        const float inv = 1.f / sqrtf(sum / (float)p.width + p.eps);
        if (live && p.inv && lane == 0) p.inv[row] = inv;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LPR + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = h[c][i] * inv * w[c][i];
            if (live && p.y && col < p.width) lcf_st8_tail((T *)p.y + row * p.width, col, p.width, h[c]);
            if (p.q8) {
                if (col + 8 > p.width) { // an infinite inv makes NaN behind the row
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (col + i >= p.width) h[c][i] = 0.f;
                }
                float top = lcf_f8_top<8>(h[c]);
                if constexpr (LPR >= 16) {
                    top = lcf_max16(top);
                } else {
#pragma unroll
                    for (int d = LPR / 2; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
                }
                const int e = lcf_f8_exponent(top, p.fmt);
                const float s = lcf_exp2i(-e);
                if (live && col < ((p.width + 15) & ~15)) {
                    lcf_u2u b;
                    b.x = lcf_f8_pack4(h[c][0] * s, h[c][1] * s, h[c][2] * s, h[c][3] * s, p.fmt);
                    b.y = lcf_f8_pack4(h[c][4] * s, h[c][5] * s, h[c][6] * s, h[c][7] * s, p.fmt);
                    *reinterpret_cast<lcf_u2u *>(p.q8 + row * p.ldq + col) = b;
                }
                if (live && (col & 127) == 0 && col < p.width) {
                    unsigned char *sr = p.scale + row * p.lds;
                    sr[col >> 7] = (unsigned char)(e + 127);
                    if (col + 128 >= p.width) // zeros up to the next multiple of four
                        for (int k = (col >> 7) + 1; k & 3; ++k) sr[k] = 0;
                }
            }
        }
    }
}

struct RnBwd {
    const void *h, *dy, *dh, *w;
    const float *inv;
    void *dx;
    float *parts; // [gridDim.x][width] or NULL
    long long ldh, lddy, lddh;
    int rows, width, wcode;
};

template <typename T, int LPR, int CH>
__global__ void __launch_bounds__(LPR > 256 ? LPR : 256) rn_bwd_kernel(RnBwd p)
{
    constexpr int NT = LPR > 256 ? LPR : 256;
    constexpr int RPB = NT / LPR;
    // the partial sums of the RPB rows that work side by side meet here at the end
    __shared__ float acc_lds[RPB > 1 ? NT * 8 * CH : 1];
    __shared__ float lds[LPR > 64 ? 2 * LPR / 64 : 1];
    const int lane = threadIdx.x % LPR;
    int flip = 0;
    float w[CH][8], acc[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * LPR + lane) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) { w[c][i] = 1.f; acc[c][i] = 0.f; }
        if (p.w && col < p.width) lcf_ld8_code(p.w, p.wcode, col, p.width, w[c]);
    }
    const float per = 1.f / (float)p.width;
    for (long long row0 = (long long)blockIdx.x * RPB; row0 < p.rows; row0 += (long long)gridDim.x * RPB) {
        const long long row = row0 + threadIdx.x / LPR;
        const bool live = row < p.rows;
        const float inv = live ? p.inv[row] : 0.f;
        float h[CH][8], g[CH][8];
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LPR + lane) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) { h[c][i] = 0.f; g[c][i] = 0.f; }
            if (live && col < p.width) {
                lcf_ld8_tail((const T *)p.h + row * p.ldh, col, p.width, h[c]);
                lcf_ld8_tail((const T *)p.dy + row * p.lddy, col, p.width, g[c]);
            }
        }
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[c][i] = fmaf(g[c][i] * inv, h[c][i], acc[c][i]);
                g[c][i] *= w[c][i];
                sum = fmaf(g[c][i], h[c][i], sum);
            }
        sum = rn_row_sum<LPR>(sum, lds, flip);
        const float k = sum * per * inv * inv;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LPR + lane) * 8;
            if (live && col < p.width) {
                float a[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = 0.f;
                if (p.dh) lcf_ld8_tail((const T *)p.dh + row * p.lddh, col, p.width, a);
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] += inv * fmaf(-h[c][i], k, g[c][i]);
                lcf_st8_tail((T *)p.dx + row * p.width, col, p.width, a);
            }
        }
    }
    if (!p.parts) return;
    float *part = p.parts + (size_t)blockIdx.x * p.width;
    if constexpr (RPB > 1) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                acc_lds[(threadIdx.x / LPR) * (LPR * CH * 8) + (c * LPR + lane) * 8 + i] = acc[c][i];
        __syncthreads();
        for (int col = threadIdx.x; col < p.width; col += NT) {
            float s = 0.f;
            for (int q = 0; q < RPB; ++q) s += acc_lds[q * (LPR * CH * 8) + col];
            part[col] = s;
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LPR + lane) * 8;
            if (col < p.width) lcf_st8_tail(part, col, p.width, acc[c]);
        }
    }
}

// dweight [width] = sum of the workgroups' parts, in 64 bits and in a fixed order.  A workgroup
// takes 16 columns: thread = (part line t / 4, four columns t % 4), 256 lines, so that a thread has
// four loads in flight and no chain of them (one line per wave took 32 us for 1024 parts).
__global__ void __launch_bounds__(1024)
rn_dweight_kernel(const float *__restrict__ parts, int nparts, int width, void *__restrict__ dw, int code)
{
    __shared__ double lds[16][16];
    const int col = blockIdx.x * 16 + (threadIdx.x & 3) * 4, line = threadIdx.x >> 2;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (int i = line; i < nparts; i += 256) {
        const float *q = parts + (size_t)i * width + col;
        if (col + 4 <= width) {
            const lcf_f4u v = *reinterpret_cast<const lcf_f4u *>(q);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += (double)v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < width) s[j] += (double)q[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int d = 32; d >= 4; d >>= 1) s[j] += __shfl_xor(s[j], d, 64);
    }
    if ((threadIdx.x & 63) < 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) lds[threadIdx.x >> 6][(threadIdx.x & 3) * 4 + j] = s[j];
    }
    __syncthreads();
    const int c = blockIdx.x * 16 + threadIdx.x;
    if (threadIdx.x < 16 && c < width) {
        double t = 0.0;
        for (int i = 0; i < 16; ++i) t += lds[i][threadIdx.x];
        if (code == LCF_F32) ((float *)dw)[c] = (float)t;
        else if (code == LCF_BF16) ((lcf_b *)dw)[c] = lcf_from_f32<lcf_b>((float)t);
        else ((lcf_h *)dw)[c] = lcf_from_f32<lcf_h>((float)t);
    }
}

// ---------------------------------------------------------------- host
// Lanes for a row: enough for its width at eight columns a lane, a wave's 64 at most, then more
// pieces a lane up to four, then workgroups.  (Two lanes at least: the 8-bit form's rows end on
// 16 bytes.)  F is called as f(LPR, CH) with integral constants.
template <int V> struct RnInt { static constexpr int value = V; };
template <typename F> static void rn_shape(int width, F f)
{
    if (width <= 16) f(RnInt<2>(), RnInt<1>());
    else if (width <= 32) f(RnInt<4>(), RnInt<1>());
    else if (width <= 64) f(RnInt<8>(), RnInt<1>());
    else if (width <= 128) f(RnInt<16>(), RnInt<1>());
    else if (width <= 256) f(RnInt<32>(), RnInt<1>());
    else if (width <= 512) f(RnInt<64>(), RnInt<1>());
    else if (width <= 1024) f(RnInt<64>(), RnInt<2>());
    else if (width <= 2048) f(RnInt<256>(), RnInt<1>());
    else if (width <= 4096) f(RnInt<256>(), RnInt<2>());
    else if (width <= 8192) f(RnInt<256>(), RnInt<4>());
    else f(RnInt<1024>(), RnInt<2>());
}

static int rn_grid(int rows, int lpr, int cap)
{
    const int rpb = (lpr > 256 ? lpr : 256) / lpr;
    const long long g = ((long long)rows + rpb - 1) / rpb;
    return (int)(g < cap ? g : cap);
}

static int rn_parts(int rows, int width)
{
    int g = 0;
    rn_shape(width, [&](auto lpr, auto) { g = rn_grid(rows, lpr.value, RN_PARTS); });
    return g;
}

extern "C" int lcf_rms_norm_fwd(const void *x, long long ldx, const void *residual, long long ldr, int rows,
                                int width, int dtype, const void *weight, int weight_dtype, float eps, void *y,
                                void *h, float *inv, void *q8, long long ldq, unsigned char *scale, int lds, int fmt,
                                void *stream)
{
    if (rows < 0 || width < 1 || !lcf_is_type(dtype) || (weight && !lcf_is_type(weight_dtype))) return LCF_ERR_ARG;
    if (rows == 0) return LCF_OK;
    if (!x || ldx < width || (residual && ldr < width) || (h && !residual)) return LCF_ERR_ARG;
    if (!(eps >= 0.f)) return LCF_ERR_ARG;
    if (q8 && (!scale || (fmt != LCF_E4M3 && fmt != LCF_E5M2) || ldq < width || (ldq & 15) || ((uintptr_t)q8 & 15) ||
               (lds & 3) || lds < (width + 127) / 128 || ((uintptr_t)scale & 3)))
        return LCF_ERR_ARG;
    if (width > RN_MAX_WIDTH) return LCF_ERR_UNSUPPORTED;
    RnFwd p{x, residual, weight, y, h, inv, (unsigned char *)q8, scale, ldx, ldr, ldq, rows, width, weight_dtype,
            lds, fmt, eps};
    hipStream_t st = (hipStream_t)stream;
    rn_shape(width, [&](auto lpr, auto ch) {
        constexpr int LPR = decltype(lpr)::value, CH = decltype(ch)::value;
        const int grid = rn_grid(rows, LPR, 2048), nt = LPR > 256 ? LPR : 256;
        if (dtype == LCF_F32) rn_fwd_kernel<float, LPR, CH><<<grid, nt, 0, st>>>(p);
        else if (dtype == LCF_BF16) rn_fwd_kernel<lcf_b, LPR, CH><<<grid, nt, 0, st>>>(p);
        else rn_fwd_kernel<lcf_h, LPR, CH><<<grid, nt, 0, st>>>(p);
    });
    LCF_CHECK_LAUNCH();
    return LCF_OK;
}

extern "C" size_t lcf_rms_norm_workspace_bytes(int rows, int width)
{
    if (rows < 1 || width < 1 || width > RN_MAX_WIDTH) return 256;
    return 256 + (size_t)rn_parts(rows, width) * width * sizeof(float);
}

extern "C" int lcf_rms_norm_bwd(const void *h, long long ldh, const void *dy, long long lddy, const void *dh,
                                long long lddh, int rows, int width, int dtype, const void *weight, int weight_dtype,
                                const float *inv, void *dx, void *dweight, void *ws, size_t ws_bytes, void *stream)
{
    if (rows < 0 || width < 1 || !lcf_is_type(dtype) || ((weight || dweight) && !lcf_is_type(weight_dtype)))
        return LCF_ERR_ARG;
    if (rows > 0 && (!h || !dy || !inv || !dx || ldh < width || lddy < width || (dh && lddh < width)))
        return LCF_ERR_ARG;
    if (width > RN_MAX_WIDTH) return LCF_ERR_UNSUPPORTED;
    if (dweight && rows > 0) {
        if (!ws) return LCF_ERR_ARG;
        if (ws_bytes < lcf_rms_norm_workspace_bytes(rows, width)) return LCF_ERR_WORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    RnBwd p{h, dy, dh, weight, inv, dx, dweight ? (float *)ws : nullptr, ldh, lddy, lddh, rows, width, weight_dtype};
    int grid = 0;
    if (rows > 0) {
        rn_shape(width, [&](auto lpr, auto ch) {
            constexpr int LPR = decltype(lpr)::value, CH = decltype(ch)::value;
            const int nt = LPR > 256 ? LPR : 256;
            grid = rn_grid(rows, LPR, RN_PARTS);
            if (dtype == LCF_F32) rn_bwd_kernel<float, LPR, CH><<<grid, nt, 0, st>>>(p);
            else if (dtype == LCF_BF16) rn_bwd_kernel<lcf_b, LPR, CH><<<grid, nt, 0, st>>>(p);
            else rn_bwd_kernel<lcf_h, LPR, CH><<<grid, nt, 0, st>>>(p);
        });
        LCF_CHECK_LAUNCH();
    }
    if (dweight) {
        rn_dweight_kernel<<<(width + 15) / 16, 1024, 0, st>>>((const float *)ws, grid, width, dweight, weight_dtype);
        LCF_CHECK_LAUNCH();
    }
    return LCF_OK;
}

extern "C" int lcf_sum_parts(const float *parts, int count, int n, void *out, int dtype, void *stream)
{
    if (count < 0 || n < 0 || !lcf_is_type(dtype)) return LCF_ERR_ARG;
    if (n > 1 << 25) return LCF_ERR_UNSUPPORTED; // a launch has fewer than 2^32 threads
    if (n == 0) return LCF_OK;
    if ((count > 0 && !parts) || !out) return LCF_ERR_ARG;
    rn_dweight_kernel<<<(n + 15) / 16, 1024, 0, (hipStream_t)stream>>>(parts, count, n, out, dtype);
    LCF_CHECK_LAUNCH();
    return LCF_OK;
}
