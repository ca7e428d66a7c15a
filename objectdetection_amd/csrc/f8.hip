// f8.hip -- matrices in 8-bit form with a power-of-two scale for each block of 128, and their
// product: the row-wise (1x1) layers of a sparse stack on the 8-bit matrix cores, forward, input
// gradient and weight gradient.
//
//   x = q 2^e per block;   out[m][n] = sum_b 2^(ea[m][b] + eb[n][b]) sum_{k in b} qa[m][k] qb[n][k]
//
// Two ways to multiply, by the output's type:
//   16-bit outputs: v_mfma_scale_f32_16x16x128_f8f6f4 sums 128 products of 8-bit values into fp32
//     and takes one E8M0 scale byte per row and 32 columns of either operand: with scale blocks of
//     128 along k one instruction covers exactly one block of both operands, and the scales cost no
//     vector work.  The instruction adds its products in groups of eight along k and keeps 13 bits
//     below the largest of a group (measured; between groups it adds in fp32): an error of at most
//     2^-10 of a group's sum of magnitudes, and 1.5e-5 of the result on random data -- a 16-bit store
//     rounds by up to 2^-8 (bf16) or 2^-11 (fp16) of it.  Not what an fp32 output promises.
//   fp32 outputs: the bytes become bf16 in registers, scaled (v_cvt_scalef32_pk_bf16_*: q 2^e is
//     exact, but below 2^-126, where it is rounded to a multiple of 2^-133, and from 2^128 on, where it is
//     infinite), and v_mfma_f32_16x16x32_bf16 adds the exact products in fp32, at half the peak rate.
#include "rows.h"

typedef int f8_v8 __attribute__((ext_vector_type(8)));
typedef int f8_v4 __attribute__((ext_vector_type(4)));
typedef float f8_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 f8_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 f8_b8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------- quantisation
struct F8Quant {
    const void *x;
    unsigned char *q, *s, *qt, *st;
    float *sums;
    long long ldx, ldq, ldqt;
    int R, C, lds, ldst, fmt, square;
};

// Rows form only: 16 lanes hold one block of 128 columns of one row (eight columns each), its
// largest magnitude is four lane rotations, nothing goes through LDS.  Rows narrower than 128 take as
// many lanes as they need (LPB).  Bound by memory; 136000 x 64 bf16 7 us (3.7 TB/s).
template <typename T, int LPB> __global__ void __launch_bounds__(256) f8_rows_kernel(F8Quant p)
{
    const int nb = (p.C + 127) >> 7;
    const int lane = threadIdx.x % LPB;
    const long long blocks = (long long)p.R * nb;
    const int room = (p.C + 15) & ~15;
    for (long long b0 = (long long)blockIdx.x * (256 / LPB); b0 < blocks; b0 += (long long)gridDim.x * (256 / LPB)) {
        const long long b = b0 + threadIdx.x / LPB;
        const bool live = b < blocks;
        const long long row = live ? b / nb : 0;
        const int kb = live ? (int)(b - row * nb) : 0;
        const int col = kb * 128 + lane * 8;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        if (live && col < p.C) lcf_ld8_tail((const T *)p.x + row * p.ldx, col, p.C, v);
        float top = lcf_f8_top<8>(v);
        if constexpr (LPB == 16) {
            top = lcf_max16(top);
        } else {
#pragma unroll
            for (int d = LPB / 2; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        }
        const int e = lcf_f8_exponent(top, p.fmt);
        const float s = lcf_exp2i(-e);
        if (live && col < room) {
            lcf_u2u o;
            o.x = lcf_f8_pack4(v[0] * s, v[1] * s, v[2] * s, v[3] * s, p.fmt);
            o.y = lcf_f8_pack4(v[4] * s, v[5] * s, v[6] * s, v[7] * s, p.fmt);
            *reinterpret_cast<lcf_u2u *>(p.q + row * p.ldq + col) = o;
        }
        if (live && lane == 0) {
            unsigned char *sr = p.s + row * p.lds;
            sr[kb] = (unsigned char)(e + 127);
            if (kb == nb - 1)
                for (int k = nb; k & 3; ++k) sr[k] = 0;
        }
    }
}

// Any of the forms from one reading: a workgroup takes 128 x 128 elements.  Thread (rl, cl) holds
// rows 8 rl .. 8 rl + 7 and columns 8 cl .. 8 cl + 7: a row's magnitudes meet over the 16 lanes of
// equal rl (rotations on the vector unit), a column's over the thread's own rows, the wave's four row
// lanes and, through LDS, the four waves.  Eight bytes of a transposed row are one thread's own;
// they are turned in LDS, four at a time, and leave as 16-byte pieces of whole rows.  (A thread with
// every 16th row wrote single bytes to two of the 64 banks: 84 us for 136000 x 256 bf16, both forms;
// the columns form alone now takes 27 us, 3.9 TB/s.)
#define F8_TP 132 // bytes of a transposed row in LDS: eight rows further on start 32 bytes further on
template <typename T> __global__ void __launch_bounds__(256) f8_tile_kernel(F8Quant p)
{
    __shared__ float colmax[4][128];
    __shared__ unsigned turn[128 * F8_TP / 4];
    const int tid = threadIdx.x, cl = tid & 15, rl = tid >> 4, wave = tid >> 6;
    const int r0 = blockIdx.y * 128, c0 = blockIdx.x * 128;
    const int col = c0 + cl * 8;
    float v[8][8], rm[8], cm[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = r0 + rl * 8 + i;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        if (row < p.R && col < p.C) lcf_ld8_tail((const T *)p.x + row * p.ldx, col, p.C, v[i]);
    }
    if (p.sums) { // the columns' sums over these 128 rows
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i][j];
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            if ((tid & 63) < 16) colmax[wave][cl * 8 + j] = s;
        }
        __syncthreads();
        if (tid < 128 && c0 + tid < p.C)
            p.sums[(long long)blockIdx.y * p.C + c0 + tid] =
                (colmax[0][tid] + colmax[1][tid]) + (colmax[2][tid] + colmax[3][tid]);
        __syncthreads();
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        rm[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) rm[i] = fmaxf(rm[i], __builtin_fabsf(v[i][j]));
        top = fmaxf(top, rm[i]);
    }
    if (__builtin_expect(__any(top > 3.402823466e38f), 0)) { // infinities become NaN
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            rm[i] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (__builtin_fabsf(v[i][j]) > 3.402823466e38f) v[i][j] = __uint_as_float(0x7FC00000u);
                rm[i] = fmaxf(rm[i], __builtin_fabsf(v[i][j]));
            }
        }
    }
    int esq = 0;
    if (p.qt || p.square) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            cm[j] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) cm[j] = fmaxf(cm[j], __builtin_fabsf(v[i][j]));
            cm[j] = fmaxf(cm[j], __shfl_xor(cm[j], 16, 64));
            cm[j] = fmaxf(cm[j], __shfl_xor(cm[j], 32, 64));
        }
        if ((tid & 63) < 16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) colmax[wave][cl * 8 + j] = cm[j];
        }
        __syncthreads();
        float all = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int w = 0; w < 4; ++w) cm[j] = fmaxf(cm[j], colmax[w][cl * 8 + j]);
            all = fmaxf(all, cm[j]);
        }
        esq = lcf_f8_exponent(lcf_max16(all), p.fmt);
    }
    if (p.q) {
        const int room = (p.C + 15) & ~15;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = r0 + rl * 8 + i;
            const int e = p.square ? esq : lcf_f8_exponent(lcf_max16(rm[i]), p.fmt);
            const float s = lcf_exp2i(-e);
            if (row < p.R && col < room) {
                lcf_u2u o;
                o.x = lcf_f8_pack4(v[i][0] * s, v[i][1] * s, v[i][2] * s, v[i][3] * s, p.fmt);
                o.y = lcf_f8_pack4(v[i][4] * s, v[i][5] * s, v[i][6] * s, v[i][7] * s, p.fmt);
                *reinterpret_cast<lcf_u2u *>(p.q + row * p.ldq + col) = o;
            }
            if (cl == 0 && (p.square ? (i == 0 && rl == 0) : row < p.R)) {
                unsigned char *sr = p.s + (long long)(p.square ? blockIdx.y : row) * p.lds;
                sr[blockIdx.x] = (unsigned char)(e + 127);
                if (blockIdx.x == gridDim.x - 1)
                    for (int k = gridDim.x; k & 3; ++k) sr[k] = 0;
            }
        }
    }
    if (p.qt) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = p.square ? esq : lcf_f8_exponent(cm[j], p.fmt);
            const float s = lcf_exp2i(-e);
            unsigned *t = turn + (cl * 8 + j) * (F8_TP / 4) + rl * 2;
            t[0] = lcf_f8_pack4(v[0][j] * s, v[1][j] * s, v[2][j] * s, v[3][j] * s, p.fmt);
            t[1] = lcf_f8_pack4(v[4][j] * s, v[5][j] * s, v[6][j] * s, v[7][j] * s, p.fmt);
            if (rl == 0 && (p.square ? (cl == 0 && j == 0) : col + j < p.C)) {
                unsigned char *sr = p.st + (long long)(p.square ? blockIdx.x : col + j) * p.ldst;
                sr[blockIdx.y] = (unsigned char)(e + 127);
                if (blockIdx.y == gridDim.y - 1)
                    for (int k = gridDim.y; k & 3; ++k) sr[k] = 0;
            }
        }
        __syncthreads();
        const int room = (p.R + 15) & ~15;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = (tid >> 3) + k * 32, part = (tid & 7) * 16;
            const unsigned *t = turn + c * (F8_TP / 4) + part / 4;
            if (c0 + c < p.C && r0 + part < room)
                *reinterpret_cast<uint4 *>(p.qt + (long long)(c0 + c) * p.ldqt + r0 + part) =
                    make_uint4(t[0], t[1], t[2], t[3]);
        }
    }
}

template <typename T> static void f8_quant_launch(const F8Quant &p, hipStream_t st)
{
    if (p.q && !p.qt && !p.square && !p.sums) {
        const long long blocks = (long long)p.R * ((p.C + 127) / 128);
        auto grid = [&](int lpb) {
            const long long g = (blocks * lpb + 255) / 256;
            return (int)(g < 4096 ? g : 4096);
        };
        if (p.C <= 16) f8_rows_kernel<T, 2><<<grid(2), 256, 0, st>>>(p);
        else if (p.C <= 32) f8_rows_kernel<T, 4><<<grid(4), 256, 0, st>>>(p);
        else if (p.C <= 64) f8_rows_kernel<T, 8><<<grid(8), 256, 0, st>>>(p);
        else f8_rows_kernel<T, 16><<<grid(16), 256, 0, st>>>(p);
    } else {
        f8_tile_kernel<T><<<dim3((p.C + 127) / 128, (p.R + 127) / 128), 256, 0, st>>>(p);
    }
}

#define F8_MOST 0x7FFFFF00 // rows or columns: the last tile's end is an int too

static bool f8_form_ok(const void *q, long long ld, const unsigned char *s, int lds, int C)
{
    return q && s && !((uintptr_t)q & 15) && !((uintptr_t)s & 3) && !(ld & 15) && !(lds & 3) && ld >= C &&
           lds >= (C + 127) / 128;
}

extern "C" int lcf_f8_quant(const void *x, long long ldx, int R, int C, int dtype, int fmt, int square, void *q,
                            long long ldq, unsigned char *s, int lds, void *qt, long long ldqt, unsigned char *st,
                            int ldst, float *sums, void *stream)
{
    if (R < 0 || C < 0 || !lcf_is_type(dtype) || (fmt != LCF_E4M3 && fmt != LCF_E5M2)) return LCF_ERR_ARG;
    if (R == 0 || C == 0) return LCF_OK;
    if (!x || ldx < C || (!q && !qt && !sums)) return LCF_ERR_ARG;
    if (q && !f8_form_ok(q, ldq, s, lds, C)) return LCF_ERR_ARG;
    if (qt && !f8_form_ok(qt, ldqt, st, ldst, R)) return LCF_ERR_ARG;
    // columns are counted in 32 bits up to the end of a block, and the grid's second dimension counts
    // 128-row tiles
    if (C > F8_MOST || ((qt || square || sums) && R > 65535 * 128)) return LCF_ERR_UNSUPPORTED;
    F8Quant p{x, (unsigned char *)q, s, (unsigned char *)qt, st, sums, ldx, ldq, ldqt, R, C, lds, ldst, fmt, square};
    if (dtype == LCF_F32) f8_quant_launch<float>(p, (hipStream_t)stream);
    else if (dtype == LCF_BF16) f8_quant_launch<lcf_b>(p, (hipStream_t)stream);
    else f8_quant_launch<lcf_h>(p, (hipStream_t)stream);
    LCF_CHECK_LAUNCH();
    return LCF_OK;
}

// ---------------------------------------------------------------- product
struct F8Gemm {
    const unsigned char *a, *sa, *b, *sb;
    const float *scale, *shift;
    void *out;
    float *ws; // parts [splits][M][N] fp32, or NULL: the kernel writes `out`
    long long lda, ldb, ldo;
    int ldsa, ldsb, b_shift; // b_shift: 7 = one scale row for 128 rows of b
    int M, N, K, relu, code;
    int tiles_m, tiles_n, splits, ksteps; // ksteps: 128-column steps of one split
};

// `count` (at most W) outputs of row m from column n on: W consecutive columns held by one lane
template <int W> __device__ __forceinline__ void f8_store(const F8Gemm &p, long long m, int n, const float *v, int count)
{
    float s[W];
#pragma unroll
    for (int i = 0; i < W; ++i) s[i] = v[i];
    if (p.scale) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i < count) s[i] *= p.scale[n + i];
    }
    if (p.shift) {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i < count) s[i] += p.shift[n + i];
    }
    if (p.relu) {
#pragma unroll
        for (int i = 0; i < W; ++i) s[i] = s[i] < 0.f ? 0.f : s[i]; // NaN stays
    }
    auto put = [&](auto *row) {
        using T = typename std::remove_pointer<decltype(row)>::type;
        if (count >= W) {
            if constexpr (W == 8) lcf_st8(row, s);
            else *reinterpret_cast<lcf_f4u *>(row) = (lcf_f4u){s[0], s[1], s[2], s[3]};
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (i < count) row[i] = lcf_from_f32<T>(s[i]);
        }
    };
    if constexpr (W == 4) put((float *)p.out + m * p.ldo + n);
    else if (p.code == LCF_BF16) put((lcf_b *)p.out + m * p.ldo + n);
    else put((lcf_h *)p.out + m * p.ldo + n);
}

// bytes [col, col + 16) of a row of K: those behind the row's end become zeros (no branches: masks)
__device__ __forceinline__ void f8_cut(int *w, int col, int K)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = min(max(K - (col + 4 * i), 0), 4);
        w[i] &= left == 4 ? -1 : (1 << (8 * left)) - 1;
    }
}

// 16 bytes a lane from a buffer straight to LDS, lane after lane behind `to` (the host's pass does not
// know the builtin at this width)
__device__ __forceinline__ void f8_lds16(__amdgpu_buffer_rsrc_t from, unsigned char *to, int off)
{
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 16, off, 0, 0, 0);
#endif
}

// Keeps the four sums of a piece where they are computed.  A matrix instruction reads its operands
// from all 64 lanes whatever the execution mask says; the compiler moves one that only a guarded
// store uses into the guarded block, and with it the vector instructions that make its operands,
// which then run in the storing lanes alone (seen: outputs of a tile that N ends in were wrong).
// The waits cover the instruction's own latency (at most 19 states before its result may be read).
__device__ __forceinline__ void f8_pin(f8_f4 (&a)[4])
{
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]));
#endif
}

template <bool V> struct F8Bool { static constexpr bool value = V; };

// Which of a wave's 64 columns n the row i of its piece t of b stands for.  The instruction's first
// operand is b, its second a, so lane (r16, g) holds rows i = 4 g + r (r = 0..3) of every piece for
// one row m of a.  fp32 outputs: n = 16 t + i, four columns (16 bytes) in a piece's four registers.
// 16-bit outputs: n = 32 (t / 2) + 8 g + 4 (t % 2) + r, eight columns (16 bytes) over two pieces.
// Either way the four lanes of a row store 64 consecutive bytes at once.
template <bool WIDE> __device__ __forceinline__ int f8_column(int t, int i)
{
    return WIDE ? 16 * t + i : 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
}

// a wave's 64 columns of row m, from column n0 on, out of its four pieces' sums
template <bool WIDE> __device__ __forceinline__ void f8_put(const F8Gemm &p, float *ws, long long m, int n0, int g,
                                                            const f8_f4 *acc)
{
    constexpr int W = WIDE ? 4 : 8;
#pragma unroll
    for (int q = 0; q < 16 / W; ++q) {
        const int n = n0 + (WIDE ? 16 * q + 4 * g : 32 * q + 8 * g);
        float v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = acc[WIDE ? q : 2 * q + (i >> 2)][i & 3];
        if (ws) {
            float *o = ws + m * p.N + n;
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                if (n + i + 4 <= p.N) {
                    *reinterpret_cast<lcf_f4u *>(o + i) = (lcf_f4u){v[i], v[i + 1], v[i + 2], v[i + 3]};
                } else {
#pragma unroll
                    for (int k = i; k < i + 4; ++k)
                        if (n + k < p.N) o[k] = v[k];
                }
            }
        } else if (n < p.N) {
            f8_store<W>(p, m, n, v, p.N - n);
        }
    }
}

// eight bytes of a row as bf16, times the block's scale
template <int F> __device__ __forceinline__ f8_b8 f8_to_bf16(int lo, int hi, float scale)
{
    f8_b2 q[4];
    if constexpr (F == LCF_E4M3) {
        q[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
        q[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
        q[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
        q[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    } else {
        q[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, false);
        q[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, scale, true);
        q[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, false);
        q[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, scale, true);
    }
    f8_b8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = q[i >> 1][i & 1];
    return v;
}

// A workgroup of WM x WN waves makes BM x BN outputs, a wave 16 MT x 64 of them.
// Bound by the matrix cores at 256 x 256 (8192 x 4096 x 8192 to bf16: 226 us, 2437 TFLOP/s): a wave's
// 128 x 64 takes 24 KB out of LDS for 1024 cycles of products, three quarters of what LDS gives, where
// 64 x 64 (492 us) took all of it.  The smaller tiles are for few tiles and are bound by a step's latency.
// LDS holds 128 bytes of k for each row of a and b, twice: the next step's bytes go from memory
// straight into LDS (16 bytes a lane, no registers) while this one multiplies.  A 16-byte piece c of
// row r sits at place c ^ swz(r), so that the lanes that read together read different banks; a
// memory-to-LDS load writes its 64 lanes' pieces side by side, so it is the lanes' addresses in
// memory that are dealt.  Rows past the end are read as the last row, and what lies behind K is cut
// from the registers in the last step.
template <int FA, int FB, bool WIDE, int WM, int WN, int MT>
__global__ void __launch_bounds__(WM *WN * 64) f8_gemm_kernel(F8Gemm p)
{
    constexpr int BM = WM * MT * 16, BN = WN * 64, NT = WM * WN * 64;
    constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT; // 16-byte pieces a thread loads for a step
    extern __shared__ __align__(16) unsigned char smem[];
    // a: [2][BM][128], b: [2][BN][128], scale words: [2][BM + BN]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r16 = lane & 15, g = lane >> 4;
    // workgroups go round-robin to the 8 XCDs: XCD x takes the x-th eighth of the tiles, in groups
    // of 8 tile rows, so that the tiles in flight on it share rows of a and b in its L2
    // (the splits of a long sum come one after the other)
    const int tiles = p.tiles_m * p.tiles_n, per = (tiles * p.splits + 7) >> 3;
    const int all = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || all >= tiles * p.splits) return;
    const int split = all / tiles, lin = all - split * tiles;
    const int band = lin / (8 * p.tiles_n), first = band * 8;
    const int high = min(8, p.tiles_m - first), in = lin - band * 8 * p.tiles_n;
    const int tm = first + in % high, tn = in / high;
    const int m0 = tm * BM, n0 = tn * BN;
    const int wm = (wave % WM) * (MT * 16), wn = (wave / WM) * 64;
    const int step0 = split * p.ksteps;
    const int step1 = min((p.K + 127) >> 7, step0 + p.ksteps);

    auto swz_a = [](int r) { return r & 7; };
    // a fragment's rows of b are f8_column(t, 0..15): their bits 0..2, or 0, 1 and 3, tell eight apart
    auto swz_b = [](int r) { return WIDE ? r & 7 : (r & 3) | ((r >> 1) & 4); };

    // this thread's pieces, as offsets from the tile's first row (ld <= 2^22: 32 bits) into buffers
    // that end with the last row's last piece: past it a load brings zeros and touches nothing
    const int rows_a = min(BM, p.M - m0), rows_b = min(BN, p.N - n0), room = (p.K + 15) & ~15;
    const __amdgpu_buffer_rsrc_t abuf = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<unsigned char *>(p.a + (long long)m0 * p.lda), 0, (rows_a - 1) * (int)p.lda + room, 0x00020000);
    const __amdgpu_buffer_rsrc_t bbuf = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<unsigned char *>(p.b + (long long)n0 * p.ldb), 0, (rows_b - 1) * (int)p.ldb + room, 0x00020000);
    int aoff[LA], boff[LB];
    static_assert((NT >> 3) % 32 == 0, "a thread's pieces have one column");
    {
        const int r = tid >> 3;
#pragma unroll
        for (int i = 0; i < LA; ++i)
            aoff[i] = min(i * (NT >> 3) + r, rows_a - 1) * (int)p.lda + (((tid & 7) ^ swz_a(r)) + step0 * 8) * 16;
#pragma unroll
        for (int i = 0; i < LB; ++i)
            boff[i] = min(i * (NT >> 3) + r, rows_b - 1) * (int)p.ldb + (((tid & 7) ^ swz_b(r)) + step0 * 8) * 16;
    }
    // the next step in turn: 128 bytes further each time
    auto load = [&](int buf) {
        unsigned char *la = smem + buf * BM * 128 + wave * 1024, *lb = smem + 2 * BM * 128 + buf * BN * 128 + wave * 1024;
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            f8_lds16(abuf, la + i * NT * 16, aoff[i]);
            aoff[i] += 128;
        }
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            f8_lds16(bbuf, lb + i * NT * 16, boff[i]);
            boff[i] += 128;
        }
    };

    f8_f4 acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = (f8_f4){0.f, 0.f, 0.f, 0.f};
    const int nb = f8_column<WIDE>(0, r16); // this lane's row of b in piece 0 of the wave
    // scale words, four steps to a word, go through LDS as well: one word a thread for each row of a and
    // b, twice
    static_assert(NT >= BM + BN && (BM + BN) % 64 == 0, "a thread for each row's scales, in whole waves");
    unsigned *ls = (unsigned *)(smem + 2 * (BM + BN) * 128);
    const unsigned char *srow =
        tid < BM ? p.sa + (long long)min(m0 + tid, p.M - 1) * p.ldsa
                 : p.sb + (long long)(min(n0 + tid - BM, p.N - 1) >> p.b_shift) * p.ldsb;
    auto load_scales = [&](int word) {
        if (NT > BM + BN && wave >= (BM + BN) / 64) return;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(srow + word * 4),
                                         (__attribute__((address_space(3))) void *)(ls + (word & 1) * (BM + BN) + wave * 64),
                                         4, 0, 0);
    };
    unsigned xa[MT], xb[4];
    auto scales = [&](int step) {
        const unsigned *l = ls + ((step >> 2) & 1) * (BM + BN);
        const int sh = (step & 3) * 8;
#pragma unroll
        for (int i = 0; i < MT; ++i) xa[i] = l[wm + i * 16 + r16] >> sh;
#pragma unroll
        for (int t = 0; t < 4; ++t) xb[t] = l[BM + wn + f8_column<WIDE>(t, r16)] >> sh;
    };

    auto multiply = [&](int buf, int step, auto tail) {
        const unsigned char *la = smem + buf * BM * 128 + (wm + r16) * 128;
        const unsigned char *lb = smem + 2 * BM * 128 + buf * BN * 128 + (wn + nb) * 128;
        const int sa = swz_a(r16), sb0 = swz_b(wn + nb);
        auto frag = [&](const unsigned char *row, int s) -> f8_v8 {
            const f8_v4 lo = *reinterpret_cast<const f8_v4 *>(row + ((g ^ s) * 16));
            const f8_v4 hi = *reinterpret_cast<const f8_v4 *>(row + (((g + 4) ^ s) * 16));
            int w[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if constexpr (decltype(tail)::value) {
                f8_cut(w, step * 128 + g * 16, p.K);
                f8_cut(w + 4, step * 128 + g * 16 + 64, p.K);
            }
            f8_v8 v;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w[i];
            return v;
        };
        if constexpr (!WIDE) {
            f8_v8 fb[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) fb[t] = frag(lb + f8_column<WIDE>(t, 0) * 128, sb0);
            // the next piece of a is on its way while this one multiplies; the scheduler is kept from
            // reading all of them first, which would cost more registers than there are
            f8_v8 fa = frag(la, sa);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                f8_v8 next = fa;
                if (i + 1 < MT) next = frag(la + (i + 1) * 2048, sa);
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[t], fa, acc[i][t], FB, FA, 0,
                                                                                 (int)xb[t], 0, (int)xa[i]);
                fa = next;
                if constexpr (!decltype(tail)::value) __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            f8_b8 wb[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f8_v8 fb = frag(lb + f8_column<WIDE>(t, 0) * 128, sb0);
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    wb[t][s] = f8_to_bf16<FB>(fb[2 * s], fb[2 * s + 1], lcf_exp2i((int)(xb[t] & 255) - 127));
            }
            f8_v8 fa = frag(la, sa);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                f8_v8 next = fa;
                if (i + 1 < MT) next = frag(la + (i + 1) * 2048, sa);
                const float ea = lcf_exp2i((int)(xa[i] & 255) - 127);
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const f8_b8 wa = f8_to_bf16<FA>(fa[2 * s], fa[2 * s + 1], ea);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[t][s], wa, acc[i][t], 0, 0, 0);
                }
                fa = next;
                if constexpr (!decltype(tail)::value) __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) xa[i] >>= 8;
#pragma unroll
        for (int t = 0; t < 4; ++t) xb[t] >>= 8;
    };

    if (step0 < step1) {
        load_scales(step0 >> 2);
        load(0);
        __syncthreads();
        const int whole = min(step1, p.K >> 7); // steps that K does not end in
        int step = step0;
        // nothing but the barrier may follow the products in the loop: behind a branch the compiler
        // would move them past the barrier, and the loads would have nothing to hide behind
#pragma clang loop unroll(disable)
        for (; step < whole; ++step) {
            const int buf = (step - step0) & 1;
            if (step + 1 < step1) {
                if (((step + 1) & 3) == 0) load_scales((step + 1) >> 2);
                load(buf ^ 1);
            }
            if (step == step0 || (step & 3) == 0) scales(step);
            multiply(buf, step, F8Bool<false>());
            __syncthreads();
        }
        if (step < step1 && (step == step0 || (step & 3) == 0)) scales(step);
        if (step < step1) multiply((step - step0) & 1, step, F8Bool<true>());
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) f8_pin(acc[i]);
    float *ws = p.ws ? p.ws + (long long)split * p.M * p.N : nullptr;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long long m = m0 + wm + i * 16 + r16;
        if (m < p.M) f8_put<WIDE>(p, ws, m, n0 + wn, g, acc[i]);
    }
}

// Thin layers (K <= 512, N <= 256) over many rows: bound by reading a and writing out.  A wave keeps
// its 64 columns of b (all of K: 32 KS registers, 64 KS widened) and walks down the rows, 16 at a
// time, straight from memory to the matrix core and back: nothing goes through LDS and nothing
// waits for another wave.  The waves of a workgroup that share rows read them through the same L1.
// The next 16 rows are asked for before this one's are used, and no load or store of the loop stands
// behind a branch: memory operations are counted in order, and one that may not have happened makes
// the wait for the rows a wait for the stores in front of them as well (5 us a turn).  What lies
// past the last row, past K or past N is an offset beyond its buffer's end instead: such a load
// brings zeros and such a store is dropped, neither touches memory.  Scale and shift wait in LDS.
// T: the rows are fp32 / bf16 / fp16 and brought into 8-bit form in registers on the way (bit for
// bit what f8_rows_kernel stores: a row's 128 columns are in the four lanes of equal r16), which
// saves writing and reading them; T = unsigned char: they are in that form already.
// Measured, 136000 rows of bf16: 64 -> 256 columns 23 us alone (3.8 TB/s; the same product in the
// library's bf16 27 us), 256 -> 64 23 us (3.8 TB/s).
template <int FA, int FB, bool WIDE, int KS, typename T>
__global__ void __launch_bounds__(256) f8_stream_kernel(F8Gemm p, int wn_shift)
{
    constexpr int E = sizeof(T), P = 2 * E; // 16-byte pieces of a row for one step of 128 columns, a lane
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int n0 = (wave & ((1 << wn_shift) - 1)) * 64;
    __shared__ __align__(16) float affine[2][256];
    {
        const int n = threadIdx.x;
        affine[0][n] = p.scale && n < p.N ? p.scale[n] : 1.f;
        affine[1][n] = p.shift && n < p.N ? p.shift[n] : 0.f;
    }
    __syncthreads();
    if (n0 >= p.N) return;
    const int rows = 16 << (2 - wn_shift), wm = (wave >> wn_shift) * 16; // rows a workgroup takes at a time

    // piece i of step k holds elements col .. col + 16 / E of the row: the lane's 16 columns from
    // 16 g on, then the 16 from 64 + 16 g on
    struct Rows {
        f8_v4 v[KS * P];
        unsigned s;
    };
    int off[KS * P];
    const int room = E == 1 ? (p.K + 15) & ~15 : p.K;
#pragma unroll
    for (int i = 0; i < KS * P; ++i) {
        const int h = i % P, col = (i / P) * 128 + (h / (P / 2)) * 64 + g * 16 + (h % (P / 2)) * (16 / E);
        off[i] = col < p.K ? (r16 * (int)p.lda + col) * E : (int)0x80000000;
    }
    auto ask = [&](long long m0, Rows &x) {
        const int left = (int)(m0 < p.M ? (p.M - m0 < 16 ? p.M - m0 : 16) : 0);
        const __amdgpu_buffer_rsrc_t buf = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<unsigned char *>(p.a + (left ? m0 * p.lda * E : 0)), 0,
            left ? ((left - 1) * (int)p.lda + room) * E : 0, 0x00020000);
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < KS * P; ++i) {
            const u4 v = __builtin_amdgcn_raw_buffer_load_b128(buf, off[i], 0, 0);
            x.v[i] = (f8_v4){(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
        }
        if constexpr (E == 1) {
            const long long m = m0 + r16 < p.M ? m0 + r16 : p.M - 1;
            x.s = *(const unsigned *)(p.sa + m * p.ldsa);
        }
    };
    const long long stride = (long long)gridDim.x * rows;
    long long m0 = (long long)blockIdx.x * rows + wm;
    // two sets of registers used in turn: copying one to the other would wait for it
    Rows x, y;
    ask(m0, x);

    // Scale bytes of the blocks that there are.  Four steps serve three blocks too: the fourth is zeros,
    // and what follows a row's scales is the caller's, 255 (no number) among it; made 0 it is 2^-127.
    const unsigned scales = KS == 4 && p.K <= 384 ? 0xFFFFFFu : 0xFFFFFFFFu;
    f8_v8 fb[KS][4];
    unsigned xb[4];
    {
        // all of b at once, then the cuts: one round trip
        const __amdgpu_buffer_rsrc_t buf = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<unsigned char *>(p.b + (long long)n0 * p.ldb), 0,
            (min(64, p.N - n0) - 1) * (int)p.ldb + ((p.K + 15) & ~15), 0x00020000);
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int n = min(f8_column<WIDE>(t, r16), p.N - 1 - n0);
            xb[t] = *(const unsigned *)(p.sb + (long long)((n0 + n) >> p.b_shift) * p.ldsb) & scales;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = k * 128 + g * 16 + h * 64;
                    const u4 v = __builtin_amdgcn_raw_buffer_load_b128(
                        buf, col < p.K ? n * (int)p.ldb + col : (int)0x80000000, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) fb[k][t][h * 4 + i] = (int)v[i];
                }
        }
        if (p.K & 15) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        int w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = fb[k][t][h * 4 + i];
                        f8_cut(w, k * 128 + g * 16 + h * 64, p.K);
#pragma unroll
                        for (int i = 0; i < 4; ++i) fb[k][t][h * 4 + i] = w[i];
                    }
        }
    }
    f8_b8 wb[WIDE ? KS : 1][4][4];
    if constexpr (WIDE) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    wb[k][t][q] = f8_to_bf16<FB>(fb[k][t][2 * q], fb[k][t][2 * q + 1],
                                                 lcf_exp2i((int)((xb[t] >> (8 * k)) & 255) - 127));
    }

    auto use = [&](long long m0, const Rows &x) {
        int fa[KS][8];
        unsigned xa = 0;
        if constexpr (E == 1) {
            xa = x.s & scales;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
#pragma unroll
                for (int i = 0; i < 8; ++i) fa[k][i] = x.v[k * 2 + (i >> 2)][i & 3];
                if (p.K & 15) {
                    f8_cut(fa[k], k * 128 + g * 16, p.K);
                    f8_cut(fa[k] + 4, k * 128 + g * 16 + 64, p.K);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int w = x.v[k * P + i * E / 16][(i * E / 4) & 3];
                    if constexpr (E == 4) v[i] = __int_as_float(w);
                    else v[i] = lcf_to_f32(__builtin_bit_cast(T, (unsigned short)((unsigned)w >> (16 * (i & 1)))));
                }
                float top = lcf_f8_top<32>(v);
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const int e = lcf_f8_exponent(top, FA);
                const float sc = lcf_exp2i(-e);
                xa |= (unsigned)(e + 127) << (8 * k);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    fa[k][i] = (int)lcf_f8_pack4(v[4 * i] * sc, v[4 * i + 1] * sc, v[4 * i + 2] * sc, v[4 * i + 3] * sc,
                                                 FA);
            }
        }
        f8_f4 acc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = (f8_f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if constexpr (WIDE) {
                const float ea = lcf_exp2i((int)((xa >> (8 * k)) & 255) - 127);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f8_b8 wa = f8_to_bf16<FA>(fa[k][2 * q], fa[k][2 * q + 1], ea);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[k][t][q], wa, acc[t], 0, 0, 0);
                }
            } else {
                f8_v8 a;
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = fa[k][i];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        fb[k][t], a, acc[t], FB, FA, 0, (int)(xb[t] >> (8 * k)), 0, (int)(xa >> (8 * k)));
            }
        }
        f8_pin(acc);
        constexpr int W = WIDE ? 4 : 8, EO = WIDE ? 4 : 2;
        const int left = p.M - m0 < 16 ? (int)(p.M - m0) : 16;
        const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(
            (char *)p.out + m0 * p.ldo * EO, 0, ((left - 1) * (int)p.ldo + p.N) * EO, 0x00020000);
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
        u4 o[16 / W];
#pragma unroll
        for (int q = 0; q < 16 / W; ++q) {
            const int n = n0 + (WIDE ? 16 * q + 4 * g : 32 * q + 8 * g);
            float v[W];
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = acc[WIDE ? q : 2 * q + (i >> 2)][i & 3];
            if (p.scale) {
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] *= affine[0][n + i];
            }
            if (p.shift) {
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] += affine[1][n + i];
            }
            if (p.relu) {
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] = v[i] < 0.f ? 0.f : v[i]; // NaN stays
            }
            if constexpr (WIDE) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[q][i] = __float_as_uint(v[i]);
            } else if (p.code == LCF_BF16) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[q][i] = __builtin_bit_cast(unsigned short, lcf_from_f32<lcf_b>(v[2 * i])) |
                              (unsigned)__builtin_bit_cast(unsigned short, lcf_from_f32<lcf_b>(v[2 * i + 1])) << 16;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[q][i] = __builtin_bit_cast(unsigned short, lcf_from_f32<lcf_h>(v[2 * i])) |
                              (unsigned)__builtin_bit_cast(unsigned short, lcf_from_f32<lcf_h>(v[2 * i + 1])) << 16;
            }
        }
        // Two pieces of a row are one 128-byte line, and a row's four lanes would store half of it at a
        // time (1.3 times the bytes then reached memory).  Lanes eight apart trade a piece, so that eight
        // lanes store whole lines of eight rows.  N is a multiple of W: a piece is inside or outside as a
        // whole.  Stored past the caches (nt): the output is as large as they are (a training step's three
        // products over 136000 rows of 64 and 256 columns: 125 -> 121 us; the same for the rows' loads
        // made it 143).
        const bool low = r16 < 8;
        const int row = r16 & 7;
#pragma unroll
        for (int q = 0; q < 16 / W; q += 2) {
            u4 first, second;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned mine = low ? o[q][i] : o[q + 1][i];
                const unsigned got = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(low ? o[q + 1][i] : o[q][i]), 0x128,
                                                                           0xF, 0xF, false);
                first[i] = low ? mine : got;
                second[i] = low ? got : mine;
            }
            const int n = n0 + (WIDE ? 16 * (q + !low) + 4 * g : 32 * (q + !low) + 8 * g);
            const int at = (row * (int)p.ldo + n) * EO;
            __builtin_amdgcn_raw_buffer_store_b128(first, to, n < p.N && row < left ? at : (int)0x80000000, 0, 2);
            __builtin_amdgcn_raw_buffer_store_b128(
                second, to, n < p.N && row + 8 < left ? at + 8 * (int)p.ldo * EO : (int)0x80000000, 0, 2);
        }
    };
    // everything asked for so far is here: the loop's waits then count its own operations only
    __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0)
    while (m0 < p.M) {
        ask(m0 + stride, y);
        use(m0, x);
        m0 += stride;
        if (m0 >= p.M) break;
        ask(m0 + stride, x);
        use(m0, y);
        m0 += stride;
    }
}

// A few rows (M <= 64, unless their sums are long and split: f8_long): bound by reading b once.  A
// workgroup takes 16 columns of the output, its waves take turns of 512 bytes along k (four steps, one scale word): everything of a turn is asked for at
// once, 8 KB of b a wave, straight into registers.  The waves' sums meet in LDS in a fixed order.
// (Tiles of 128 rows leave a compute unit one 16 KB step in flight: 11.6 us and a join of 3.9 us at
// 8 x 8192 x 4096; now 12.4 us, 2.7 TB/s with the launch and the first latency in it.)
template <int FA, int FB, bool WIDE, int MT> // (16 waves leave a wave 128 registers, which do for MT = 1)
__global__ void __launch_bounds__(MT == 1 ? 1024 : 512) f8_few_kernel(F8Gemm p)
{
    extern __shared__ __align__(16) float few_sums[]; // [waves][MT][64][4]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r16 = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, room = (p.K + 15) & ~15;
    const __amdgpu_buffer_rsrc_t bbuf = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<unsigned char *>(p.b + (long long)n0 * p.ldb), 0, (min(16, p.N - n0) - 1) * (int)p.ldb + room, 0x00020000);
    const __amdgpu_buffer_rsrc_t abuf = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<unsigned char *>(p.a), 0, (p.M - 1) * (int)p.lda + room, 0x00020000);
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    const unsigned char *sb = p.sb + (long long)(min(n0 + r16, p.N - 1) >> p.b_shift) * p.ldsb;
    f8_f4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = (f8_f4){0.f, 0.f, 0.f, 0.f};
    auto piece = [&](__amdgpu_buffer_rsrc_t buf, int row, int ld, int col) -> u4 {
        return __builtin_amdgcn_raw_buffer_load_b128(buf, col < p.K ? row * ld + col : (int)0x80000000, 0, 0);
    };
    auto whole = [&](const u4 &lo, const u4 &hi, int col) -> f8_v8 {
        int w[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) { w[i] = (int)lo[i]; w[4 + i] = (int)hi[i]; }
        if (p.K & 15) {
            f8_cut(w, col, p.K);
            f8_cut(w + 4, col + 64, p.K);
        }
        f8_v8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = w[i];
        return v;
    };
    const int turns = (p.K + 511) >> 9;
    for (int turn = wave; turn < turns; turn += waves) {
        u4 b[4][2], a[MT][4][2];
        unsigned xa[MT];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) b[k][h] = piece(bbuf, r16, (int)p.ldb, turn * 512 + k * 128 + g * 16 + h * 64);
        const unsigned xb = *(const unsigned *)(sb + turn * 4);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int row = i * 16 + r16;
            xa[i] = *(const unsigned *)(p.sa + (long long)min(row, p.M - 1) * p.ldsa + turn * 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    a[i][k][h] = piece(abuf, row, (int)p.lda, turn * 512 + k * 128 + g * 16 + h * 64);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int col = turn * 512 + k * 128 + g * 16;
            if (turn * 512 + k * 128 >= p.K) break; // nothing of this step is there (its scale byte is not either)
            const f8_v8 vb = whole(b[k][0], b[k][1], col);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const f8_v8 va = whole(a[i][k][0], a[i][k][1], col);
                if constexpr (WIDE) {
                    const float eb = lcf_exp2i((int)((xb >> (8 * k)) & 255) - 127);
                    const float ea = lcf_exp2i((int)((xa[i] >> (8 * k)) & 255) - 127);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            f8_to_bf16<FB>(vb[2 * q], vb[2 * q + 1], eb), f8_to_bf16<FA>(va[2 * q], va[2 * q + 1], ea),
                            acc[i], 0, 0, 0);
                } else {
                    acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb, va, acc[i], FB, FA, 0,
                                                                              (int)(xb >> (8 * k)), 0,
                                                                              (int)(xa[i] >> (8 * k)));
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
        *reinterpret_cast<f8_f4 *>(few_sums + ((wave * MT + i) * 64 + lane) * 4) = acc[i];
    __syncthreads();
    // lane (r16, g) holds columns n0 + 4 g + r of row 16 i + r16
    const int m = wave * 16 + r16, n = n0 + 4 * g;
    if (wave >= MT || m >= p.M) return;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < waves; ++w) {
        const f8_f4 q = *reinterpret_cast<const f8_f4 *>(few_sums + ((w * MT + wave) * 64 + lane) * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += q[r];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (n + r >= p.N) break;
        float x = v[r];
        if (p.scale) x *= p.scale[n + r];
        if (p.shift) x += p.shift[n + r];
        if (p.relu) x = x < 0.f ? 0.f : x;
        const long long at = (long long)m * p.ldo + n + r;
        if (p.code == LCF_F32) ((float *)p.out)[at] = x;
        else if (p.code == LCF_BF16) ((lcf_b *)p.out)[at] = lcf_from_f32<lcf_b>(x);
        else ((lcf_h *)p.out)[at] = lcf_from_f32<lcf_h>(x);
    }
}

// joins the splits' parts in a fixed order and applies the epilogue.  A workgroup takes 64
// consecutive elements: thread = (split line t / 16, four elements t % 16); 16 lines run over the
// splits side by side and meet in LDS.
__global__ void __launch_bounds__(256) f8_join_kernel(F8Gemm p, int splits)
{
    __shared__ float lds[16][64];
    const long long total = (long long)p.M * p.N;
    const int part = threadIdx.x & 15, line = threadIdx.x >> 4;
    const long long e = (long long)blockIdx.x * 64 + part * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = line; s < splits; s += 16) {
        const float *o = p.ws + s * total + e;
        if (e + 4 <= total) {
            const lcf_f4u q = *reinterpret_cast<const lcf_f4u *>(o);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += q[k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (e + k < total) v[k] += o[k];
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) lds[line][part * 4 + k] = v[k];
    __syncthreads();
    const long long i = (long long)blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x >= 64 || i >= total) return;
    float x = 0.f;
#pragma unroll
    for (int l = 0; l < 16; ++l) x += lds[l][threadIdx.x];
    const long long m = i / p.N;
    const int n = (int)(i - m * p.N);
    if (p.scale) x *= p.scale[n];
    if (p.shift) x += p.shift[n];
    if (p.relu) x = x < 0.f ? 0.f : x;
    if (p.code == LCF_F32) ((float *)p.out)[m * p.ldo + n] = x;
    else if (p.code == LCF_BF16) ((lcf_b *)p.out)[m * p.ldo + n] = lcf_from_f32<lcf_b>(x);
    else ((lcf_h *)p.out)[m * p.ldo + n] = lcf_from_f32<lcf_h>(x);
}

static bool f8_is_thin(int M, int N, int K, bool wide);
enum { F8_256, F8_128, F8_64, F8_NARROW };
struct F8Plan {
    int thin, few, shape, tiles_m, tiles_n, splits, ksteps;
};
// A few rows over a long sum: f8_few_kernel has a workgroup for 16 columns walk all of k, and every piece
// of 16 rows adds to a turn, where the tiles divide k over the chip.  The border, us of f8_few_kernel and of
// the tiles with their split: 8 x 1024 columns, K 4096 6.4 / 8.5, 8192 9.7 / 8.6, 16384 16.6 / 9.3, 131072
// 107 / 31; 64 x 1024 columns, K 2048 8.3 / 9.3, 4096 13.4 / 9.9, 131072 328 / 34; 50 x 200 over 136000 rows
// (a weight gradient) 226 / 19.  Up to 16 rows more than 8192 columns are workgroups enough by themselves
// (8 x 16384, K 16384 63 / 100; 8 x 8192 38 / 30, and past 256 MB of b 121 / 141, left to the tiles).
static bool f8_long(int M, int N, int K)
{
    const int mt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    return (long long)mt * K > 8192 && (M > 16 || N <= 8192);
}
// divided: whether there is a workspace for dividing the sums of a few rows
static F8Plan f8_plan(int M, int N, int K, bool wide, bool divided)
{
    F8Plan q;
    q.thin = f8_is_thin(M, N, K, wide);
    q.few = M <= 64 && K > 0 && !(divided && f8_long(M, N, K));
    const long long t256 = (long long)((M + 255) / 256) * ((N + 255) / 256);
    const long long t128 = (long long)((M + 127) / 128) * ((N + 127) / 128);
    // the largest tile that still gives the 256 units work: 256 x 256 (one workgroup fills a unit),
    // 128 x 128 (two do), 64 x 128 (three do); 128 x 64 where there are no more columns
    q.shape = N <= 64 ? F8_NARROW : M <= 64 ? F8_64 : t256 >= 192 ? F8_256 : t128 >= 512 ? F8_128 : F8_64;
    const int bm = q.shape == F8_256 ? 256 : q.shape == F8_64 ? 64 : 128;
    const int bn = q.shape == F8_256 ? 256 : q.shape == F8_NARROW ? 64 : 128;
    q.tiles_m = (M + bm - 1) / bm;
    q.tiles_n = (N + bn - 1) / bn;
    const int steps = (K + 127) / 128;
    const long long tiles = (long long)q.tiles_m * q.tiles_n;
    // a few tiles over a long sum: split it until the chip's 256 units have work, at least four
    // steps to a split
    int splits = 1;
    if (!q.thin && !q.few && tiles < 128) {
        splits = (int)(256 / tiles);
        if (splits > steps / 4) splits = steps / 4;
        if (splits < 1) splits = 1;
    }
    q.ksteps = (steps + splits - 1) / splits;
    if (q.ksteps < 1) q.ksteps = 1;
    q.splits = steps ? (steps + q.ksteps - 1) / q.ksteps : 1;
    return q;
}

static size_t f8_parts_bytes(const F8Plan &q, int M, int N)
{
    return q.splits > 1 ? (size_t)q.splits * M * N * sizeof(float) : 0;
}
extern "C" size_t lcf_f8_gemm_split_bytes(int M, int N, int K, int out_dtype)
{
    if (M < 1 || N < 1 || K < 1 || M > F8_MOST || N > F8_MOST || K > F8_MOST) return 0;
    return f8_parts_bytes(f8_plan(M, N, K, out_dtype == LCF_F32, true), M, N);
}
extern "C" size_t lcf_f8_gemm_workspace_bytes(int M, int N, int K, int out_dtype)
{
    return M <= 64 ? 0 : lcf_f8_gemm_split_bytes(M, N, K, out_dtype);
}

// whether f8_stream_kernel takes a product: b in registers, rows enough for every wave, and whole
// 16-byte pieces of an output row
static bool f8_is_thin(int M, int N, int K, bool wide)
{
    return K > 0 && K <= (wide ? 256 : 512) && N <= 256 && N % (wide ? 4 : 8) == 0 && M >= 4096;
}
// (buffer stores want four-byte addresses; an output that has none takes the tiles, which for these
// sizes are never split and need no workspace either)
static bool f8_out_ok(const void *out, long long ldo, int code)
{
    return !((uintptr_t)out & 3) && !(ldo * lcf_type_size(code) & 3) && ldo <= (1 << 22);
}

template <int FA, int FB, bool WIDE, typename T> static int f8_stream_launch(const F8Gemm &p, hipStream_t st)
{
    const int wn_shift = p.N <= 64 ? 0 : p.N <= 128 ? 1 : 2, rows = 16 << (2 - wn_shift);
    const long long want = ((long long)p.M + rows - 1) / rows;
    // as many workgroups as the chip holds at once (by the registers they need)
    const int ks = (p.K + 127) / 128, most = 256 * (WIDE ? (ks == 1 ? 3 : 2) : ks == 1 ? 5 : ks == 2 ? 3 : 2);
    // and rows enough for each wave that fetching its 64 columns of b is the smaller part (M = 40000,
    // N = 64, K = 256: 11.1 us with one turn a wave, 8.5 with three or four)
    const long long three = (want + 2) / 3;
    const int grid = (int)(three < most ? three : most);
    if (ks == 1) f8_stream_kernel<FA, FB, WIDE, 1, T><<<grid, 256, 0, st>>>(p, wn_shift);
    else if (ks == 2) f8_stream_kernel<FA, FB, WIDE, 2, T><<<grid, 256, 0, st>>>(p, wn_shift);
    else if constexpr (!WIDE) f8_stream_kernel<FA, FB, WIDE, 4, T><<<grid, 256, 0, st>>>(p, wn_shift);
    LCF_CHECK_LAUNCH();
    return LCF_OK;
}

template <int FA, int FB, bool WIDE, int WM, int WN, int MT>
static int f8_tile_launch(const F8Gemm &p, unsigned grid, hipStream_t st)
{
    constexpr int room = 2 * (WM * MT * 16 + WN * 64) * 132;
    // more LDS than a launch may take unasked
    if (room > 65536 && hipFuncSetAttribute((const void *)f8_gemm_kernel<FA, FB, WIDE, WM, WN, MT>,
                                            hipFuncAttributeMaxDynamicSharedMemorySize, room) != hipSuccess)
        return LCF_ERR_LAUNCH;
    f8_gemm_kernel<FA, FB, WIDE, WM, WN, MT><<<grid, WM * WN * 64, room, st>>>(p);
    LCF_CHECK_LAUNCH();
    return LCF_OK;
}

template <int FA, int FB, bool WIDE> static int f8_gemm_launch2(const F8Gemm &p, const F8Plan &q, hipStream_t st)
{
    if (q.thin && f8_out_ok(p.out, p.ldo, p.code)) return f8_stream_launch<FA, FB, WIDE, unsigned char>(p, st);
    if (q.few) {
        // a wave for each turn along k, eight at most, 16 where there are few columns; and as many as
        // there are pieces of 16 rows to write
        const int turns = (p.K + 511) / 512, most = p.N >= 4096 || p.M > 16 ? 8 : 16, mt = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
        int waves = turns < most ? turns : most;
        if (waves < mt) waves = mt;
        const unsigned g = (unsigned)((p.N + 15) / 16), nt = waves * 64, room = waves * mt * 1024;
        if (mt == 1) f8_few_kernel<FA, FB, WIDE, 1><<<g, nt, room, st>>>(p);
        else if (mt == 2) f8_few_kernel<FA, FB, WIDE, 2><<<g, nt, room, st>>>(p);
        else f8_few_kernel<FA, FB, WIDE, 4><<<g, nt, room, st>>>(p);
        LCF_CHECK_LAUNCH();
        return LCF_OK;
    }
    const unsigned grid = (unsigned)(((long long)q.tiles_m * q.tiles_n * q.splits + 7) / 8 * 8);
    switch (q.shape) {
    case F8_256: return f8_tile_launch<FA, FB, WIDE, 2, 4, 8>(p, grid, st);
    case F8_128: return f8_tile_launch<FA, FB, WIDE, 2, 2, 4>(p, grid, st);
    case F8_64: return f8_tile_launch<FA, FB, WIDE, 2, 2, 2>(p, grid, st);
    default: return f8_tile_launch<FA, FB, WIDE, 4, 1, 2>(p, grid, st);
    }
}
template <int FA, int FB> static int f8_gemm_launch(const F8Gemm &p, const F8Plan &q, hipStream_t st)
{
    return p.code == LCF_F32 ? f8_gemm_launch2<FA, FB, true>(p, q, st) : f8_gemm_launch2<FA, FB, false>(p, q, st);
}

// x [M, K] of fp32 / bf16 / fp16 rows through b [N, K] in one launch
extern "C" int lcf_f8_linear(const void *x, long long ldx, int dtype, const void *b, long long ldb,
                             const unsigned char *sb, int ldsb, int b_square, int M, int N, int K, const float *scale,
                             const float *shift, int relu, void *out, long long ldo, int out_dtype, void *stream)
{
    if (M < 0 || N < 0 || K < 0 || !lcf_is_type(dtype) || !lcf_is_type(out_dtype)) return LCF_ERR_ARG;
    if (M == 0 || N == 0) return LCF_OK;
    if (!out || ldo < N) return LCF_ERR_ARG;
    if (K > 0 && (!x || ldx < K || !f8_form_ok(b, ldb, sb, ldsb, K))) return LCF_ERR_ARG;
    // rows are read 16 bytes at a time, by buffer loads that want four-byte addresses
    if (!f8_is_thin(M, N, K, out_dtype == LCF_F32) || dtype != out_dtype || (K & 7) || ((uintptr_t)x & 3) ||
        (ldx * lcf_type_size(dtype) & 3) || ldx > (1 << 22) || ldb > (1 << 22) ||
        !f8_out_ok(out, ldo, out_dtype))
        return LCF_ERR_UNSUPPORTED;
    F8Gemm p{};
    p.a = (const unsigned char *)x;
    p.lda = ldx;
    p.b = (const unsigned char *)b;
    p.ldb = ldb;
    p.sb = sb;
    p.ldsb = ldsb;
    p.b_shift = b_square ? 7 : 0;
    p.scale = scale;
    p.shift = shift;
    p.relu = relu;
    p.out = out;
    p.ldo = ldo;
    p.code = out_dtype;
    p.M = M;
    p.N = N;
    p.K = K;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == LCF_F32) return f8_stream_launch<0, 0, true, float>(p, st);
    if (dtype == LCF_BF16) return f8_stream_launch<0, 0, false, lcf_b>(p, st);
    return f8_stream_launch<0, 0, false, lcf_h>(p, st);
}

extern "C" int lcf_f8_gemm(const void *a, long long lda, const unsigned char *sa, int ldsa, int a_fmt, const void *b,
                           long long ldb, const unsigned char *sb, int ldsb, int b_fmt, int b_square, int M, int N,
                           int K, const float *scale, const float *shift, int relu, void *out, long long ldo,
                           int out_dtype, void *ws, size_t ws_bytes, void *stream)
{
    if (M < 0 || N < 0 || K < 0 || !lcf_is_type(out_dtype)) return LCF_ERR_ARG;
    if ((a_fmt != LCF_E4M3 && a_fmt != LCF_E5M2) || (b_fmt != LCF_E4M3 && b_fmt != LCF_E5M2)) return LCF_ERR_ARG;
    if (M == 0 || N == 0) return LCF_OK;
    if (!out || ldo < N) return LCF_ERR_ARG;
    if (K > 0 && (!f8_form_ok(a, lda, sa, ldsa, K) || !f8_form_ok(b, ldb, sb, ldsb, K))) return LCF_ERR_ARG;
    // a tile's rows are addressed in 32 bits, and a launch has fewer than 2^32 threads (512 a tile at
    // most, 1024 for 16 columns of a few rows)
    if (lda > (1 << 22) || ldb > (1 << 22) || M > F8_MOST || N > F8_MOST) return LCF_ERR_UNSUPPORTED;
    F8Plan q = f8_plan(M, N, K, out_dtype == LCF_F32, true);
    if (M <= 64 && q.splits > 1 && (!ws || ws_bytes < f8_parts_bytes(q, M, N)))
        q = f8_plan(M, N, K, out_dtype == LCF_F32, false);
    const bool thin = q.thin && f8_out_ok(out, ldo, out_dtype);
    if (!thin && (M <= 64 && K > 0 ? N > 1 << 25 : (long long)q.tiles_m * q.tiles_n * q.splits > (1 << 23) - 8))
        return LCF_ERR_UNSUPPORTED;
    if (q.splits > 1) {
        if (!ws) return LCF_ERR_ARG;
        if (ws_bytes < f8_parts_bytes(q, M, N)) return LCF_ERR_WORKSPACE;
    }
    F8Gemm p{(const unsigned char *)a, sa, (const unsigned char *)b, sb, scale, shift, out,
             q.splits > 1 ? (float *)ws : nullptr, lda, ldb, ldo, ldsa, ldsb, b_square ? 7 : 0, M, N, K, relu,
             out_dtype, q.tiles_m, q.tiles_n, q.splits, q.ksteps};
    hipStream_t st = (hipStream_t)stream;
    int rc;
    if (a_fmt == LCF_E4M3 && b_fmt == LCF_E4M3) rc = f8_gemm_launch<0, 0>(p, q, st);
    else if (a_fmt == LCF_E4M3) rc = f8_gemm_launch<0, 1>(p, q, st);
    else if (b_fmt == LCF_E4M3) rc = f8_gemm_launch<1, 0>(p, q, st);
    else rc = f8_gemm_launch<1, 1>(p, q, st);
    if (rc != LCF_OK) return rc;
    if (q.splits > 1) {
        f8_join_kernel<<<(unsigned)(((long long)M * N + 63) / 64), 256, 0, st>>>(p, q.splits);
        LCF_CHECK_LAUNCH();
    }
    return LCF_OK;
}

// ---------------------------------------------------------------- a thin layer's weight gradient
// out [M, N] = A^T B for A [R, M] and B [R, N] of fp32 / bf16 / fp16, both brought into columns form
// (blocks of 128 rows of a column) on the way: one reading of each and nothing written but the sums.
// A workgroup takes 128 rows at a time.  A wave holds 32 columns of them, a lane 8 rows x 8 columns
// (rl, cl): a column's largest magnitude is the lane's own rows and four lane swaps, without a barrier.
// The bytes are turned into LDS (a column's 128 rows, one behind the other, columns 144 bytes apart:
// 16 columns start in 16 different sets of four banks), and the next 128 rows are asked for before the
// products of these, 32 x 64 outputs a wave, begin.  Rows behind R read as zeros (offsets past the
// buffer's end).  As many workgroups as there are compute units, each with its own sums, joined in a
// fixed order.  Bound by memory: 136000 rows, 64 x 256, bf16 25 us (3.5 TB/s; a unit waits while it
// turns), fp32 36 us (4.8 TB/s), and 6 us for the join; the two columns forms, their product and its
// join took 59 us.  Outputs of 256 columns are kept whole beside 64 of the other side, where dividing
// them in two takes 28 us; 256 x 256 is made in four parts (136000 rows 57 us).  Beyond that each part
// reads its sides again and the columns forms take over.
#define F8_TURN 144
#define F8_SLOTS 256 // workgroups of a launch: 384 take 30 us and 192 28 us where 256 take 25
struct F8Wgrad {
    const unsigned char *a, *b;
    float *parts, *sums; // [workgroups][M][N]; [workgroups][width of the summed side] or NULL
    long long lda, ldb;
    int R, M, N, steps, sum_a; // steps: blocks of 128 rows of a workgroup
};

typedef unsigned short f8_h2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned f8_max16(unsigned a, unsigned b)
{
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(f8_h2, a), __builtin_bit_cast(f8_h2, b)));
}

template <typename T, bool WIDE, int MC, int NC> // MC, NC: 64 columns of A, of B
__global__ void __launch_bounds__(128 * (MC + NC), sizeof(T) == 2 && MC + NC < 5 ? 4 : 3) f8_wgrad_kernel(F8Wgrad p)
{
    constexpr int E = sizeof(T), D = 2 * E; // dwords of eight columns
    __shared__ __align__(16) unsigned char turn[64 * (MC + NC) * F8_TURN];
    __shared__ __align__(8) unsigned char exps[64 * (MC + NC)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = lane & 3, rl = lane >> 2, r16 = lane & 15, g = lane >> 4;
    const int mine = wave < 2 * MC * NC ? wave : 0;
    const bool of_b = wave >= 2 * MC;
    const int a0 = blockIdx.y * 64 * MC, b0 = blockIdx.z * 64 * NC; // the workgroup's first columns
    const int col = of_b ? b0 + (wave - 2 * MC) * 32 + cl * 8 : a0 + wave * 32 + cl * 8, width = of_b ? p.N : p.M;
    const int ld = (int)(of_b ? p.ldb : p.lda);
    const unsigned char *src = of_b ? p.b : p.a;
    const bool summed = p.sums && (p.sum_a ? !of_b && blockIdx.z == 0 : of_b && blockIdx.y == 0);
    const int off = col < width ? (rl * 8 * ld + col) * E : (int)0x80000000;
    unsigned v[8][D];
    auto ask = [&](int block) {
        const int left = min(p.R - block * 128, 128);
        const __amdgpu_buffer_rsrc_t buf = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<unsigned char *>(src + (long long)block * 128 * ld * E), 0, ((left - 1) * ld + width) * E, 0x00020000);
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int d = 0; d < D; d += 4) {
                const u4 q = __builtin_amdgcn_raw_buffer_load_b128(buf, off + i * ld * E + d * 4, 0, 0);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][d + k] = q[k];
            }
    };
    auto value = [&](int i, int j) -> float {
        if constexpr (E == 4) return __uint_as_float(v[i][j]);
        else return lcf_to_f32(__builtin_bit_cast(T, (unsigned short)(v[i][j >> 1] >> (16 * (j & 1)))));
    };
    f8_f4 acc[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = (f8_f4){0.f, 0.f, 0.f, 0.f};
    __shared__ float totals[64 * (MC + NC)]; // a wave's own 32 columns
    if (lane < 32) totals[wave * 32 + lane] = 0.f;

    const int blocks = (p.R + 127) >> 7, first = blockIdx.x * p.steps, last = min(first + p.steps, blocks);
    ask(first);
    for (int block = first; block < last; ++block) {
        if (summed) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += value(i, j);
#pragma unroll
                for (int x = 4; x <= 32; x <<= 1) s += __shfl_xor(s, x, 64);
                if (rl == 0) totals[wave * 32 + cl * 8 + j] += s;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the columns' largest finite magnitudes; infinities become NaN where one is found
        float top[8];
        if constexpr (E == 2) {
            constexpr unsigned INF = __is_same(T, lcf_b) ? 0x7F80u : 0x7C00u;
            unsigned m[4];
            // magnitudes of 16 bits order as whole numbers do
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                m[d] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) m[d] = f8_max16(m[d], v[i][d] & 0x7FFF7FFFu);
            }
            const unsigned all = f8_max16(f8_max16(m[0], m[1]), f8_max16(m[2], m[3]));
            if (__builtin_expect(__any((all & 0xFFFF) >= INF || (all >> 16) >= INF), 0)) {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    m[d] = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        unsigned u = v[i][d] & 0x7FFF7FFFu;
                        if ((u & 0xFFFF) >= INF) { v[i][d] |= 0x7FFFu; u &= 0xFFFF0000u; }
                        if ((u >> 16) >= INF) { v[i][d] |= 0x7FFF0000u; u &= 0xFFFFu; }
                        m[d] = f8_max16(m[d], u);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
#pragma unroll
                for (int x = 4; x <= 32; x <<= 1) m[d] = f8_max16(m[d], (unsigned)__shfl_xor((int)m[d], x, 64));
                top[2 * d] = lcf_to_f32(__builtin_bit_cast(T, (unsigned short)(m[d] & 0xFFFF)));
                top[2 * d + 1] = lcf_to_f32(__builtin_bit_cast(T, (unsigned short)(m[d] >> 16)));
            }
        } else {
            float all = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                top[j] = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) top[j] = fmaxf(top[j], __builtin_fabsf(value(i, j)));
                all = fmaxf(all, top[j]);
            }
            if (__builtin_expect(__any(all > 3.402823466e38f), 0)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    top[j] = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (__builtin_fabsf(value(i, j)) > 3.402823466e38f) v[i][j] = 0x7FC00000u;
                        top[j] = fmaxf(top[j], __builtin_fabsf(value(i, j)));
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int x = 4; x <= 32; x <<= 1) top[j] = fmaxf(top[j], __shfl_xor(top[j], x, 64));
        }
        if (block != first) __syncthreads(); // the last products have read their bytes
        unsigned e4[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int e = lcf_f8_exponent(top[j], LCF_E4M3);
            const float s = lcf_exp2i(-e);
            e4[j >> 2] |= (unsigned)(e + 127) << (8 * (j & 3));
            lcf_u2u w;
            w.x = lcf_f8_pack4(value(0, j) * s, value(1, j) * s, value(2, j) * s, value(3, j) * s, LCF_E4M3);
            w.y = lcf_f8_pack4(value(4, j) * s, value(5, j) * s, value(6, j) * s, value(7, j) * s, LCF_E4M3);
            *reinterpret_cast<uint2 *>(turn + (wave * 32 + cl * 8 + j) * F8_TURN + rl * 8) = make_uint2(w.x, w.y);
            __builtin_amdgcn_sched_barrier(0); // one column at a time: all at once would not fit the registers
        }
        if (rl == 0) *reinterpret_cast<uint2 *>(exps + wave * 32 + cl * 8) = make_uint2(e4[0], e4[1]);
        __builtin_amdgcn_sched_barrier(0);
        if (block + 1 < last) ask(block + 1);
        __syncthreads();
        { // (waves that have no outputs of their own make the first one's: around a branch the sums would
          // be held twice)
            const int m0 = mine % (2 * MC) * 32 + r16, n0 = 64 * MC + mine / (2 * MC) * 64 + r16;
            auto bytes = [&](int c) -> f8_v8 {
                const f8_v4 *t = reinterpret_cast<const f8_v4 *>(turn + c * F8_TURN + g * 32);
                const f8_v4 lo = t[0], hi = t[1];
                return (f8_v8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            };
            if constexpr (WIDE) { // few registers are left beside the rows asked for: 16 of a lane's 32 bytes at a time
                auto wide = [&](int c, int k, f8_b8 *w) {
                    const f8_v4 q = *reinterpret_cast<const f8_v4 *>(turn + c * F8_TURN + g * 32 + k * 16);
                    const float s = lcf_exp2i((int)exps[c] - 127);
                    w[0] = f8_to_bf16<LCF_E4M3>(q[0], q[1], s);
                    w[1] = f8_to_bf16<LCF_E4M3>(q[2], q[3], s);
                };
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    f8_b8 wa[2][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) wide(m0 + i * 16, k, wa[i]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        f8_b8 wb[2];
                        wide(n0 + t * 16, k, wb);
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[h], wa[i][h], acc[i][t], 0, 0, 0);
                        if (t == 1 || t == 3) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            } else {
                f8_v8 qa[2];
                int ea[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    qa[i] = bytes(m0 + i * 16);
                    ea[i] = exps[m0 + i * 16];
                }
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const f8_v8 qb = bytes(n0 + t * 16);
                    const int eb = exps[n0 + t * 16];
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(qb, qa[i], acc[i][t], LCF_E4M3, LCF_E4M3,
                                                                                     0, eb, 0, ea[i]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) f8_pin(acc[i]);
    if (wave < 2 * MC * NC) {
        float *o = p.parts + (long long)blockIdx.x * p.M * p.N;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int m = a0 + wave % (2 * MC) * 32 + i * 16 + r16, n = b0 + wave / (2 * MC) * 64 + t * 16 + 4 * g;
                if (m < p.M && n < p.N)
                    *reinterpret_cast<lcf_f4u *>(o + (long long)m * p.N + n) =
                        (lcf_f4u){acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]};
            }
    }
    if (summed && lane < 32 && col - cl * 8 + lane < width)
        p.sums[(long long)blockIdx.x * width + col - cl * 8 + lane] = totals[wave * 32 + lane];
}

struct F8WgradShape { // parts = 0: sizes that the kernel does not take
    int a, b, parts, steps; // a, b: columns of either side in a workgroup, in 64
};
static F8WgradShape f8_wgrad_shape(int R, int M, int N)
{
    F8WgradShape s{M <= 64 ? 1 : M <= 128 || N > 64 ? 2 : 4, N <= 64 ? 1 : N <= 128 || M > 64 ? 2 : 4, 0, 0};
    if (R < 1 || R > F8_MOST || M < 8 || N < 8 || (M & 7) || (N & 7) || M > 256 || N > 256) return s;
    const int blocks = (R + 127) / 128, groups = (M + 64 * s.a - 1) / (64 * s.a) * ((N + 64 * s.b - 1) / (64 * s.b));
    s.steps = ((long long)blocks * groups + F8_SLOTS - 1) / F8_SLOTS;
    s.parts = (blocks + s.steps - 1) / s.steps;
    return s;
}

template <typename T, bool WIDE> static void f8_wgrad_launch(const F8Wgrad &p, const F8WgradShape &s, hipStream_t st)
{
    const dim3 grid(s.parts, (p.M + 64 * s.a - 1) / (64 * s.a), (p.N + 64 * s.b - 1) / (64 * s.b));
    if (s.a == 1 && s.b == 1) f8_wgrad_kernel<T, WIDE, 1, 1><<<grid, 256, 0, st>>>(p);
    else if (s.a == 2 && s.b == 1) f8_wgrad_kernel<T, WIDE, 2, 1><<<grid, 384, 0, st>>>(p);
    else if (s.a == 1 && s.b == 2) f8_wgrad_kernel<T, WIDE, 1, 2><<<grid, 384, 0, st>>>(p);
    else if (s.a == 4) f8_wgrad_kernel<T, WIDE, 4, 1><<<grid, 640, 0, st>>>(p);
    else if (s.b == 4) f8_wgrad_kernel<T, WIDE, 1, 4><<<grid, 640, 0, st>>>(p);
    else f8_wgrad_kernel<T, WIDE, 2, 2><<<grid, 512, 0, st>>>(p);
}

extern "C" size_t lcf_f8_weight_grad_workspace_bytes(int R, int K, int N)
{
    const F8WgradShape s = f8_wgrad_shape(R, K, N);
    return s.parts == 0 ? 0 : (size_t)s.parts * ((size_t)K * N + N) * sizeof(float);
}

extern "C" int lcf_f8_weight_grad(const void *x, long long ldx, const void *dy, long long lddy, int R, int K, int N,
                                  int dtype, int turned, void *dw, int dw_dtype, void *db, int db_dtype, void *ws,
                                  size_t ws_bytes, void *stream)
{
    if (R < 0 || K < 0 || N < 0 || !lcf_is_type(dtype) || !lcf_is_type(dw_dtype) || (db && !lcf_is_type(db_dtype)))
        return LCF_ERR_ARG;
    const F8WgradShape s = turned ? f8_wgrad_shape(R, K, N) : f8_wgrad_shape(R, N, K);
    if (s.parts == 0) return LCF_ERR_UNSUPPORTED;
    if (!x || !dy || !dw || ldx < K || lddy < N) return LCF_ERR_ARG;
    // rows are read 16 bytes at a time by buffer loads that want four-byte addresses and 32-bit offsets
    const int e = lcf_type_size(dtype);
    if (((uintptr_t)x & 3) || ((uintptr_t)dy & 3) || (ldx * e & 3) || (lddy * e & 3) || ldx > 1 << 20 || lddy > 1 << 20)
        return LCF_ERR_UNSUPPORTED;
    if (!ws) return LCF_ERR_ARG;
    if (ws_bytes < lcf_f8_weight_grad_workspace_bytes(R, K, N)) return LCF_ERR_WORKSPACE;
    F8Wgrad p{};
    p.a = (const unsigned char *)(turned ? x : dy);
    p.lda = turned ? ldx : lddy;
    p.b = (const unsigned char *)(turned ? dy : x);
    p.ldb = turned ? lddy : ldx;
    p.M = turned ? K : N;
    p.N = turned ? N : K;
    p.R = R;
    p.steps = s.steps;
    p.parts = (float *)ws;
    p.sums = db ? p.parts + (size_t)s.parts * K * N : nullptr;
    p.sum_a = !turned;
    hipStream_t st = (hipStream_t)stream;
    const bool wide = dw_dtype == LCF_F32;
    if (dtype == LCF_F32) wide ? f8_wgrad_launch<float, true>(p, s, st) : f8_wgrad_launch<float, false>(p, s, st);
    else if (dtype == LCF_BF16) wide ? f8_wgrad_launch<lcf_b, true>(p, s, st) : f8_wgrad_launch<lcf_b, false>(p, s, st);
    else wide ? f8_wgrad_launch<lcf_h, true>(p, s, st) : f8_wgrad_launch<lcf_h, false>(p, s, st);
    LCF_CHECK_LAUNCH();
    F8Gemm j{};
    j.ws = p.parts;
    j.out = dw;
    j.ldo = p.N;
    j.code = dw_dtype;
    j.M = p.M;
    j.N = p.N;
    f8_join_kernel<<<(unsigned)((K * N + 63) / 64), 256, 0, st>>>(j, s.parts);
    LCF_CHECK_LAUNCH();
    return db ? lcf_sum_parts(p.sums, s.parts, N, db, db_dtype, stream) : LCF_OK;
}
