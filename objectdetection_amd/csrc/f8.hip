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
//     below the largest of a group (measured; between groups it adds in fp32): an error of up to
//     2^-10 of a group's sum of magnitudes, 1.5e-5 of the result on random data -- below a 16-bit
//     store's half step (2^-9 bf16, 2^-12 fp16), but not what an fp32 output promises.
//   fp32 outputs: the bytes become bf16 in registers, scaled (v_cvt_scalef32_pk_bf16_*: q 2^e is
//     exact), and v_mfma_f32_16x16x32_bf16 adds the exact products in fp32, at half the peak rate.
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
    long long ldx, ldq, ldqt;
    int R, C, lds, ldst, fmt, square;
};

// Rows form only: 16 lanes hold one block of 128 columns of one row (eight columns each), its
// largest magnitude is four lane swaps, nothing goes through LDS.  Rows narrower than 128 take as
// many lanes as they need (LPB).
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
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, lcf_finite_abs(v[i]));
#pragma unroll
        for (int d = LPB / 2; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
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
// rows rl + 16 i (i < 8) and columns 8 cl .. 8 cl + 7; a row's magnitudes meet over the 16 lanes of
// equal rl, a column's over the thread's own rows, the wave's four row lanes and, through LDS, the
// four waves.  The transposed bytes are turned in LDS and leave as 16-byte pieces of whole rows.
#define F8_TP 144 // bytes of a transposed row in LDS: 128 and a pad of 16 (other banks for the next)
template <typename T> __global__ void __launch_bounds__(256) f8_tile_kernel(F8Quant p)
{
    __shared__ float colmax[4][128];
    __shared__ __align__(16) unsigned char turn[128 * F8_TP];
    const int tid = threadIdx.x, cl = tid & 15, rl = tid >> 4, wave = tid >> 6;
    const int r0 = blockIdx.y * 128, c0 = blockIdx.x * 128;
    const int col = c0 + cl * 8;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = r0 + rl + i * 16;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        if (row < p.R && col < p.C) lcf_ld8_tail((const T *)p.x + row * p.ldx, col, p.C, v[i]);
    }
    float cm[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        cm[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) cm[j] = fmaxf(cm[j], lcf_finite_abs(v[i][j]));
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
    if (p.square) {
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) all = fmaxf(all, __shfl_xor(all, d, 64));
    }
    const int esq = lcf_f8_exponent(all, p.fmt);
    if (p.q) {
        const int room = (p.C + 15) & ~15;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = r0 + rl + i * 16;
            int e = esq;
            if (!p.square) {
                float top = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, lcf_finite_abs(v[i][j]));
#pragma unroll
                for (int d = 8; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
                e = lcf_f8_exponent(top, p.fmt);
            }
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
        int e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            e[j] = p.square ? esq : lcf_f8_exponent(cm[j], p.fmt);
            const float s = lcf_exp2i(-e[j]);
            const unsigned a = lcf_f8_pack4(v[0][j] * s, v[1][j] * s, v[2][j] * s, v[3][j] * s, p.fmt);
            const unsigned b = lcf_f8_pack4(v[4][j] * s, v[5][j] * s, v[6][j] * s, v[7][j] * s, p.fmt);
            unsigned char *t = turn + (cl * 8 + j) * F8_TP + rl;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t[i * 16] = (unsigned char)(a >> (8 * i));
                t[i * 16 + 64] = (unsigned char)(b >> (8 * i));
            }
        }
        if (rl == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (p.square ? (cl == 0 && j == 0) : col + j < p.C) {
                    unsigned char *sr = p.st + (long long)(p.square ? blockIdx.x : col + j) * p.ldst;
                    sr[blockIdx.y] = (unsigned char)(e[j] + 127);
                    if (blockIdx.y == gridDim.y - 1)
                        for (int k = gridDim.y; k & 3; ++k) sr[k] = 0;
                }
            }
        }
        __syncthreads();
        const int room = (p.R + 15) & ~15;
        for (int k = tid; k < 128 * 8; k += 256) {
            const int c = k >> 3, part = (k & 7) * 16;
            if (c0 + c < p.C && r0 + part < room)
                *reinterpret_cast<uint4 *>(p.qt + (long long)(c0 + c) * p.ldqt + r0 + part) =
                    *reinterpret_cast<const uint4 *>(turn + c * F8_TP + part);
        }
    }
}

template <typename T> static void f8_quant_launch(const F8Quant &p, hipStream_t st)
{
    if (p.q && !p.qt && !p.square) {
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

static bool f8_form_ok(const void *q, long long ld, const unsigned char *s, int lds, int C)
{
    return q && s && !((uintptr_t)q & 15) && !((uintptr_t)s & 3) && !(ld & 15) && !(lds & 3) && ld >= C &&
           lds >= (C + 127) / 128;
}

extern "C" int lcf_f8_quant(const void *x, long long ldx, int R, int C, int dtype, int fmt, int square, void *q,
                            long long ldq, unsigned char *s, int lds, void *qt, long long ldqt, unsigned char *st,
                            int ldst, void *stream)
{
    if (R < 0 || C < 0 || !lcf_is_type(dtype) || (fmt != LCF_E4M3 && fmt != LCF_E5M2)) return LCF_ERR_ARG;
    if (R == 0 || C == 0) return LCF_OK;
    if (!x || ldx < C || (!q && !qt)) return LCF_ERR_ARG;
    if (q && !f8_form_ok(q, ldq, s, lds, C)) return LCF_ERR_ARG;
    if (qt && !f8_form_ok(qt, ldqt, st, ldst, R)) return LCF_ERR_ARG;
    // the grid's second dimension counts 128-row tiles
    if ((qt || square) && (R + 127) / 128 > 65535) return LCF_ERR_UNSUPPORTED;
    F8Quant p{x, (unsigned char *)q, s, (unsigned char *)qt, st, ldx, ldq, ldqt, R, C, lds, ldst, fmt, square};
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
    int tiles_m, tiles_n, ksteps; // ksteps: 128-column steps of one split
};

__device__ __forceinline__ void f8_store(const F8Gemm &p, long long m, int n, const float *v, int count)
{
    // v: out columns n .. n + 15 of row m
    float s[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float x = v[i];
        if (i < count) {
            if (p.scale) x *= p.scale[n + i];
            if (p.shift) x += p.shift[n + i];
        }
        s[i] = p.relu ? (x < 0.f ? 0.f : x) : x; // NaN stays
    }
    auto put = [&](auto *row) {
        if (count >= 16) {
            lcf_st8(row, s);
            lcf_st8(row + 8, s + 8);
        } else {
            using T = typename std::remove_pointer<decltype(row)>::type;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < count) row[i] = lcf_from_f32<T>(s[i]);
        }
    };
    if (p.code == LCF_F32) put((float *)p.out + m * p.ldo + n);
    else if (p.code == LCF_BF16) put((lcf_b *)p.out + m * p.ldo + n);
    else put((lcf_h *)p.out + m * p.ldo + n);
}

// bytes [col, col + 16) of a row of K: those behind the row's end become zeros
__device__ __forceinline__ void f8_cut(int *w, int col, int K)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = K - (col + 4 * i);
        if (left <= 0) w[i] = 0;
        else if (left < 4) w[i] &= (1 << (8 * left)) - 1;
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

// One workgroup of four waves makes BM x BN outputs, a wave BM/2 x BN/2 of them (WN = BN/2 = 64).
// The instruction's first operand is b, its second a: a lane then holds four consecutive columns n
// of one row m for each 16 x 16 piece, and with the pieces' rows dealt as n = 16 g + 4 t + r
// (g = lane / 16, t = piece, r = register) sixteen consecutive columns over the four pieces of a
// wave: whole 128-byte lines of a bf16 output leave straight from the registers.
// LDS holds 128 bytes of k for each row of a and b, twice (the next step's loads are in flight
// while this one multiplies).  A 16-byte piece c of row r sits at place c ^ swz(r), so that the
// eight lanes of a bank group read eight different places.
template <int FA, int FB, bool WIDE, int BM>
__global__ void __launch_bounds__(256) f8_gemm_kernel(F8Gemm p)
{
    constexpr int BN = 128, MT = BM / 32; // MT: 16-row pieces of a wave
    extern __shared__ __align__(16) unsigned char smem[];
    // a: [2][BM][128], b: [2][BN][128]
    unsigned char *la = smem, *lb = smem + 2 * BM * 128;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r16 = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x;
    const int tm = tile % p.tiles_m, tn = tile / p.tiles_m;
    const int m0 = tm * BM, n0 = tn * BN;
    const int wm = (wave & 1) * (BM / 2), wn = (wave >> 1) * 64;
    const int steps_all = (p.K + 127) >> 7;
    const int step0 = blockIdx.y * p.ksteps;
    const int step1 = min(steps_all, step0 + p.ksteps);

    auto swz_a = [](int r) { return r & 7; };
    auto swz_b = [](int r) { return (r & 3) | ((r >> 2) & 4); }; // rows 16 apart take the other half

    auto load = [&](int buf, int step) {
#pragma unroll
        for (int i = 0; i < BM / 32; ++i) {
            const int slot = i * 256 + tid, r = slot >> 3, c = (slot & 7) ^ swz_a(r);
            const int row = min(m0 + r, p.M - 1);
            int col = step * 128 + c * 16;
            if (col >= p.K) col = 0; // read, but cut away below
            *reinterpret_cast<uint4 *>(la + buf * BM * 128 + slot * 16) =
                *reinterpret_cast<const uint4 *>(p.a + row * p.lda + col);
        }
#pragma unroll
        for (int i = 0; i < BN / 32; ++i) {
            const int slot = i * 256 + tid, r = slot >> 3, c = (slot & 7) ^ swz_b(r);
            const int row = min(n0 + r, p.N - 1);
            int col = step * 128 + c * 16;
            if (col >= p.K) col = 0;
            *reinterpret_cast<uint4 *>(lb + buf * BN * 128 + slot * 16) =
                *reinterpret_cast<const uint4 *>(p.b + row * p.ldb + col);
        }
    };

    f8_f4 acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][t] = (f8_f4){0.f, 0.f, 0.f, 0.f};
    int rowa[MT], rowb[4];   // LDS rows of this lane's pieces
    const unsigned *sap[MT]; // their scales, four steps to a word
    const unsigned *sbp[4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        rowa[i] = wm + i * 16 + r16;
        sap[i] = (const unsigned *)(p.sa + (long long)min(m0 + rowa[i], p.M - 1) * p.ldsa);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        rowb[t] = wn + (r16 >> 2) * 16 + t * 4 + (r16 & 3);
        sbp[t] = (const unsigned *)(p.sb + (long long)(min(n0 + rowb[t], p.N - 1) >> p.b_shift) * p.ldsb);
    }
    if (step0 < step1) load(0, step0);
    __syncthreads();
    for (int step = step0; step < step1; ++step) {
        const int buf = (step - step0) & 1;
        if (step + 1 < step1) load(buf ^ 1, step + 1);
        int xa[MT], xb[4];
        const int sh = (step & 3) * 8;
#pragma unroll
        for (int i = 0; i < MT; ++i) xa[i] = sap[i][step >> 2] >> sh;
#pragma unroll
        for (int t = 0; t < 4; ++t) xb[t] = sbp[t][step >> 2] >> sh;
        const bool tail = step * 128 + 128 > p.K;
        auto frag = [&](const unsigned char *base, int r, int s) -> f8_v8 {
            f8_v8 v;
            const f8_v4 lo = *reinterpret_cast<const f8_v4 *>(base + r * 128 + ((g ^ s) * 16));
            const f8_v4 hi = *reinterpret_cast<const f8_v4 *>(base + r * 128 + (((g + 4) ^ s) * 16));
            int w[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (tail) {
                f8_cut(w, step * 128 + g * 16, p.K);
                f8_cut(w + 4, step * 128 + g * 16 + 64, p.K);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w[i];
            return v;
        };
        f8_v8 fb[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) fb[t] = frag(lb + buf * BN * 128, rowb[t], swz_b(rowb[t]));
        if constexpr (!WIDE) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const f8_v8 fa = frag(la + buf * BM * 128, rowa[i], swz_a(rowa[i]));
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    acc[i][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[t], fa, acc[i][t], FB, FA, 0,
                                                                                 xb[t], 0, xa[i]);
            }
        } else {
            f8_b8 wb[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    wb[t][s] = f8_to_bf16<FB>(fb[t][2 * s], fb[t][2 * s + 1], lcf_exp2i((xb[t] & 255) - 127));
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const f8_v8 fa = frag(la + buf * BM * 128, rowa[i], swz_a(rowa[i]));
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const f8_b8 wa = f8_to_bf16<FA>(fa[2 * s], fa[2 * s + 1], lcf_exp2i((xa[i] & 255) - 127));
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        acc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[t][s], wa, acc[i][t], 0, 0, 0);
                }
            }
        }
        __syncthreads();
    }
    const int n = n0 + wn + g * 16;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long long m = m0 + wm + i * 16 + r16;
        if (m >= p.M || n >= p.N) continue;
        float v[16];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[t * 4 + r] = acc[i][t][r];
        if (p.ws) {
            float *o = p.ws + ((long long)blockIdx.y * p.M + m) * p.N + n;
            if (n + 16 <= p.N) {
                lcf_st8(o, v);
                lcf_st8(o + 8, v + 8);
            } else {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (n + k < p.N) o[k] = v[k];
            }
        } else {
            f8_store(p, m, n, v, p.N - n);
        }
    }
}

// joins the splits' parts in their order and applies the epilogue; 16 columns a thread
__global__ void __launch_bounds__(256) f8_join_kernel(F8Gemm p, int splits)
{
    const int per = (p.N + 15) >> 4;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)p.M * per) return;
    const long long m = i / per;
    const int n = (int)(i - m * per) * 16, count = p.N - n;
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = 0.f;
    for (int s = 0; s < splits; ++s) {
        const float *o = p.ws + ((long long)s * p.M + m) * p.N + n;
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (k < count) v[k] += o[k];
    }
    f8_store(p, m, n, v, count);
}

struct F8Plan {
    int bm, tiles_m, tiles_n, splits, ksteps;
};
static F8Plan f8_plan(int M, int N, int K)
{
    F8Plan q;
    q.bm = 128;
    q.tiles_m = (M + 127) / 128;
    q.tiles_n = (N + 127) / 128;
    const int steps = (K + 127) / 128;
    const long long tiles = (long long)q.tiles_m * q.tiles_n;
    // a few tiles over a long sum: split it until the chip's 256 units have work, at least four
    // steps to a split
    int splits = 1;
    if (tiles < 128) {
        splits = (int)(256 / tiles);
        if (splits > steps / 4) splits = steps / 4;
        if (splits < 1) splits = 1;
    }
    q.ksteps = (steps + splits - 1) / splits;
    if (q.ksteps < 1) q.ksteps = 1;
    q.splits = steps ? (steps + q.ksteps - 1) / q.ksteps : 1;
    return q;
}

extern "C" size_t lcf_f8_gemm_workspace_bytes(int M, int N, int K)
{
    if (M < 1 || N < 1 || K < 1) return 0;
    const F8Plan q = f8_plan(M, N, K);
    return q.splits > 1 ? (size_t)q.splits * M * N * sizeof(float) : 0;
}

template <int FA, int FB> static void f8_gemm_launch(const F8Gemm &p, const F8Plan &q, hipStream_t st)
{
    const dim3 grid(q.tiles_m * q.tiles_n, q.splits);
    if (p.code == LCF_F32) f8_gemm_kernel<FA, FB, true, 128><<<grid, 256, 2 * (128 + 128) * 128, st>>>(p);
    else f8_gemm_kernel<FA, FB, false, 128><<<grid, 256, 2 * (128 + 128) * 128, st>>>(p);
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
    const F8Plan q = f8_plan(M, N, K);
    if ((long long)q.tiles_m * q.tiles_n > 0x7FFFFFFFll) return LCF_ERR_UNSUPPORTED;
    if (q.splits > 1) {
        if (!ws) return LCF_ERR_ARG;
        if (ws_bytes < (size_t)q.splits * M * N * sizeof(float)) return LCF_ERR_WORKSPACE;
    }
    F8Gemm p{(const unsigned char *)a, sa, (const unsigned char *)b, sb, scale, shift, out,
             q.splits > 1 ? (float *)ws : nullptr, lda, ldb, ldo, ldsa, ldsb, b_square ? 7 : 0, M, N, K, relu,
             out_dtype, q.tiles_m, q.tiles_n, q.ksteps};
    hipStream_t st = (hipStream_t)stream;
    if (a_fmt == LCF_E4M3 && b_fmt == LCF_E4M3) f8_gemm_launch<0, 0>(p, q, st);
    else if (a_fmt == LCF_E4M3) f8_gemm_launch<0, 1>(p, q, st);
    else if (b_fmt == LCF_E4M3) f8_gemm_launch<1, 0>(p, q, st);
    else f8_gemm_launch<1, 1>(p, q, st);
    LCF_CHECK_LAUNCH();
    if (q.splits > 1) {
        const long long n = (long long)M * ((N + 15) / 16);
        f8_join_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p, q.splits);
        LCF_CHECK_LAUNCH();
    }
    return LCF_OK;
}
