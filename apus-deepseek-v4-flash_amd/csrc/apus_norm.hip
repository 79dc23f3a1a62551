/*
 * apus_norm.hip — row kernels that feed the quantised products: RMS norm with
 * the residual's addition and 8-bit output, and the per-row integer
 * quantiser.
 *
 * Norm of a row: r = T(x + res) (T: fp32, or BF16 where the arrays are), v =
 * 1 / sqrt(sum r^2 / K + eps), y = fp32((r gamma) v). The sum, v and both
 * products are 64-bit (r gamma is exact there), so y is the correctly rounded
 * value but for one case in about 2^28 and its codes do not depend on how a
 * kernel splits the row; the vector units do 64-bit multiply-adds at half the
 * fp32 rate, and the kernel waits for memory either way.
 *
 * Codes are made of b = bf16(y): E4M3 with the act quant's rule (a power-of-two
 * scale per 128 columns), or integers with one scale a row: a = max(max |b|,
 * 2^-100), scale = fp32(a / 127), q = rint(fp32(b * fp32(127 / a))). All
 * roundings are monotone: where a row is read twice its max |b| is bf16 of its max
 * |r gamma|, known with the sum.
 *
 * A row with a non-finite r gives y as the formula does (0 or NaN) and codes 0
 * under the scale +inf (E4M3, as the act quant) or NaN (integers): a product's
 * row comes out NaN and the other rows are not touched.
 */
#include "apus_device.h"
#include "apus_internal.h"

#include <algorithm>

namespace {

template <bool BF>
__device__ __forceinline__ float ld_elem(const void *p, size_t i) {
    if constexpr (BF) return apus_u2f((uint32_t)((const uint16_t *)p)[i] << 16);
    else              return ((const float *)p)[i];
}
template <bool BF>
__device__ __forceinline__ void st_elem(void *p, size_t i, float v) {
    if constexpr (BF) ((uint16_t *)p)[i] = apus_bf16_bits(apus_bf16_rne(v));
    else              ((float *)p)[i] = v;
}

}  // namespace

/* Very short and very long rows, a workgroup a row: a pass for the sum, a pass for
 * the outputs, which reads r back from res_out (or forms it again). */
template <bool XB, bool YB>
__global__ __launch_bounds__(256) void apus_rmsnorm_any_kernel(ApusNormArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t K = a.K;
    __shared__ double red[2][4];
    for (size_t m = blockIdx.x; m < (size_t)a.M; m += gridDim.x) {
        const size_t xo = m * (size_t)a.ldx, ro = m * K;
        auto gam = [&](size_t k) { return (double)(a.gamma_bf16 ? ld_elem<true>(a.gamma, k) : ld_elem<false>(a.gamma, k)); };
        auto sum_r = [&](size_t k) {
            float r = ld_elem<XB>(a.x, xo + k);
            if (a.res) r += ld_elem<XB>(a.res, ro + k);
            return XB ? apus_bf16_rne(r) : r;
        };
        double ss = 0.0, pm = 0.0;
        for (size_t k = tid; k < K; k += 256) {
            const float r = sum_r(k);
            if (a.res_out) st_elem<XB>(a.res_out, ro + k, r);
            const double d = r;
            ss = fma(d, d, ss);
            pm = fmax(pm, fabs(d * gam(k)));
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            ss += __shfl_xor(ss, o, 64);
            pm = fmax(pm, __shfl_xor(pm, o, 64));
        }
        if (lane == 0) {
            red[0][wave] = ss;
            red[1][wave] = pm;
        }
        __syncthreads();                       /* res_out written too */
        ss = ((red[0][0] + red[0][1]) + red[0][2]) + red[0][3];
        pm = fmax(fmax(red[1][0], red[1][1]), fmax(red[1][2], red[1][3]));
        const bool bad = !(ss < __builtin_inf());
        const double v = 1.0 / sqrt(ss / (double)a.K + (double)a.eps);
        auto norm = [&](size_t k) {
            const float r = a.res_out ? ld_elem<XB>(a.res_out, ro + k) : sum_r(k);
            const float y = (float)(((double)r * gam(k)) * v);
            if (a.y) st_elem<YB>(a.y, ro + k, a.round_y ? apus_bf16_rne(y) : y);
            return apus_bf16_rne(y);
        };
        if (!a.codes) {
            for (size_t k = tid; k < K; k += 256) norm(k);
        } else if (a.q_i8) {
            float scale, inv;
            apus_i8_scale(bad ? __builtin_inff() : apus_bf16_rne((float)(pm * v)), scale, inv);
            for (size_t k = tid; k < K; k += 256) a.codes[ro + k] = (uint8_t)(int8_t)apus_i8_code(norm(k), inv);
            if (tid == 0) a.scales[m] = scale;
        } else {
            const int nab = a.K >> 7;
            for (int b = wave; b < nab; b += 4) {
                const size_t k = (size_t)b * 128 + lane * 2;
                const float h0 = norm(k), h1 = norm(k + 1);
                const float amax = apus_wave_max(fmaxf(fabsf(h0), fabsf(h1)));
                const uint32_t e = bad ? 255u : apus_act_scale_exp(amax);
                const float inv = apus_inv_pow2_from_exp(e);
                const uint32_t c = bad ? 0u : apus_e4m3_pack2_hw(h0 * inv, h1 * inv);
                a.codes[ro + k] = (uint8_t)c;
                a.codes[ro + k + 1] = (uint8_t)(c >> 8);
                if (lane == 0) a.scales[m * nab + b] = apus_pow2_from_exp(e);
            }
        }
        __syncthreads();                   /* red is free again */
    }
}

/* rows of a launch with a workgroup each; more are looped over */
constexpr int ROWS_MAX = 1 << 20;

/* Eight neighbouring elements at any element's alignment (the vector unit takes
 * 16-byte accesses at any address). */
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

/* two values to BF16 bits, ties to even (a lower) */
__device__ __forceinline__ unsigned pk_bf16(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ float lo_bf16(unsigned u) { return apus_u2f(u << 16); }
__device__ __forceinline__ float hi_bf16(unsigned u) { return apus_u2f(u & 0xffff0000u); }

template <bool BF>
struct Raw8 {                                   /* loaded, not yet unpacked */
    u4_any u;
    f4_any f[2];
    __device__ __forceinline__ void load(const void *p, size_t i) {
        if constexpr (BF) {
            u = *(const APUS_GLOBAL u4_any *)((const uint16_t *)p + i);
        } else {
            f[0] = *(const APUS_GLOBAL f4_any *)((const float *)p + i);
            f[1] = *(const APUS_GLOBAL f4_any *)((const float *)p + i + 4);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if constexpr (BF) v[j] = j & 1 ? hi_bf16(u[j >> 1]) : lo_bf16(u[j >> 1]);
            else              v[j] = f[j >> 2][j & 3];
    }
};
template <bool BF>
__device__ __forceinline__ void store8(void *p, size_t i, const float (&v)[8]) {
    if constexpr (BF) {
        *(APUS_GLOBAL u4_any *)((uint16_t *)p + i) =
            u4_any{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])};
    } else {
        *(APUS_GLOBAL f4_any *)((float *)p + i) = f4_any{v[0], v[1], v[2], v[3]};
        *(APUS_GLOBAL f4_any *)((float *)p + i + 4) = f4_any{v[4], v[5], v[6], v[7]};
    }
}

/* bytes of four integer codes: b inv, rounded to an integer (ties to even) by the
 * addition of 1.5 * 2^23, whose low byte then is the code; |b inv| < 128 */
__device__ __forceinline__ unsigned pk_i8(float a, float b, float c, float d, float inv) {
    const float m = 12582912.0f;
    const unsigned p = apus_f2u(a * inv + m), q = apus_f2u(b * inv + m), r = apus_f2u(c * inv + m), s = apus_f2u(d * inv + m);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(s, r, 0x0c0c0400u), __builtin_amdgcn_perm(q, p, 0x0c0c0400u), 0x05040100u);
}

/*
 * Rows of 8 to 8 C TPR elements: TPR threads a row (16 or 32: several rows a wave), 8
 * neighbouring elements a thread and chunk, the row and the thread's part of gamma in registers, rows in a stride.
 * A chunk past the row's end, or over it where K is no multiple of 8, is the row's
 * last 8 elements again: they are left out of the sum, and what is stored twice is
 * the same. Every store comes after the barrier behind all loads of the row, so
 * arrays may be updated in place.
 */
template <int TPR, int C, bool XB, bool YB>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void apus_rmsnorm_kernel(ApusNormArgs a) {
    constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR, NWR = (TPR + 63) / 64, HALF = TPR < 64 ? TPR / 2 : 32;
    const int tid = threadIdx.x % TPR, lane = threadIdx.x & 63, wr = tid >> 6;
    const int K = a.K;
    __shared__ double lss[2][NWR];
    __shared__ unsigned lmx[2][NWR];
    float gm[C][8];
    int k0[C], dup[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k = (c * TPR + tid) * 8;
        k0[c] = min(k, K - 8);
        dup[c] = k - k0[c];
        if (a.gamma_bf16) {
            Raw8<true> g;
            g.load(a.gamma, k0[c]);
            g.get(gm[c]);
        } else {
            Raw8<false> g;
            g.load(a.gamma, k0[c]);
            g.get(gm[c]);
        }
    }
    const bool ragged = K & 7;
    int flip = 0;
    for (size_t m = (size_t)blockIdx.x * RPB + threadIdx.x / TPR; m < (size_t)a.M; m += (size_t)gridDim.x * RPB) {
        const size_t xo = m * (size_t)a.ldx, ro = m * (size_t)K;
        /* gamma stays in fp32: taken to 64 bits before the loop it would need twice the registers */
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) asm("" : "+v"(gm[c][j]));
        float r[C][8];
        {
            Raw8<XB> rx[C], rr[C];
#pragma unroll
            for (int c = 0; c < C; ++c) rx[c].load(a.x, xo + k0[c]);
            if (a.res) {
#pragma unroll
                for (int c = 0; c < C; ++c) rr[c].load(a.res, ro + k0[c]);
            }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                rx[c].get(r[c]);
                if (a.res) {
                    float t[8];
                    rr[c].get(t);
#pragma unroll
                    for (int j = 0; j < 8; ++j) r[c][j] += t[j];
                    if constexpr (XB) {
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const unsigned u = pk_bf16(r[c][j], r[c][j + 1]);
                            r[c][j] = lo_bf16(u);
                            r[c][j + 1] = hi_bf16(u);
                        }
                    }
                }
            }
        }
        double ss = 0.0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            double s = 0.0;
            if (ragged) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double d = j >= dup[c] ? r[c][j] : 0.0f;
                    s = fma(d, d, s);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double d = r[c][j];
                    s = fma(d, d, s);
                }
                s = dup[c] ? 0.0 : s;
            }
            ss += s;
        }
#pragma unroll
        for (int o = HALF; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
        if constexpr (NWR > 1) {
            if (lane == 0) lss[flip][wr] = ss;
            __syncthreads();
            ss = lss[flip][0];
#pragma unroll
            for (int w = 1; w < NWR; ++w) ss += lss[flip][w];
        }
        const bool bad = !(ss < __builtin_inff());
        const double v = 1.0 / sqrt(ss / (double)K + (double)a.eps);
        if (a.res_out) {
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (dup[c] < 8) store8<XB>(a.res_out, ro + k0[c], r[c]);
        }
        unsigned b[C][4], mx = 0;                /* bf16(y), two a word */
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[c][j] = (float)(((double)r[c][j] * (double)gm[c][j]) * v);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[c][j] = pk_bf16(r[c][2 * j], r[c][2 * j + 1]);
            if (a.y && dup[c] < 8) {
                if constexpr (YB) {
                    *(APUS_GLOBAL u4_any *)((uint16_t *)a.y + ro + k0[c]) = u4_any{b[c][0], b[c][1], b[c][2], b[c][3]};
                } else {
                    if (a.round_y) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) r[c][j] = j & 1 ? hi_bf16(b[c][j >> 1]) : lo_bf16(b[c][j >> 1]);
                    }
                    store8<false>(a.y, ro + k0[c], r[c]);
                }
            }
        }
        if (!a.codes) {
            flip ^= 1;
            continue;
        }
        if (a.q_i8) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) mx = max(mx, max(b[c][j] & 0x7fffu, (b[c][j] >> 16) & 0x7fffu));
#pragma unroll
            for (int o = HALF; o >= 1; o >>= 1) mx = max(mx, (unsigned)__shfl_xor((int)mx, o, 64));
            if constexpr (NWR > 1) {
                if (lane == 0) lmx[flip][wr] = mx;
                __syncthreads();
                mx = lmx[flip][0];
#pragma unroll
                for (int w = 1; w < NWR; ++w) mx = max(mx, lmx[flip][w]);
            }
            float scale, inv;
            apus_i8_scale(bad ? __builtin_inff() : apus_u2f(mx << 16), scale, inv);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                u2_any q;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    q[h] = bad ? 0u : pk_i8(lo_bf16(b[c][2 * h]), hi_bf16(b[c][2 * h]), lo_bf16(b[c][2 * h + 1]), hi_bf16(b[c][2 * h + 1]), inv);
                if (dup[c] < 8) *(APUS_GLOBAL u2_any *)(a.codes + ro + k0[c]) = q;
            }
            if (tid == 0) a.scales[m] = scale;
        } else {
            const int nab = K >> 7;
#pragma unroll
            for (int c = 0; c < C; ++c) {        /* a group of 128: 16 lanes */
                unsigned g = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) g = max(g, max(b[c][j] & 0x7fffu, (b[c][j] >> 16) & 0x7fffu));
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) g = max(g, (unsigned)__shfl_xor((int)g, o, 64));
                const uint32_t e = bad ? 255u : apus_act_scale_exp(apus_u2f(g << 16));
                const float inv = apus_inv_pow2_from_exp(e);
                u2_any q;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    q[h] = bad ? 0u : apus_e4m3_pack4_hw(lo_bf16(b[c][2 * h]) * inv, hi_bf16(b[c][2 * h]) * inv,
                                                         lo_bf16(b[c][2 * h + 1]) * inv, hi_bf16(b[c][2 * h + 1]) * inv);
                if (!dup[c]) {
                    *(APUS_GLOBAL u2_any *)(a.codes + ro + k0[c]) = q;
                    if ((lane & 15) == 0) a.scales[m * nab + (k0[c] >> 7)] = apus_pow2_from_exp(e);
                }
            }
        }
        flip ^= 1;
    }
}

/* Threads a row and chunks a thread (us, BF16 in and out, residual, y and codes, one row /
 * 512 / 8192 rows unless said):
 *   K = 44     (25011 rows, fp32, codes alone) 16 x 1 5.6   32 x 1 8.8   64 x 1 14.8
 *   K = 128    16 x 1  2.4 / -   / 4.3     32 x 1   2.4 / -   / 5.0     64 x 1   2.5 / -   / 7.4
 *   K = 256    32 x 1  2.4 / -   / 6.8     64 x 1   2.4 / -   / 8.8     16 x 2   2.8 / -   / 6.6
 *   K = 512    64 x 1  2.4 / 3.1 / 11.7    64 x 2   2.9 / 3.5 / 12.9    256 x 1  2.7 / 3.7 / 22.9
 *   K = 1024   64 x 2  2.9 / 3.9 / 18.4    64 x 4   4.1 / 5.1 / 24.8    256 x 1  2.8 / 4.0 / 25.1
 *   K = 2048   256 x 1 2.8 / 4.7 / 31.3    64 x 4   4.1 / 5.7 / 32.5    256 x 2  3.2 / 5.3 / 38.9
 *   K = 4096   512 x 1 2.9 / 6.9           256 x 2  3.3 / 7.0    1024 x 1  3.8 / 9.9
 *              1024 rows 11.7 / 10.8 / 17.4, 16384 rows 123 / 108
 *   K = 8192   512 x 2 3.9 / 11.3          256 x 4  4.3 / 11.5   1024 x 1  4.4 / 13.9
 *   K = 16384  512 x 4 5.5 / 22.1 / 4096 rows 130               256 x 8  7.0 / 24.8 / 146
 * A row a workgroup (or wave): 16384 rows of 4096 108 us, 604 MB at 5.6 TB/s, where a copy
 * of 1 GiB moves 5.1; in rounds of 2048 workgroups 116. Bound by HBM; of few rows by the
 * launch and the latency of load, sum and store after each other. */
template <bool XB, bool YB>
hipError_t apus_launch_rmsnorm_t(const ApusNormArgs &a, hipStream_t st) {
    auto go = [&](auto kernel, int nt, int rows) {
        hipLaunchKernelGGL(kernel, dim3(std::min((a.M + rows - 1) / rows, ROWS_MAX)), dim3(nt), 0, st, a);
        return hipGetLastError();
    };
    if (a.K < 8 || a.K > 16384) return go(apus_rmsnorm_any_kernel<XB, YB>, 256, 1);
    if (a.K <= 128)  return go(apus_rmsnorm_kernel<16, 1, XB, YB>, 256, 16);
    if (a.K <= 256)  return go(apus_rmsnorm_kernel<32, 1, XB, YB>, 256, 8);
    if (a.K <= 512)  return go(apus_rmsnorm_kernel<64, 1, XB, YB>, 256, 4);
    if (a.K <= 1024) return go(apus_rmsnorm_kernel<64, 2, XB, YB>, 256, 4);
    if (a.K <= 2048) return go(apus_rmsnorm_kernel<256, 1, XB, YB>, 256, 1);
    if (a.K <= 4096) return a.M <= 768 ? go(apus_rmsnorm_kernel<512, 1, XB, YB>, 512, 1) : go(apus_rmsnorm_kernel<256, 2, XB, YB>, 256, 1);
    if (a.K <= 8192) return go(apus_rmsnorm_kernel<512, 2, XB, YB>, 512, 1);
    return go(apus_rmsnorm_kernel<512, 4, XB, YB>, 512, 1);
}

hipError_t apus_launch_rmsnorm(const ApusNormArgs *a, hipStream_t st) {
    if (a->M <= 0) return hipSuccess;
    return a->x_bf16 ? (a->y_bf16 ? apus_launch_rmsnorm_t<true, true>(*a, st) : apus_launch_rmsnorm_t<true, false>(*a, st))
                     : (a->y_bf16 ? apus_launch_rmsnorm_t<false, true>(*a, st) : apus_launch_rmsnorm_t<false, false>(*a, st));
}

/* Integer codes of very short and very long rows, a workgroup a row. The maximum is
 * taken over the bits of |b|, where NaN lies above infinity. */
template <bool XB>
__global__ __launch_bounds__(256) void apus_i8_quant_any_kernel(const void *__restrict__ x, int M, int K,
                                                                int8_t *__restrict__ codes,
                                                                float *__restrict__ scales) {
    const int tid = threadIdx.x;
    __shared__ unsigned red[4];
    /* 64 bits: up to ROWS_MAX rows further, an int may pass its end */
    for (size_t row = blockIdx.x; row < (size_t)M; row += gridDim.x) {
        const size_t off = row * K;
        unsigned m = 0;
        for (int k = tid; k < K; k += 256)
            m = max(m, apus_f2u(apus_bf16_rne(ld_elem<XB>(x, off + k))) & 0x7fffffffu);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
        if ((tid & 63) == 0) red[tid >> 6] = m;
        __syncthreads();
        float scale, inv;
        apus_i8_scale(apus_u2f(max(max(red[0], red[1]), max(red[2], red[3]))), scale, inv);
        for (int k = tid; k < K; k += 256)
            codes[off + k] = (int8_t)apus_i8_code(apus_bf16_rne(ld_elem<XB>(x, off + k)), inv);
        if (tid == 0) scales[row] = scale;
        __syncthreads();                   /* red is free again */
    }
}

/* Rows of 8 to 8 C TPR elements, held as in apus_rmsnorm_kernel. */
template <int TPR, int C, bool XB>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void apus_i8_quant_kernel(const void *__restrict__ x, int M, int K,
                                                                              int8_t *__restrict__ codes,
                                                                              float *__restrict__ scales) {
    constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR, NWR = (TPR + 63) / 64, HALF = TPR < 64 ? TPR / 2 : 32;
    const int tid = threadIdx.x % TPR, lane = threadIdx.x & 63, wr = tid >> 6;
    __shared__ unsigned lmx[2][NWR];
    int flip = 0;
    for (size_t m = (size_t)blockIdx.x * RPB + threadIdx.x / TPR; m < (size_t)M; m += (size_t)gridDim.x * RPB) {
        const size_t ro = m * (size_t)K;
        Raw8<XB> rx[C];
        unsigned b[C][4], mx = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) rx[c].load(x, ro + min((c * TPR + tid) * 8, K - 8));
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float v[8];
            rx[c].get(v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                b[c][j] = pk_bf16(v[2 * j], v[2 * j + 1]);
                mx = max(mx, max(b[c][j] & 0x7fffu, (b[c][j] >> 16) & 0x7fffu));
            }
        }
#pragma unroll
        for (int o = HALF; o >= 1; o >>= 1) mx = max(mx, (unsigned)__shfl_xor((int)mx, o, 64));
        if constexpr (NWR > 1) {
            if (lane == 0) lmx[flip][wr] = mx;
            __syncthreads();
            mx = lmx[flip][0];
#pragma unroll
            for (int w = 1; w < NWR; ++w) mx = max(mx, lmx[flip][w]);
        }
        const bool bad = mx >= 0x7f80u;
        float scale, inv;
        apus_i8_scale(apus_u2f(mx << 16), scale, inv);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int k = (c * TPR + tid) * 8, k0 = min(k, K - 8);
            u2_any q;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                q[h] = bad ? 0u : pk_i8(lo_bf16(b[c][2 * h]), hi_bf16(b[c][2 * h]), lo_bf16(b[c][2 * h + 1]), hi_bf16(b[c][2 * h + 1]), inv);
            if (k - k0 < 8) *(APUS_GLOBAL u2_any *)((uint8_t *)codes + ro + k0) = q;
        }
        if (tid == 0) scales[m] = scale;
        flip ^= 1;
    }
}

template <bool XB>
hipError_t apus_launch_i8_quant_t(const void *x, int M, int K, int8_t *codes, float *scales, hipStream_t st) {
    auto go = [&](auto kernel, int nt, int rows) {
        hipLaunchKernelGGL(kernel, dim3(std::min((M + rows - 1) / rows, ROWS_MAX)), dim3(nt), 0, st, x, M, K, codes, scales);
        return hipGetLastError();
    };
    if (K < 8 || K > 16384) return go(apus_i8_quant_any_kernel<XB>, 256, 1);
    if (K <= 128)  return go(apus_i8_quant_kernel<16, 1, XB>, 256, 16);
    if (K <= 256)  return go(apus_i8_quant_kernel<32, 1, XB>, 256, 8);
    if (K <= 512)  return go(apus_i8_quant_kernel<64, 1, XB>, 256, 4);
    if (K <= 1024) return go(apus_i8_quant_kernel<64, 2, XB>, 256, 4);
    if (K <= 2048) return go(apus_i8_quant_kernel<256, 1, XB>, 256, 1);
    if (K <= 4096) return go(apus_i8_quant_kernel<256, 2, XB>, 256, 1);
    if (K <= 8192) return go(apus_i8_quant_kernel<512, 2, XB>, 512, 1);
    return go(apus_i8_quant_kernel<512, 4, XB>, 512, 1);
}

hipError_t apus_launch_i8_quant(const void *x, int x_bf16, int M, int K, int8_t *codes, float *scales,
                                hipStream_t st) {
    if (M <= 0) return hipSuccess;
    return x_bf16 ? apus_launch_i8_quant_t<true>(x, M, K, codes, scales, st) : apus_launch_i8_quant_t<false>(x, M, K, codes, scales, st);
}
