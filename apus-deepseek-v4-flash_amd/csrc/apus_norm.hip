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
 * roundings are monotone, so a row's max |b| is b of its max |r gamma|, known
 * with the sum: one reduction a row, not two.
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

/* One workgroup a row, any K and alignment: a pass for the sum, a pass for the
 * outputs, which reads r back from res_out (or forms it again). */
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

hipError_t apus_launch_rmsnorm(const ApusNormArgs *a, hipStream_t st) {
    if (a->M <= 0) return hipSuccess;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(std::min(a->M, ROWS_MAX)), dim3(256), 0, st, *a);
        return hipGetLastError();
    };
    return a->x_bf16 ? (a->y_bf16 ? go(apus_rmsnorm_any_kernel<true, true>) : go(apus_rmsnorm_any_kernel<true, false>))
                     : (a->y_bf16 ? go(apus_rmsnorm_any_kernel<false, true>) : go(apus_rmsnorm_any_kernel<false, false>));
}

/* Integer codes of rows, any K and alignment: one workgroup a row. The maximum
 * is taken over the bits of |b|, where NaN lies above infinity. */
template <bool XB>
__global__ __launch_bounds__(256) void apus_i8_quant_any_kernel(const void *__restrict__ x, int M, int K,
                                                                int8_t *__restrict__ codes,
                                                                float *__restrict__ scales) {
    const int tid = threadIdx.x;
    __shared__ unsigned red[4];
    for (int row = blockIdx.x; row < M; row += gridDim.x) {
        const size_t off = (size_t)row * K;
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

hipError_t apus_launch_i8_quant(const void *x, int x_bf16, int M, int K, int8_t *codes, float *scales,
                                hipStream_t st) {
    if (M <= 0) return hipSuccess;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(std::min(M, ROWS_MAX)), dim3(256), 0, st, x, M, K, codes, scales);
        return hipGetLastError();
    };
    return x_bf16 ? go(apus_i8_quant_any_kernel<true>) : go(apus_i8_quant_any_kernel<false>);
}
