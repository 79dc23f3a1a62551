/*
 * apus_route.hip — expert choice from router logits: scores, balance bias,
 * groups, top-k, weights (the form of the routed dispatch's idx / wgt).
 *
 * For a token's logits z[0..E): p = 1 / (1 + exp(-z)), exp(z - max) / sum, or
 * sqrt(log(1 + exp z)); sel = p + bias; with groups, a group's score is the sum
 * of its one or two largest sel and only the keep best groups take part; the
 * topk largest sel are chosen, ties to the lowest index, w = p / (sum of the
 * chosen p) * scale. Selection goes by 64-bit values: in fp32 two experts whose
 * scores differ by less than a rounding would be chosen by whichever way the
 * exponential was rounded.
 *
 * Masked experts (logit or bias -inf or NaN) come after all others, lowest index
 * first, with weight 0; a weight sum of zero gives zeros.
 */
#include "apus_device.h"
#include "apus_internal.h"

#include <algorithm>

namespace {

__device__ __forceinline__ double score_at(int kind, double z, double zmax, double inv_sum) {
    if (kind == APUS_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-z));
    if (kind == APUS_SCORE_SOFTMAX) return exp(z - zmax) * inv_sum;
    return sqrt(fmax(z, 0.0) + log1p(exp(-fabs(z))));
}

/* logit as it is read: NaN masks like -inf, +inf is the largest number */
__device__ __forceinline__ float logit_of(float z) {
    return z != z ? -__builtin_inff() : fminf(z, 3.402823466e38f);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

}  // namespace

/* One wave a token; expert e = 64 i + lane. LDS: sel of every expert. */
template <int NE>
__global__ __launch_bounds__(256) void apus_route_kernel(ApusRouteArgs a) {
    extern __shared__ __align__(16) double sel_all[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int E = a.E;
    double *sel = sel_all + wave * (NE * 64);
    const double NINF = -__builtin_inf();
    for (size_t t = (size_t)blockIdx.x * 4 + wave; t < (size_t)a.s; t += (size_t)gridDim.x * 4) {
        const float *zr = a.logits + t * E;
        float z[NE];
        float zm = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = 64 * i + lane;
            z[i] = e < E ? logit_of(zr[e]) : -__builtin_inff();
            zm = fmaxf(zm, z[i]);
        }
        zm = apus_wave_max(zm);
        double inv_sum = 0.0;
        if (a.score == APUS_SCORE_SOFTMAX && zm > -__builtin_inff()) {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < NE; ++i) sum += z[i] > -__builtin_inff() ? exp((double)z[i] - (double)zm) : 0.0;
            inv_sum = 1.0 / wave_sum_f64(sum);
        }
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = 64 * i + lane;
            double p = 0.0, s = NINF;
            if (z[i] > -__builtin_inff()) {
                p = score_at(a.score, z[i], zm, inv_sum);
                s = p;
                if (a.bias) {
                    const float b = a.bias[e];
                    s = b == b ? p + (double)b : NINF;
                }
            }
            if (a.scores && e < E) a.scores[t * E + e] = (float)p;
            sel[e] = s;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       /* the wave's own LDS writes */
        bool keep_me = true;
        if (a.groups > 1) {
            const int per = E / a.groups;
            double best = NINF;
            if (lane < a.groups) {
                double m1 = NINF, m2 = NINF;
                for (int j = 0; j < per; ++j) {
                    const double v = sel[lane * per + j];
                    m2 = v > m1 ? m1 : fmax(m2, v);
                    m1 = fmax(m1, v);
                }
                best = a.group_top == 2 && m2 > NINF ? m1 + m2 : m1;
            }
            int rank = 0;
            for (int g = 0; g < a.groups; ++g) {
                const double o = __shfl(best, g, 64);
                rank += o > best || (o == best && g < lane) ? 1 : 0;
            }
            keep_me = lane < a.groups && rank < a.keep;
        }
        const uint64_t kept = __ballot(keep_me);
        /* taken: this lane's experts that are out of the running */
        unsigned taken = 0;
        double v[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = 64 * i + lane;
            v[i] = sel[e];
            const int grp = a.groups > 1 && e < E ? e / (E / a.groups) : 0;
            if (e >= E || !((kept >> grp) & 1)) taken |= 1u << i;
        }
        int mine = 0;
        for (int j = 0; j < a.topk; ++j) {
            double bv = NINF;
            int be = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const int e = 64 * i + lane;
                if (!((taken >> i) & 1) && (v[i] > bv || be == 0x7fffffff)) {
                    bv = v[i];
                    be = e;
                }
            }
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) {
                const double ov = __shfl_xor(bv, o, 64);
                const int oe = __shfl_xor(be, o, 64);
                if (oe != 0x7fffffff && (be == 0x7fffffff || ov > bv || (ov == bv && oe < be))) {
                    bv = ov;
                    be = oe;
                }
            }
            if ((be & 63) == lane) taken |= 1u << (be >> 6);
            if (lane == j) mine = be;
        }
        /* lane j < topk: expert mine; p again from its logit */
        const bool act = lane < a.topk;
        double p = 0.0;
        if (act && sel[mine] > NINF) p = score_at(a.score, logit_of(zr[mine]), zm, inv_sum);
        double w = p;
        if (a.renorm) {
            double sum = 0.0;
            for (int j = 0; j < a.topk; ++j) sum += __shfl(p, j, 64);
            w = sum > 0.0 ? p / sum : 0.0;
        }
        if (act) {
            a.idx[t * a.topk + lane] = mine;
            a.wgt[t * a.topk + lane] = (float)(w * (double)a.route_scale);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   /* sel read before the next token's */
    }
}

hipError_t apus_launch_route(const ApusRouteArgs *a, hipStream_t st) {
    if (a->s <= 0) return hipSuccess;
    if (a->E <= 0 || a->E > 1024 || a->topk <= 0 || a->topk > 16 || a->topk > a->E) return hipErrorInvalidValue;
    const int ne = (a->E + 63) / 64;
    auto go = [&](auto kernel, int n) {
        hipLaunchKernelGGL(kernel, dim3(std::min((int)(((size_t)a->s + 3) / 4), 1 << 20)), dim3(256), n * 64 * 4 * sizeof(double), st, *a);
        return hipGetLastError();
    };
    return ne <= 1 ? go(apus_route_kernel<1>, 1) : ne <= 2 ? go(apus_route_kernel<2>, 2) : ne <= 4 ? go(apus_route_kernel<4>, 4)
         : ne <= 8 ? go(apus_route_kernel<8>, 8) : go(apus_route_kernel<16>, 16);
}
