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
 * Evaluating E 64-bit exponentials a token costs several times the reading of its
 * logits, and nearly always fp32 tells the same. So a token is chosen from fp32
 * scores whose error is bounded (2^-21 of p), and where two neighbours of the order
 * that decides it (the topk + 1 largest, the groups' scores) are not further apart
 * than that error allows, it is chosen again from 64-bit ones. The weights come from
 * 64-bit p of the chosen experts.
 *
 * Masked experts (logit or bias -inf or NaN) come after all others, lowest index
 * first, with weight 0; a weight sum of zero gives zeros.
 */
#include "apus_device.h"
#include "apus_internal.h"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace {

constexpr float F_NINF = -__builtin_inff();

/* A score's error goes by the score. Known of it in value v = p + bias is p <= |v| + the largest
 * |bias|: good where all biases are small, but one expert switched off by a bias of -1e9 would
 * leave every token undecided (8192 x 256, sigmoid: 31.6 us for 7.9). Sigmoid and softmax end at 1;
 * with a bias beyond this sqrt-softplus takes the largest score of the row too, which costs a
 * reduction a token. */
constexpr float APUS_LARGE_BIAS = 16.0f;

/* logit as it is read: NaN masks like -inf, +inf is the largest number */
__device__ __forceinline__ float logit_of(float z) { return z != z ? F_NINF : fminf(z, 3.402823466e38f); }

/* p without the softmax's sum */
template <int KIND>
__device__ __forceinline__ double score64(float z, float zmax) {
    if constexpr (KIND == APUS_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-(double)z));
    else if constexpr (KIND == APUS_SCORE_SOFTMAX) return exp((double)z - (double)zmax);
    else return sqrt(fmax((double)z, 0.0) + log1p(exp(-fabs((double)z))));
}

/* exp(a + b), |b| far below |a|: 2^t with t = a log2(e) rounded, times 1 + the rest of
 * the exponent; within 1.5 * 2^-23 (v_exp_f32 one step, the product half a step) */
__device__ __forceinline__ float exp32(float a, float b) {
    const float L = 1.44269504f, LL = 1.92596299e-8f;            /* log2(e) = L + LL */
    const float t = a * L, rest = fmaf(a, LL, fmaf(a, L, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, fmaf(rest, 0.693147181f, b), e);
}
/* p in fp32 (softmax: without the sum), within 2^-21: sigmoid 3.5 * 2^-23 (exponential,
 * sum, v_rcp_f32, product); sqrt-softplus 2.25 * 2^-23 (the library's exponential and
 * log1p, half of them after the root) */
template <int KIND>
__device__ __forceinline__ float score32(float z, float zmax) {
    if constexpr (KIND == APUS_SCORE_SIGMOID) {
        const float e = exp32(fmaxf(-fabsf(z), -150.0f), 0.0f);
        return (z < 0.0f ? e : 1.0f) * __builtin_amdgcn_rcpf(1.0f + e);
    } else if constexpr (KIND == APUS_SCORE_SOFTMAX) {
        /* z - zmax = d + r exactly */
        const float d = z - zmax, bb = d - z, r = (z - (d - bb)) + (-zmax - bb);
        return d < -150.0f ? 0.0f : exp32(d, r);
    } else {
        /* far below zero exp(z) leaves the range before its root does: there the root is
         * e^(z / 2) within e^z / 4 */
        return z < -20.0f ? exp32(fmaxf(0.5f * z, -150.0f), 0.0f) : sqrtf(fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z))));
    }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
template <int N>
__device__ __forceinline__ float ror(float v) {                   /* lane l: lane l - N of its row */
    return dpp<0x120 + N>(v);
}
template <int N>
__device__ __forceinline__ int ror(int v) { return __builtin_amdgcn_mov_dpp(v, 0x120 + N, 0xF, 0xF, true); }
template <int N>
__device__ __forceinline__ double ror(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)ror<N>((int)(uint32_t)u) | (uint64_t)(uint32_t)ror<N>((int)(u >> 32)) << 32);
}
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, ror<8>(v));
    v = fmaxf(v, ror<4>(v));
    v = fmaxf(v, ror<2>(v));
    return fmaxf(v, ror<1>(v));
}
__device__ __forceinline__ double row_sum(double v) {
    v += ror<8>(v);
    v += ror<4>(v);
    v += ror<2>(v);
    return v + ror<1>(v);
}
/* one step of a reduction over 16 lanes: with partners 1, 2, 4 and 8 lanes away, or their
 * mirror images, which hold the same */
template <int CTRL>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, true); }
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)dpp<CTRL>((int)(uint32_t)u) | (uint64_t)(uint32_t)dpp<CTRL>((int)(u >> 32)) << 32);
}
template <class T>
__device__ __forceinline__ T lane_of(T v, int l) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, l) |
                                         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), l) << 32);
    }
}
/* op over the wave, the same in every lane */
template <class T, class F>
__device__ __forceinline__ T wave_all(T v, F op) {
    v = op(v, ror<8>(v));
    v = op(v, ror<4>(v));
    v = op(v, ror<2>(v));
    v = op(v, ror<1>(v));
    return op(op(lane_of(v, 0), lane_of(v, 16)), op(lane_of(v, 32), lane_of(v, 48)));
}
/* the two largest of each `size` neighbouring lanes (size 1 .. 16), in all of them */
template <class T>
__device__ __forceinline__ void top2_lanes(T &m1, T &m2, int size) {
    auto step = [&](T b1, T b2) {
        const T lo = m1 < b1 ? m1 : b1, hi = m2 < b2 ? b2 : m2;
        m2 = lo < hi ? hi : lo;
        m1 = m1 < b1 ? b1 : m1;
    };
    if (size >= 2)  step(dpp<0xB1>(m1), dpp<0xB1>(m2));          /* quad_perm [1, 0, 3, 2] */
    if (size >= 4)  step(dpp<0x4E>(m1), dpp<0x4E>(m2));          /* quad_perm [2, 3, 0, 1] */
    if (size >= 8)  step(dpp<0x141>(m1), dpp<0x141>(m2));        /* row_half_mirror */
    if (size >= 16) step(dpp<0x140>(m1), dpp<0x140>(m2));        /* row_mirror */
}
/* f(1) .. f(15) as constants */
template <class F, int... I>
__device__ __forceinline__ void each_ror(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I + 1>{}), ...);
}
template <class F>
__device__ __forceinline__ void each_ror(F &&f) { each_ror(f, std::make_integer_sequence<int, 15>{}); }

/* LDS of a wave: the candidates of a token, the largest of them in order, the chosen
 * experts of the wave's tokens */
struct WaveLds {
    float2 cand[64], best[64];
    int chosen[64];
};

/* the wave's own LDS operations run in order; the compiler keeps them so */
__device__ __forceinline__ void wave_lds_order() { asm volatile("" ::: "memory"); }

constexpr int MASKED = 1 << 16;      /* beside an expert's number: it has no weight */

/* One token by 64-bit values; lane j < topk returns its expert. sel: LDS of E doubles. */
template <int KIND>
__device__ __forceinline__ int route_exact(const ApusRouteArgs &a, const float *zr, float zmax, double inv_sum, double *sel) {
    const int lane = threadIdx.x & 63, E = a.E;
    const double NINF = -__builtin_inf();
    for (int e = lane; e < E; e += 64) {
        const float z = logit_of(zr[e]);
        double s = NINF;
        if (z > F_NINF) {
            s = score64<KIND>(z, zmax);
            if constexpr (KIND == APUS_SCORE_SOFTMAX) s *= inv_sum;
            if (a.bias) s = a.bias[e] == a.bias[e] ? s + (double)a.bias[e] : NINF;
        }
        sel[e] = s;
    }
    wave_lds_order();
    const int per = E / a.groups, none = 0x7fffffff;
    uint64_t kept = ~0ull;                       /* bit: group */
    if (a.groups > 1) {
        double best = NINF;
        if (lane < a.groups) {
            double m1 = NINF, m2 = NINF;
#pragma unroll 8
            for (int j = 0; j < per; ++j) {
                const double v = sel[lane * per + j];
                m2 = v > m1 ? m1 : fmax(m2, v);
                m1 = fmax(m1, v);
            }
            best = a.group_top == 2 && m2 > NINF ? m1 + m2 : m1;
        }
        int rank = 0;
        for (int g = 0; g < a.groups; ++g) {
            const double o = lane_of(best, g);
            rank += o > best || (o == best && g < lane) ? 1 : 0;
        }
        kept = __ballot(lane < a.groups && rank < a.keep);
    }
    int mine = 0;
    unsigned taken = 0;                          /* bit i: expert 64 i + lane is out (E <= 1024) */
    for (int e = lane; e < E; e += 64)
        if (!((kept >> (a.groups > 1 ? e / per : 0)) & 1)) taken |= 1u << (e >> 6);
    for (int j = 0; j < a.topk; ++j) {
        double bv = NINF;
        int be = none;
#pragma unroll 4
        for (int e = lane; e < E; e += 64) {
            const double v = sel[e];
            if (!((taken >> (e >> 6)) & 1) && (be == none || v > bv)) {
                bv = v;
                be = e;
            }
        }
        const double top = wave_all(bv, [](double x, double y) { return fmax(x, y); });
        be = wave_all(bv == top ? be : none, [](int x, int y) { return min(x, y); });
        if ((be & 63) == lane) taken |= 1u << (be >> 6);
        if (lane == j) mine = be;
    }
    if (lane < a.topk && !(sel[mine] > NINF)) mine |= MASKED;
    wave_lds_order();
    return mine;
}

}  // namespace

/*
 * A wave takes `tpw` tokens one after the other, the next one's logits under way. Lane
 * (group, s) has NE experts of its group, lpg lanes a group (all 64 without groups): V,
 * neighbouring fours, loaded 16 bytes at a time; else every lpg-th. The order of a token:
 * a threshold that at least topk values reach (the least of the maxima, or of the second
 * largest where topk > 8, of topk or a few more runs of lanes); the values that reach
 * it, about 20 for topk 8, compacted through LDS, one a lane; their ranks by comparing
 * all with all. Where two neighbours are too close, the candidates (the threshold is
 * lowered by the error, so every expert that could be chosen is among them) are ranked
 * again by 64-bit values; where the groups' border is, the whole token (route_exact). The
 * weights of all the wave's tokens are worked out together at the end, a lane each.
 */
template <int KIND, int NE, bool V>
__global__ __launch_bounds__(256) void apus_route_kernel(ApusRouteArgs a, int lpg, int ne, int tpw, int slots) {
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr bool SOFTMAX = KIND == APUS_SCORE_SOFTMAX;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    WaveLds *w = reinterpret_cast<WaveLds *>(lds) + wave;
    double *sel64 = reinterpret_cast<double *>(lds + 4 * sizeof(WaveLds)) + wave * a.E;
    const int E = a.E, k = a.topk, per = E / a.groups, grp = lane / lpg, s0 = lane % lpg;
    const bool mine_ok = grp < a.groups;
    const int id0 = grp * per + (V ? 4 * s0 : s0);
    /* expert i of the lane; V: as many in every lane */
    auto id = [&](int i) { return id0 + (V ? 4 * lpg * (i >> 2) + (i & 3) : lpg * i); };
    auto has = [&](int i) { return mine_ok && (V ? i < ne : s0 + lpg * i < per); };
    auto load = [&](const float *zr, float (&z)[NE]) {
        if constexpr (V) {
#pragma unroll
            for (int i = 0; i < NE; i += 4) {
                float4 f = make_float4(F_NINF, F_NINF, F_NINF, F_NINF);
                if (has(i)) f = apus_gld<float4>(zr + id(i));
                z[i] = f.x; z[i + 1] = f.y; z[i + 2] = f.z; z[i + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i) z[i] = has(i) ? apus_gld<float>(zr + id(i)) : F_NINF;
        }
    };
    float bias[NE], bmax = 0.0f, zn[NE];
    size_t t0 = ((size_t)blockIdx.x * 4 + wave) * tpw;
    if (t0 < (size_t)a.s) load(a.logits + t0 * E, zn);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        bias[i] = 0.0f;
        if (a.bias && has(i)) {
            const float b = a.bias[id(i)];
            bias[i] = b == b ? b : F_NINF;
            if (fabsf(bias[i]) < __builtin_inff()) bmax = fmaxf(bmax, fabsf(bias[i]));
        }
    }
    bmax = apus_wave_max_dpp(bmax);
    /* the largest score that value v = p + bias may hold: |v| + bmax, which bounds it best where
     * the biases are small, and `top` */
    float top = 1.0f;
    auto reach = [&](float v, int n) { return fminf(v + n * bmax, n * top); };
    const bool sum_all = SOFTMAX && !a.renorm;
    const size_t step = (size_t)gridDim.x * 4 * tpw;
    for (; t0 < (size_t)a.s; t0 += step) {
        const int nt = (int)min((size_t)tpw, (size_t)a.s - t0);
        double my_inv_sum = 1.0;                                  /* of token lane / slots */
        float my_zmax = 0.0f;
        for (int tt = 0; tt < nt; ++tt) {
            const float *zr = a.logits + (t0 + tt) * E;
            float z[NE], v[NE], zmax = 0.0f;
#pragma unroll
            for (int i = 0; i < NE; ++i) z[i] = logit_of(zn[i]);
            const size_t tn = tt + 1 < nt ? t0 + tt + 1 : t0 + step;
            if (tn < (size_t)a.s) load(a.logits + tn * E, zn);
            double inv_sum = 1.0;
            if constexpr (SOFTMAX) {
                zmax = F_NINF;
#pragma unroll
                for (int i = 0; i < NE; ++i) zmax = fmaxf(zmax, z[i]);
                zmax = apus_wave_max_dpp(zmax);
            }
            /* 1 / the 64-bit sum of 64-bit terms (in a loop over memory: unrolled over the
             * registers it would need twice as many of them) */
            auto exact_inv = [&]() {
                double sum = 0.0;
#pragma unroll 1
                for (int e = lane; e < E; e += 64) {
                    const float x = logit_of(zr[e]);
                    sum += x > F_NINF ? score64<KIND>(x, zmax) : 0.0;
                }
                sum = wave_all(sum, [](double x, double y) { return x + y; });
                return sum > 0.0 ? 1.0 / sum : 0.0;
            };
            {
                float p[NE];
#pragma unroll
                for (int i = 0; i < NE; ++i) {
                    p[i] = z[i] > F_NINF ? score32<KIND>(z[i], zmax) : 0.0f;
                    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);    /* four at a time: fewer registers */
                }
                if constexpr (SOFTMAX) {
                    if (sum_all) {
                        inv_sum = exact_inv();
                    } else {
                        double sum = 0.0;
#pragma unroll
                        for (int i = 0; i < NE; ++i) sum += (double)p[i];
                        sum = wave_all(sum, [](double x, double y) { return x + y; });
                        inv_sum = sum > 0.0 ? 1.0 / sum : 0.0;
                    }
                    const float is = (float)inv_sum;
#pragma unroll
                    for (int i = 0; i < NE; ++i) p[i] *= is;
                }
                if (a.scores) {
                    float *sc = a.scores + (t0 + tt) * E;
                    if constexpr (V) {
#pragma unroll
                        for (int i = 0; i < NE; i += 4)
                            if (has(i)) apus_gst<apus_v4f>(sc + id(i), apus_v4f{p[i], p[i + 1], p[i + 2], p[i + 3]});
                    } else {
#pragma unroll
                        for (int i = 0; i < NE; ++i)
                            if (has(i)) apus_gst<float>(sc + id(i), p[i]);
                    }
                }
                if constexpr (KIND == APUS_SCORE_SQRTSOFTPLUS) {
                    top = __builtin_inff();
                    if (bmax > APUS_LARGE_BIAS) {
                        top = 0.0f;
#pragma unroll
                        for (int i = 0; i < NE; ++i) top = fmaxf(top, p[i]);
                        top = apus_wave_max_dpp(top);
                    }
                }
#pragma unroll
                for (int i = 0; i < NE; ++i) v[i] = z[i] > F_NINF ? p[i] + bias[i] : F_NINF;
            }
            /* the two largest of the lane */
            float m1 = F_NINF, m2 = F_NINF;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                m2 = __builtin_amdgcn_fmed3f(m1, m2, v[i]);
                m1 = fmaxf(m1, v[i]);
            }
            bool active = mine_ok, border = false;
            if (a.groups > 1) {
                float g1 = m1, g2 = m2;
                top2_lanes(g1, g2, lpg);
                const bool two = a.group_top == 2 && g2 > F_NINF;
                const float mine = two ? g1 + g2 : g1, mag = two ? fabsf(g1) + fabsf(g2) : fabsf(g1);
                int rank = 0;
                for (int g = 0; g < a.groups; ++g) {
                    const float o = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), g * lpg));
                    rank += o > mine ? 1 : 0;
                }
                /* the worst group kept less its error and the best one left out with its own;
                 * where they meet, or fewer or more than `keep` are kept (equal scores), the
                 * choice is not sure */
                if (a.keep < a.groups) {
                    const float err = fminf(0x1p-20f * reach(mag, 2) + 0x1p-22f * mag + 1e-36f, 3.402823466e38f);
                    const bool in = active && rank < a.keep;
                    const float lo = -apus_wave_max_dpp(in ? err - mine : F_NINF);
                    const float hi = apus_wave_max_dpp(active && !in ? mine + err : F_NINF);
                    border = __popcll(__ballot(in)) != a.keep * lpg || !(lo > hi);
                    active = active && rank < a.keep;
#pragma unroll
                    for (int i = 0; i < NE; ++i) v[i] = active ? v[i] : F_NINF;
                    m1 = active ? m1 : F_NINF;
                    m2 = active ? m2 : F_NINF;
                }
            }
            /* threshold: runs of lanes, at least k values in their (two) largest */
            const int lanes = a.groups > 1 ? a.keep * lpg : 64, of = k <= 8 ? lanes / k : 2 * lanes / k;
            float thr = F_NINF;
            if (of > 0) {
                float r1 = m1, r2 = m2;
                top2_lanes(r1, r2, of);
                thr = -apus_wave_max_dpp(active ? -(k <= 8 ? r1 : r2) : F_NINF);
                thr -= 0x1p-19f * reach(fabsf(thr), 1) + 0x1p-22f * fabsf(thr) + 1e-36f;
            }
            thr = fmaxf(thr, -3.402823466e38f);                   /* masked ones never */
            int n = 0;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const bool in = v[i] >= thr;
                const uint64_t mask = __ballot(in);
                const int pos = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                                               __builtin_amdgcn_mbcnt_lo((uint32_t)mask, n));
                if (in && pos < 64) w->cand[pos] = make_float2(v[i], __builtin_bit_cast(float, id(i)));
                n += __popcll(mask);
            }
            w->best[lane] = make_float2(__builtin_nanf(""), 0.0f);
            wave_lds_order();
            int e = 0;
            if (!border && n <= 64 && n >= k) {
                const float2 c = w->cand[lane];
                const float cv = lane < n ? c.x : F_NINF;
                const int ce = __builtin_bit_cast(int, c.y);
                int rank = 0;
#pragma unroll
                for (int b = 0; b < 64; b += 8) {                 /* lanes past n hold -inf */
                    if (b < n) {
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const float o = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, cv), b + q));
                            rank += o > cv ? 1 : 0;
                        }
                    }
                }
                if (lane < n && rank <= k) w->best[rank] = make_float2(cv, c.y);   /* of equal ones a slot stays NaN */
                wave_lds_order();
                const float sv = w->best[lane].x, nx = w->best[min(lane + 1, 63)].x;
                const bool last = lane == k - 1 && n == k;        /* none left that could be chosen */
                const bool apart = sv - nx > 0x1p-19f * reach(fabsf(sv), 1) + 0x1p-22f * fabsf(sv) + 1e-36f || (last && sv == sv);
                if (__any(lane < k && !apart)) {
                    double inv = inv_sum, s = -__builtin_inf();
                    if (SOFTMAX && !sum_all && a.bias) inv = exact_inv();          /* beside a bias the sum counts */
                    if (lane < n) {
                        s = score64<KIND>(logit_of(zr[ce]), zmax);
                        if constexpr (SOFTMAX) s *= inv;
                        if (a.bias) s += (double)a.bias[ce];
                    }
                    rank = 0;
                    for (int q = 0; q < n; ++q) {
                        const double o = __shfl(s, q, 64);
                        const int oe = __builtin_amdgcn_readlane(ce, q);
                        rank += o > s || (o == s && oe < ce) ? 1 : 0;
                    }
                    if (lane < n && rank < k) w->best[rank] = make_float2(cv, c.y);
                    wave_lds_order();
                }
                e = __builtin_bit_cast(int, w->best[lane].y);
            } else {
                double inv = inv_sum;
                if (SOFTMAX && !sum_all && a.bias) inv = exact_inv();
                e = route_exact<KIND>(a, zr, zmax, inv, sel64);
            }
            wave_lds_order();
            if (lane < k) w->chosen[tt * slots + lane] = e;
            if (SOFTMAX && lane / slots == tt) {
                my_inv_sum = inv_sum;
                my_zmax = zmax;
            }
        }
        wave_lds_order();
        /* lane: slot lane % slots of token lane / slots */
        const int tt = lane / slots, j = lane % slots;
        const bool act = tt < nt && j < k;
        const int e = act ? w->chosen[lane] : MASKED;
        double p = 0.0;
        if (!(e & MASKED)) p = score64<KIND>(logit_of(a.logits[(t0 + tt) * E + e]), my_zmax);
        double wt = sum_all ? p * my_inv_sum : p;
        if (a.renorm) {
            double sum = p;
            for (int o = 1; o < slots; o <<= 1) sum += __shfl_xor(sum, o, 64);
            wt = sum > 0.0 ? p / sum : 0.0;
        }
        if (act) {
            const size_t at = (t0 + tt) * k + j;
            a.idx[at] = e & (MASKED - 1);
            a.wgt[at] = (float)(wt * (double)a.route_scale);
        }
        wave_lds_order();
    }
}

/* --- four tokens a wave, a row of 16 lanes each (DPP moves stay inside a row) --- */

namespace {

/* p in fp32 from the bare instructions (softmax: without the sum): where no scores are
 * asked for, only its order counts. Absolute error, with x = |z| or zmax - z, exponents
 * within (x + 2) 2^-24 relative: sigmoid p (1 - p) (x + 2) 2^-24 + 2^-23 p < 2^-22;
 * softmax e^-x (2 x + 3) 2^-24 < 2^-22; sqrt-softplus 2^-22 / (2 p) + 1.25 * 2^-23 p, of
 * which the first is 2^-21 at most from p = 0.25 on, and 2^-12 at most below. */
template <int KIND>
__device__ __forceinline__ float quick32(float z, float zmax) {
    const float L = 1.44269504f;
    if constexpr (KIND == APUS_SCORE_SIGMOID) {
        return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -L));
    } else if constexpr (KIND == APUS_SCORE_SOFTMAX) {
        return __builtin_amdgcn_exp2f((z - zmax) * L);
    } else {
        const float e = __builtin_amdgcn_exp2f(fabsf(z) * -L);
        return __builtin_amdgcn_sqrtf(fmaf(__builtin_amdgcn_logf(1.0f + e), 0.693147181f, fmaxf(z, 0.0f)));
    }
}

struct RowLds {
    float2 cand[64], best[64];           /* [row][16] */
    int chosen[64];
};

}  // namespace

/*
 * topk <= 8, up to 16 experts a lane: lane s of a row has NE experts of group s / lpg
 * (V: neighbouring fours). As above but for the threshold: the topk-th largest of the
 * lanes' two largest values, found by comparing all 32 with each other; about topk + 1
 * experts reach it, a lane each behind their compaction.
 */
template <int KIND, int NE, bool V>
__global__ __launch_bounds__(256) void apus_route_row_kernel(ApusRouteArgs a, int lpg, int ne) {
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr bool SOFTMAX = KIND == APUS_SCORE_SOFTMAX;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = lane >> 4, l = lane & 15;
    RowLds *w = reinterpret_cast<RowLds *>(lds) + wave;
    double *sel64 = reinterpret_cast<double *>(lds + 4 * sizeof(RowLds)) + wave * a.E;
    const int E = a.E, k = a.topk, per = E / a.groups, grp = l / lpg, s0 = l % lpg;
    int id0 = grp * per + (V ? 4 * s0 : s0);
    auto id = [&](int i) { return id0 + (V ? 4 * lpg * (i >> 2) + (i & 3) : lpg * i); };
    auto has = [&](int i) { return V ? i < ne : s0 + lpg * i < per; };
    const bool sum_all = SOFTMAX && !a.renorm, norm = SOFTMAX && (!a.renorm || a.bias || a.scores);
    /* largest |bias| of the finite ones, and a bound of their largest: where |bias| is small the
     * former will do */
    float *lbias = reinterpret_cast<float *>(lds + 4 * sizeof(RowLds) + 4 * E * sizeof(double)), bmax = 0.0f, btop = 0.0f;
    if (a.bias) {
        for (int e = threadIdx.x; e < E; e += 256) lbias[e] = a.bias[e] == a.bias[e] ? a.bias[e] : F_NINF;
        __syncthreads();
        for (int e = lane; e < E; e += 64)
            if (fabsf(lbias[e]) < __builtin_inff()) bmax = fmaxf(bmax, fabsf(lbias[e]));
        btop = bmax = apus_wave_max_dpp(bmax);
        if (KIND == APUS_SCORE_SQRTSOFTPLUS && bmax > APUS_LARGE_BIAS) {
            btop = 0.0f;
            for (int e = lane; e < E; e += 64)
                if (lbias[e] < __builtin_inff()) btop = fmaxf(btop, lbias[e]);
            btop = apus_wave_max_dpp(btop);
        }
    }
    const size_t step = (size_t)gridDim.x * 16;
    for (size_t t0 = ((size_t)blockIdx.x * 4 + wave) * 4; t0 < (size_t)a.s; t0 += step) {
        /* worked out in each round: kept over all of them, the experts' numbers and addresses take 40
         * registers (32768 tokens, sqrt-softplus 26.6 us so, 20.6 without, sigmoid and groups
         * 23.6, 22.6; 64 tokens 6.1, 6.25). For a softmax in fours three waves a SIMD have
         * room for them (15.7, 16.1) */
        if constexpr (!(SOFTMAX && V)) asm volatile("" : "+v"(id0));
        const size_t t = min(t0 + row, (size_t)a.s - 1);
        const bool real = t0 + row < (size_t)a.s;
        const float *zr = a.logits + t * E;
        float z[NE], v[NE], zmax = 0.0f;
        if constexpr (V) {
#pragma unroll
            for (int i = 0; i < NE; i += 4) {
                float4 f = make_float4(F_NINF, F_NINF, F_NINF, F_NINF);
                if (has(i)) f = apus_gld<float4>(zr + id(i));
                z[i] = f.x; z[i + 1] = f.y; z[i + 2] = f.z; z[i + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i) z[i] = has(i) ? apus_gld<float>(zr + id(i)) : F_NINF;
        }
#pragma unroll
        for (int i = 0; i < NE; ++i) z[i] = logit_of(z[i]);
        if constexpr (SOFTMAX) {
            zmax = F_NINF;
#pragma unroll
            for (int i = 0; i < NE; ++i) zmax = fmaxf(zmax, z[i]);
            zmax = fmaxf(row_max(zmax), -3.402823466e38f);
        }
        /* 64-bit values in loops over memory: unrolled over the registers they would need
         * twice as many of them, in a path that hardly a token takes */
        auto exact_inv = [&]() {
            double sum = 0.0;
#pragma unroll 1
            for (int e = l; e < E; e += 16) {
                const float x = logit_of(zr[e]);
                sum += x > F_NINF ? score64<KIND>(x, zmax) : 0.0;
            }
            sum = row_sum(sum);
            return sum > 0.0 ? 1.0 / sum : 0.0;
        };
        double inv_sum = 1.0;
        if (a.scores) {
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                v[i] = z[i] > F_NINF ? score32<KIND>(z[i], zmax) : 0.0f;
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);        /* four at a time: fewer registers */
            }
        } else {
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                v[i] = quick32<KIND>(z[i], zmax);
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (norm) {
            if (sum_all) {
                inv_sum = exact_inv();
            } else {
                double sum = 0.0;
#pragma unroll
                for (int i = 0; i < NE; ++i) sum += (double)v[i];
                sum = row_sum(sum);
                inv_sum = sum > 0.0 ? 1.0 / sum : 0.0;
            }
            const float is = (float)inv_sum;
#pragma unroll
            for (int i = 0; i < NE; ++i) v[i] *= is;
        }
        if (a.scores && real) {
            float *sc = a.scores + t * E;
            if constexpr (V) {
#pragma unroll
                for (int i = 0; i < NE; i += 4)
                    if (has(i)) apus_gst<apus_v4f>(sc + id(i), apus_v4f{v[i], v[i + 1], v[i + 2], v[i + 3]});
            } else {
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if (has(i)) apus_gst<float>(sc + id(i), v[i]);
            }
        }
        /* as above: the largest score that v = p + bias may hold (sqrt-softplus alone asks) */
        float top = __builtin_inff();
        if (KIND == APUS_SCORE_SQRTSOFTPLUS && bmax > APUS_LARGE_BIAS) {
            top = 0.0f;
#pragma unroll
            for (int i = 0; i < NE; ++i) top = fmaxf(top, v[i]);
            top = row_max(top);
        }
        auto reach = [&](float v, int n) { return fminf(v + n * bmax, n * top); };
        if (a.bias) {
            if constexpr (V) {
#pragma unroll
                for (int i = 0; i < NE; i += 4)
                    if (has(i)) {
                        const float4 b = *reinterpret_cast<const float4 *>(lbias + id(i));
                        v[i] += b.x; v[i + 1] += b.y; v[i + 2] += b.z; v[i + 3] += b.w;
                    }
            } else {
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if (has(i)) v[i] += lbias[id(i)];
            }
        }
        /* the two largest of the lane */
        float m1 = F_NINF, m2 = F_NINF;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            v[i] = z[i] > F_NINF ? v[i] : F_NINF;
            m2 = fmaxf(m2, fminf(m1, v[i]));
            m1 = fmaxf(m1, v[i]);
        }
        bool whole = false, active = true;                        /* whole: the row's token by route_exact */
        if (a.groups > 1 && a.keep < a.groups) {
            float g1 = m1, g2 = m2;
            top2_lanes(g1, g2, lpg);
            const bool two = a.group_top == 2 && g2 > F_NINF;
            const float mine = two ? g1 + g2 : g1, mag = two ? fabsf(g1) + fabsf(g2) : fabsf(g1);
            int above = 0;                                        /* lpg times the groups above */
            each_ror([&](auto c) { above += ror<decltype(c)::value>(mine) > mine ? 1 : 0; });
            active = above < a.keep * lpg;
            /* a group's error: that of its values (as for tol below; the smaller one may be small
             * where the sum is not) and the roundings of three sums */
            float err = 0x1p-19f + 0x1p-22f * mag;
            if (KIND == APUS_SCORE_SQRTSOFTPLUS) err += 0x1p-21f * reach(mag, 2) + ((two ? g2 : g1) - btop < 0.25f ? 0x1p-10f : 0.0f);
            err = fminf(err, 3.402823466e38f);                    /* a sum of -inf stays that */
            const float lo = -row_max(active ? err - mine : F_NINF), hi = row_max(active ? F_NINF : mine + err);
            const int kept = __popc((uint32_t)(__ballot(active) >> (lane & 48)) & 0xffffu);
            const bool border = kept != a.keep * lpg || !(lo > hi);
            if (__any(border)) {                                  /* the groups by 64-bit values */
                const double NINF = -__builtin_inf(), inv = SOFTMAX && !sum_all && a.bias ? exact_inv() : inv_sum;
                double d1 = NINF, d2 = NINF;
#pragma unroll 1
                for (int i = s0; i < per; i += lpg) {
                    const int e = grp * per + i;
                    const float ze = logit_of(zr[e]), b = a.bias ? lbias[e] : 0.0f;
                    double x = NINF;
                    if (ze > F_NINF && b > F_NINF) {
                        x = score64<KIND>(ze, zmax);
                        if constexpr (SOFTMAX) x *= inv;
                        x += (double)b;
                    }
                    d2 = fmax(d2, fmin(d1, x));
                    d1 = fmax(d1, x);
                }
                top2_lanes(d1, d2, lpg);
                const double best = a.group_top == 2 && d2 > NINF ? d1 + d2 : d1;
                int ahead = 0;
                each_ror([&](auto c) {
                    const double o = ror<decltype(c)::value>(best);
                    const int og = ror<decltype(c)::value>(grp);  /* with every lane active */
                    ahead += o > best || (o == best && og < grp) ? 1 : 0;
                });
                active = border ? ahead < a.keep * lpg : active;
            }
            m1 = active ? m1 : F_NINF;
            m2 = active ? m2 : F_NINF;
        }
        /* threshold: the k-th of the lanes' two largest */
        int r1 = 0, r2 = m1 > m2 ? 1 : 0;
        each_ror([&](auto c) {
            const float x1 = ror<decltype(c)::value>(m1), x2 = ror<decltype(c)::value>(m2);
            r1 += x1 > m1 ? 1 : 0;
            r2 += x1 > m2 ? 1 : 0;
            r1 += x2 > m1 ? 1 : 0;
            r2 += x2 > m2 ? 1 : 0;
        });
        float thr = -row_max(fmaxf(r1 < k ? -m1 : F_NINF, r2 < k ? -m2 : F_NINF));
        /* Twice the error of value v = p + bias and of the sum's rounding. The constant part holds
         * for scores up to 1; those of sqrt-softplus have no upper end. Its scores that decide
         * may be small (p = v - bias) where the k-th value does not say otherwise */
        const float least = KIND == APUS_SCORE_SQRTSOFTPLUS && thr - btop < 0.25f ? 0x1p-10f : 0x1p-20f;
        auto tol = [&](float v) {
            const float t = least + 0x1p-22f * fabsf(v);
            return KIND == APUS_SCORE_SQRTSOFTPLUS ? t + 0x1.4p-21f * reach(fabsf(v), 1) : t;
        };
        thr = fmaxf(thr - tol(thr), -3.402823466e38f);            /* masked ones never */
        thr = active ? thr : __builtin_inff();
        int cnt = 0;
#pragma unroll
        for (int i = 0; i < NE; ++i) cnt += v[i] >= thr ? 1 : 0;
        int at = cnt;                                             /* sum up to this lane of the row */
        at += __builtin_amdgcn_update_dpp(0, at, 0x111, 0xF, 0xF, true);
        at += __builtin_amdgcn_update_dpp(0, at, 0x112, 0xF, 0xF, true);
        at += __builtin_amdgcn_update_dpp(0, at, 0x114, 0xF, 0xF, true);
        at += __builtin_amdgcn_update_dpp(0, at, 0x118, 0xF, 0xF, true);
        int n = max(at, ror<8>(at));
        n = max(n, ror<4>(n));
        n = max(n, ror<2>(n));
        n = max(n, ror<1>(n));
        at -= cnt;
        whole |= n > 16 || n < k;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (v[i] >= thr) {
                if (at < 16) w->cand[row * 16 + at] = make_float2(v[i], __builtin_bit_cast(float, id(i)));
                ++at;
            }
        w->best[lane] = make_float2(__builtin_nanf(""), 0.0f);
        wave_lds_order();
        const float2 c = w->cand[lane];
        const float cv = l < n ? c.x : F_NINF;
        const int ce = l < n ? __builtin_bit_cast(int, c.y) : 0;
        int rank = 0;
        each_ror([&](auto q) { rank += ror<decltype(q)::value>(cv) > cv ? 1 : 0; });
        if (l < n && rank <= k) w->best[row * 16 + rank] = make_float2(cv, __builtin_bit_cast(float, ce));
        wave_lds_order();                                         /* of equal ones a slot stays NaN */
        const float sv = w->best[lane].x, next = w->best[min(lane + 1, 63)].x;
        const bool last = l == k - 1 && n == k;                   /* none left that could be chosen */
        const bool apart = sv - next > tol(sv) || (last && sv == sv);
        if (__any(l < k && !apart && !whole)) {
            double inv = inv_sum;
            if (SOFTMAX && !sum_all && a.bias) inv = exact_inv(); /* beside a bias the sum counts */
            double s = -__builtin_inf();
            if (l < n) {
                s = score64<KIND>(logit_of(zr[ce]), zmax);
                if constexpr (SOFTMAX) s *= inv;
                if (a.bias) s += (double)a.bias[ce];
            }
            rank = 0;
            each_ror([&](auto q) {
                const double o = ror<decltype(q)::value>(s);
                const int oe = ror<decltype(q)::value>(ce);
                rank += o > s || (o == s && oe < ce) ? 1 : 0;
            });
            if (l < n && rank < k) w->best[row * 16 + rank] = make_float2(cv, __builtin_bit_cast(float, ce));
            wave_lds_order();
        }
        w->chosen[lane] = l < k ? __builtin_bit_cast(int, w->best[lane].y) : MASKED;
        wave_lds_order();
        const uint64_t bad = __ballot(whole && real);
        if (bad) {
            double inv = inv_sum;
            if (SOFTMAX && !sum_all && a.bias) inv = exact_inv();
            for (int q = 0; q < 4; ++q) {
                if (!((bad >> (16 * q)) & 0xffffu)) continue;
                const int e = route_exact<KIND>(a, a.logits + (t0 + q) * E, __shfl(zmax, 16 * q, 64), __shfl(inv, 16 * q, 64), sel64);
                if (lane < k) w->chosen[16 * q + lane] = e;
                wave_lds_order();
            }
        }
        const int e = w->chosen[lane];
        double p = 0.0;
        if (!(e & MASKED)) p = score64<KIND>(logit_of(zr[e]), zmax);
        double wt = sum_all ? p * inv_sum : p;
        if (a.renorm) {
            const double sum = row_sum(p);
            wt = sum > 0.0 ? p / sum : 0.0;
        }
        if (l < k && real) {
            a.idx[t * k + l] = e & (MASKED - 1);
            a.wgt[t * k + l] = (float)(wt * (double)a.route_scale);
        }
        wave_lds_order();
    }
}

/* One row of 16 lanes a token where a lane then has 16 experts at most, else a wave a
 * token. us, 256 experts (wave / row): 8 of 4 groups of 8, sigmoid and bias, 64 / 4095 /
 * 32768 tokens 6.6 / 18.7 / 49.4 -> 6.0 / 9.0 / 22.4; 6 of all, softmax 6.0 / 11.4 / 39.8 ->
 * 5.1 / 5.9 / 15.7. Before both, every score in 64 bits and topk rounds of a wave-wide
 * maximum, 14.3 / - / 121 (scores written) and - / 13.7 / -. Bound by the latency of
 * dependent steps: 241 vector instructions a token, four tokens' at once, which keep the units
 * busy half of the time; a wave waits 40 % of its cycles for an operand and 27 % for its turn. 32768
 * tokens' logits take 6.6 us at the rate of a copy. The next round's logits fetched ahead
 * cost a wave a SIMD and 13 to 25 %. */
hipError_t apus_launch_route(const ApusRouteArgs *a, hipStream_t st) {
    if (a->s <= 0) return hipSuccess;
    if (a->E <= 0 || a->E > 1024 || a->topk <= 0 || a->topk > 16 || a->topk > a->E) return hipErrorInvalidValue;
    const int per = a->E / a->groups;
    const bool al = (((uintptr_t)a->logits | (uintptr_t)a->scores) & 15) == 0;
    const auto by_kind = [&](auto go) {
        return a->score == APUS_SCORE_SIGMOID ? go(std::integral_constant<int, APUS_SCORE_SIGMOID>{})
             : a->score == APUS_SCORE_SOFTMAX ? go(std::integral_constant<int, APUS_SCORE_SOFTMAX>{})
                                              : go(std::integral_constant<int, APUS_SCORE_SQRTSOFTPLUS>{});
    };
    if (a->topk <= 8 && 16 % a->groups == 0 && per <= 16 * (16 / a->groups)) {
        const int lpg = 16 / a->groups, ne = (per + lpg - 1) / lpg;
        const size_t lds = 4 * (sizeof(RowLds) + a->E * sizeof(double)) + a->E * sizeof(float);
        const bool v = per % (4 * lpg) == 0 && al;
        /* as many workgroups as are resident, four a CU for a sigmoid's 113 registers, else three;
         * more would only start over (32768 tokens as above 25.2 us with a workgroup for each
         * 16, 22.6 in rounds; sqrt-softplus 24.5 with four, 20.5 with three) */
        const size_t resident = a->score == APUS_SCORE_SIGMOID ? 1024 : 768;
        const unsigned wgs = (unsigned)std::min(((size_t)a->s + 15) / 16, resident);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(wgs), dim3(256), lds, st, *a, lpg, ne);
            return hipGetLastError();
        };
        return by_kind([&](auto kc) {
            constexpr int KIND = kc;
            if (v)
                return ne <= 4 ? go(apus_route_row_kernel<KIND, 4, true>) : ne <= 8 ? go(apus_route_row_kernel<KIND, 8, true>)
                                                                                  : go(apus_route_row_kernel<KIND, 16, true>);
            return ne <= 2 ? go(apus_route_row_kernel<KIND, 2, false>) : ne <= 4 ? go(apus_route_row_kernel<KIND, 4, false>)
                 : ne <= 8 ? go(apus_route_row_kernel<KIND, 8, false>) : go(apus_route_row_kernel<KIND, 16, false>);
        });
    }
    int lpg = a->groups > 1 ? 16 : 64;
    if (a->groups > 1)
        while (lpg > 1 && (lpg * a->groups > 64 || lpg / 2 >= per)) lpg >>= 1;
    const int ne = (per + lpg - 1) / lpg, slots = a->topk <= 8 ? 8 : 16;
    /* tokens a wave: four waves a SIMD, then more tokens each */
    const int tpw = (int)std::min((size_t)64 / slots, ((size_t)a->s + 4095) / 4096);
    const size_t waves = ((size_t)a->s + tpw - 1) / tpw;
    const unsigned wgs = (unsigned)std::min((waves + 3) / 4, (size_t)1024);
    const size_t lds = 4 * (sizeof(WaveLds) + a->E * sizeof(double));
    const bool v = per % (4 * lpg) == 0 && ne <= 16 && al;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(wgs), dim3(256), lds, st, *a, lpg, ne, tpw, slots);
        return hipGetLastError();
    };
    return by_kind([&](auto kc) {
        constexpr int KIND = kc;
        if (v)
            return ne <= 4 ? go(apus_route_kernel<KIND, 4, true>) : ne <= 8 ? go(apus_route_kernel<KIND, 8, true>)
                                                                          : go(apus_route_kernel<KIND, 16, true>);
        return ne <= 2 ? go(apus_route_kernel<KIND, 2, false>) : ne <= 4 ? go(apus_route_kernel<KIND, 4, false>)
             : ne <= 8 ? go(apus_route_kernel<KIND, 8, false>) : ne <= 16 ? go(apus_route_kernel<KIND, 16, false>)
                                                               : go(apus_route_kernel<KIND, 32, false>);
    });
}
