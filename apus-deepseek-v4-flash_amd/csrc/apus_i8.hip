/*
 * apus_i8.hip — products of 8-bit integers with a scale per token and per
 * channel: out[m, o] = (fp32(sum_k a[m, k] w[o, k]) * as[m]) * ws[o]. The sum is
 * exact in 32-bit integers (|sum| <= 2^14 K, K <= 131068), so every schedule
 * gives the same bits; fp32() rounds it once, each scale once.
 */
#include "apus_device.h"
#include "apus_internal.h"

#include <algorithm>

namespace {

template <bool YB>
__device__ __forceinline__ void i8_store(void *out, size_t i, int acc, float sa, float sw, int round_out) {
    float v = ((float)acc * sa) * sw;
    if constexpr (YB) {
        apus_gst<uint16_t>((uint16_t *)out + i, apus_bf16_bits(apus_bf16_rne(v)));
    } else {
        apus_gst<float>((float *)out + i, round_out ? apus_bf16_rne(v) : v);
    }
}

}  // namespace

/* Any shape with K % 4 == 0, 4-byte alignment: 64 x 64 outputs a workgroup,
 * 4 x 4 a thread, steps of 64 bytes of K through LDS. */
template <bool YB>
__global__ __launch_bounds__(256) void apus_i8_any_kernel(ApusI8Args a) {
    __shared__ int la[64][17], lw[64][17];
    const int nt = (a.O + 63) / 64, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int K4 = a.K >> 2;
    const size_t tiles = (((size_t)a.M + 63) / 64) * nt;
    for (size_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int m0 = (int)(t / nt) * 64, o0 = (int)(t % nt) * 64;
        int acc[4][4] = {};
        for (int k0 = 0; k0 < K4; k0 += 16) {
            for (int i = tid; i < 64 * 16; i += 256) {
                const int r = i >> 4, c = i & 15, k = k0 + c;
                la[r][c] = k < K4 && m0 + r < a.M ? *(const int *)(a.a + (size_t)(m0 + r) * a.K + 4 * (size_t)k) : 0;
                lw[r][c] = k < K4 && o0 + r < a.O ? *(const int *)(a.w + (size_t)(o0 + r) * a.K + 4 * (size_t)k) : 0;
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < 16; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[i][j] = __builtin_amdgcn_sdot4(la[ty + 16 * i][c], lw[tx + 16 * j][c], acc[i][j], false);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int m = m0 + ty + 16 * i, o = o0 + tx + 16 * j;
                if (m < a.M && o < a.O) i8_store<YB>(a.out, (size_t)m * a.O + o, acc[i][j], a.as[m], a.ws[o], a.round_out);
            }
    }
}

hipError_t apus_launch_i8_gemm(const ApusI8Args *a, hipStream_t st) {
    if (a->M <= 0) return hipSuccess;
    const size_t tiles = ((size_t)a->M + 63) / 64 * (((size_t)a->O + 63) / 64);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(tiles, (size_t)1 << 20)), dim3(256), 0, st, *a);
        return hipGetLastError();
    };
    return a->y_bf16 ? go(apus_i8_any_kernel<true>) : go(apus_i8_any_kernel<false>);
}
