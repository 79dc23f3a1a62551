/*
 * apus_i8.hip — products of 8-bit integers with a scale per token and per
 * channel: out[m, o] = (fp32(sum_k a[m, k] w[o, k]) * as[m]) * ws[o]. The sum is
 * exact in 32-bit integers (|sum| <= 2^14 K, K <= 131068), so every schedule
 * gives the same bits; fp32() rounds it once, each scale once.
 */
#include "apus_device.h"
#include "apus_internal.h"

#include <algorithm>
#include <type_traits>

typedef int apus_v4i __attribute__((ext_vector_type(4)));
/* the vector unit takes 8- and 16-byte accesses at any address (2997 x 18270 x 112, BF16 rows of
 * outputs of no whole 16 bytes: 42 us, element by element 124) */
typedef unsigned apus_v4u_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned apus_v2u_any __attribute__((ext_vector_type(2), aligned(2)));
typedef float apus_v4f_any __attribute__((ext_vector_type(4), aligned(4)));

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

/* the bits of four BF16 values */
__device__ __forceinline__ uint64_t bf16x4(const float (&v)[4]) {
    return (uint64_t)apus_bf16_bits(v[0]) | (uint64_t)apus_bf16_bits(v[1]) << 16 | (uint64_t)apus_bf16_bits(v[2]) << 32 |
           (uint64_t)apus_bf16_bits(v[3]) << 48;
}

/* outputs (m, o .. o + 3) */
template <bool YB>
__device__ __forceinline__ void i8_store4(const ApusI8Args &a, int m, int o, apus_v4i acc) {
    const float sa = a.as[m];
    const size_t i = (size_t)m * a.O + o;
    if (o + 4 <= a.O) {
        const apus_v4f_any sw = *(const APUS_GLOBAL apus_v4f_any *)(a.ws + o);
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = ((float)acc[k] * sa) * sw[k];
            if (YB || a.round_out) v[k] = apus_bf16_rne(v[k]);
        }
        if constexpr (YB)
            *(APUS_GLOBAL apus_v2u_any *)((uint16_t *)a.out + i) = __builtin_bit_cast(apus_v2u_any, bf16x4(v));
        else
            *(APUS_GLOBAL apus_v4f_any *)((float *)a.out + i) = apus_v4f_any{v[0], v[1], v[2], v[3]};
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (o + k < a.O) i8_store<YB>(a.out, i + k, acc[k], sa, a.ws[o + k], a.round_out);
}

/* tile of workgroup b: each XCD (workgroups are dealt to the 8 XCDs round robin)
 * takes a contiguous band of tiles */
__device__ __forceinline__ unsigned apus_i8_band(unsigned b, unsigned tiles) {
    const unsigned per = tiles >> 3, rem = tiles & 7, x = b & 7;
    return x * per + min(x, rem) + (b >> 3);
}
/* row and column block of a workgroup: in groups of up to 8 row blocks by every column
 * block, so that the tiles running together on an XCD share both operands in its L2 */
__device__ __forceinline__ void apus_i8_tile(unsigned b, int mt, int nt, int &mb, int &nb) {
    const unsigned t = apus_i8_band(b, (unsigned)mt * nt);
    const unsigned grp = t / (8u * nt), g0 = grp * 8, gm = min(8u, mt - g0), in = t - grp * 8 * nt;
    mb = g0 + in % gm;
    nb = in / gm;
}

}  // namespace

/* K % 16 != 0 or codes not 16-byte aligned (K % 4 == 0, 4-byte alignment): 64 x 64 outputs a
 * workgroup, 4 x 4 a thread, steps of 64 bytes of K through LDS, dot products on the vector
 * units. 4096 x 8192 x 4096 1546 us (121-127 with 16-byte pieces), 40 x 32768 x 1024 47 (8.5). */
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

/*
 * Block schedule: a workgroup of WM x WN waves owns BM activation rows x BN
 * weight rows. Both operands travel global -> LDS in steps of 128 bytes of K (8
 * whole 128-byte rows a load, NST stages), chunk c of row i in slot c ^ (i / 2 %
 * 8): the 16 rows that a quarter of a wave reads lie in 64 different banks. From
 * there fragments go into a second set of registers one matrix instruction's
 * depth ahead, so that a stage is free for its next load at the barrier behind
 * its last read. The weights are the first operand, so a lane has four neighbouring
 * outputs of one row. Rows past M or O repeat the last one; past K the activations are
 * zeroed in LDS (0 times whatever the clamped weight bytes are).
 * 4096 x 8192 x 4096, 256 x 256 tiles: 122-127 us, 2.2 POP/s (a large library product of
 * these sizes 130); the matrix cores are busy 49-51 % of its cycles at 2.1 GHz, without loads it
 * takes 15 % less, with the matrix instructions and barriers alone 30 %; the 64 MB of outputs
 * go out in two bursts. 1000 x 4096 x 8192, 128 x 128 tiles four stages deep, one round: 42 us
 * (46 with a step's loads in a burst behind its barrier); without loads 35, the matrix
 * instructions and barriers alone 29, the loads alone 26 (22 TB/s out of L2). Tried there: 4
 * waves of 64 x 64 56, 16 waves 46; two waves on the halves of each step's K, for two thirds of
 * the fragment reads, 42; one barrier for two steps 51. Outputs straight from registers
 * (4096 x 8192 x 4096) 191 instead of 129 (stores of 8 bytes to 16 rows); 32x32x32 instructions
 * 139 (fragments of half the depth); the wave's priority raised around the instructions 130.
 */
template <int BM_, int BN_, int WM_, int WN_, int NST_>
struct ApusI8Blk {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NST = NST_, NW = WM * WN;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int LX = BM / 8, LT = (BM + BN) / 8, LPW = LT / NW;  /* loads: activations, all, a wave's */
    static constexpr int STB = (BM + BN) * 128, LDS = NST * STB + (BM + BN) * 4;  /* stages; scales */
    static_assert(BM % (WM * 16) == 0 && BN % (WN * 16) == 0 && (BM + BN) % 64 == 0 && LT % NW == 0 && LDS <= 160 * 1024, "block shape");
};

template <class B, bool YB>
__global__ __launch_bounds__(64 * B::NW) void apus_i8_block_kernel(ApusI8Args a) {
    constexpr int TM = B::TM, TN = B::TN, NST = B::NST;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4, wm = wave / B::WN, wn = wave % B::WN;
    const int mt = (a.M + B::BM - 1) / B::BM, nt = (a.O + B::BN - 1) / B::BN;
    int mb, nb;
    apus_i8_tile(blockIdx.x, mt, nt, mb, nb);
    const int m0 = mb * B::BM, n0 = nb * B::BN, K = a.K, nq = (K + 127) >> 7, tail = K & 127;
    const unsigned lbase = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)lds);
    /* a wave's loads: a uniform base and 32-bit lane offsets; the last step's chunks past K
     * read the row's last chunk */
    const uint8_t *xb = (const uint8_t *)a.a + (size_t)m0 * K, *wb = (const uint8_t *)a.w + (size_t)n0 * K;
    unsigned off[B::LPW];
    auto load_of = [&](int u) { return wave * B::LPW + u; };
    /* the lane's chunk of row 8 j + lane / 8, j = load_of(u) or, of a weight, an even LX less */
    auto chunk_in = [&](int u) { return (lane & 7) ^ ((4 * load_of(u) + (lane >> 4)) & 7); };
#pragma unroll
    for (int u = 0; u < B::LPW; ++u) {
        const int ii = load_of(u), i = 8 * (ii < B::LX ? ii : ii - B::LX) + (lane >> 3);
        off[u] = (unsigned)min(i, (ii < B::LX ? a.M - m0 : a.O - n0) - 1) * (unsigned)K + chunk_in(u) * 16;
    }
    auto issue1 = [&](int u, int q, int slot, bool last) {
        const int ii = load_of(u);
        unsigned o = off[u];
        if (last) o -= max(0, chunk_in(u) * 16 - (tail - 16));
        asm("" : "+v"(o));                                   /* 32 bits beside the uniform base */
        apus_g2lds16((ii < B::LX ? xb : wb) + (size_t)q * 128 + o, lbase + slot * B::STB + ii * 1024);
    };
    auto issue = [&](int q, int slot) {
        const bool last = tail && q == nq - 1;
#pragma unroll
        for (int u = 0; u < B::LPW; ++u) issue1(u, q, slot, last);
    };
    /* the activation chunks past K that this wave loaded, once they are in LDS */
    auto zero_tail = [&](int slot) {
#pragma unroll
        for (int u = 0; u < B::LPW; ++u)
            if (load_of(u) < B::LX && chunk_in(u) * 16 >= tail)
                *reinterpret_cast<apus_v4i *>(lds + slot * B::STB + load_of(u) * 1024 + lane * 16) = apus_v4i{0, 0, 0, 0};
    };
    struct Frag { apus_v4i w[TN], x[TM]; };
    const int sw = (r >> 1) & 7;
    /* fragment j of half s of a stage: the weights', then the activations' */
    auto read1 = [&](Frag &f, int j, const uint8_t *stg, int c) {
        if (j < TN) f.w[j] = *reinterpret_cast<const apus_v4i *>(stg + (B::BM + (wn * TN + j) * 16 + r) * 128 + c);
        else        f.x[j - TN] = *reinterpret_cast<const apus_v4i *>(stg + ((wm * TM + j - TN) * 16 + r) * 128 + c);
    };
    auto chunk_of = [&](int s) { return ((4 * s + g) ^ sw) << 4; };
    apus_v4i acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[i][t] = apus_v4i{0, 0, 0, 0};
    /* Products of half a stage, and among them the reads of the next half's fragments and
     * (load) the wave's loads of stage q: a wave issues in order, and in a burst behind the
     * barrier its loads wait for the address unit while no matrix instruction goes out */
    auto half = [&](const Frag &now, Frag &next, int from, int s, bool more, bool load, int q, int to, bool last) {
        constexpr int NM = TN * TM, NR = TN + TM, P = NM < B::LPW ? NM : B::LPW;
        const uint8_t *stg = lds + from * B::STB;
        const int c = chunk_of(s);
        auto one = [&](int j) {
            acc[j / TM][j % TM] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now.w[j / TM], now.x[j % TM], acc[j / TM][j % TM], 0, 0, 0);
        };
#pragma unroll
        for (int p = 0; p < P; ++p) {
            one(p * NM / P);
            __builtin_amdgcn_sched_barrier(0);
            if (load) {
#pragma unroll
                for (int u = p * B::LPW / P; u < (p + 1) * B::LPW / P; ++u) issue1(u, q, to, last);
            }
            if (more) {
#pragma unroll
                for (int j = p * NR / P; j < (p + 1) * NR / P; ++j) read1(next, j, stg, c);
            }
#pragma unroll
            for (int j = p * NM / P + 1; j < (p + 1) * NM / P; ++j) one(j);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    /* scales of the block's rows, then of its columns, to LDS */
    for (int i = wave; i < (B::BM + B::BN) / 64; i += B::NW) {     /* older than every stage: counted with the first */
        const int k = 64 * i + lane;
        apus_g2lds4(k < B::BM ? a.as + min(m0 + k, a.M - 1) : a.ws + min(n0 + k - B::BM, a.O - 1),
                    lbase + NST * B::STB + i * 256);
    }
    const int pre = min(nq, NST);
    for (int q = 0; q < pre; ++q) issue(q, q);
    /* stage q complete: only the stages behind it may be in flight */
    auto arrive = [&](int q, int slot, int issued) {
        const int behind = issued - 1 - q;
        if (NST > 3 && behind >= 3)      apus_wait_vm<3 * B::LPW>();
        else if (NST > 2 && behind >= 2) apus_wait_vm<2 * B::LPW>();
        else if (behind >= 1)            apus_wait_vm<B::LPW>();
        else                             apus_wait_vm<0>();
        if (tail && q == nq - 1) zero_tail(slot);
        apus_lds_barrier();
    };
    arrive(0, 0, pre);
    Frag fr[2];
#pragma unroll
    for (int j = 0; j < TN + TM; ++j) read1(fr[0], j, lds, chunk_of(0));
    int slot = 0;
    /* stage q, whose first half is in fr[0] */
    auto step = [&](int q, bool more, bool load, bool last) {
        const int nxt = slot + 1 == NST ? 0 : slot + 1;
        half(fr[0], fr[1], slot, 1, true, false, 0, 0, false);
        if (more) arrive(q + 1, nxt, min(nq, q + NST));
        __builtin_amdgcn_sched_barrier(0);
        half(fr[1], fr[0], nxt, 0, more, load, q + NST, slot, last);
        slot = nxt;
    };
    int q = 0;
    for (; q + 1 + NST < nq; ++q) step(q, true, true, false);
    for (; q < nq; ++q) step(q, q + 1 < nq, q + NST < nq, tail && q + NST == nq - 1);
    /* Outputs: 16 rows at a time through a wave's own LDS, so that a store writes whole
     * lines. A lane holds row r, columns 4 g .. 4 g + 3 of each tile. */
    constexpr int E = YB ? 2 : 4, CW = TN * 16, PITCH = CW * E + 16;
    constexpr int LR = CW * E / 16;                             /* 16-byte pieces of a row */
    static_assert(B::NW * 16 * PITCH <= NST * B::STB && 64 % LR == 0, "output staging");
    __syncthreads();
    const float *las = reinterpret_cast<const float *>(lds + NST * B::STB) + wm * TM * 16;
    const float *lws = reinterpret_cast<const float *>(lds + NST * B::STB) + B::BM + wn * CW;
    uint8_t *ob = lds + wave * (16 * PITCH);
    apus_v4f sw4[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) sw4[i] = *reinterpret_cast<const apus_v4f *>(lws + i * 16 + 4 * g);
    const int col = n0 + wn * CW + lane % LR * (16 / E);
    const bool whole = col + 16 / E <= a.O;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const float sa = las[t * 16 + r];
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = ((float)acc[i][t][k] * sa) * sw4[i][k];
                if (YB || a.round_out) v[k] = apus_bf16_rne(v[k]);
            }
            uint8_t *d = ob + r * PITCH + (i * 16 + 4 * g) * E;
            if constexpr (YB) *reinterpret_cast<uint64_t *>(d) = bf16x4(v);
            else              *reinterpret_cast<apus_v4f *>(d) = apus_v4f{v[0], v[1], v[2], v[3]};
        }
        asm volatile("" ::: "memory");                          /* a wave's LDS operations run in order */
#pragma unroll
        for (int p = 0; p < (16 * LR + 63) / 64; ++p) {
            const int row = p * (64 / LR) + lane / LR, m = m0 + (wm * TM + t) * 16 + row;
            if (row >= 16) break;
            const apus_v4u v = *reinterpret_cast<const apus_v4u *>(ob + row * PITCH + lane % LR * 16);
            uint8_t *d = (uint8_t *)a.out + ((size_t)m * a.O + col) * E;
            if (m < a.M && whole) {
                *(APUS_GLOBAL apus_v4u_any *)d = v;
            } else if (m < a.M) {
#pragma unroll
                for (int k = 0; k < 16 / E; ++k)
                    if (col + k < a.O) {
                        if constexpr (YB) apus_gst<uint16_t>(d + 2 * k, (uint16_t)(v[k >> 1] >> (16 * (k & 1))));
                        else              apus_gst<uint32_t>(d + 4 * k, v[k]);
                    }
            }
        }
        asm volatile("" ::: "memory");
    }
}

/* Kernel's limit of dynamic LDS raised to LDS bytes, once. The kernel is a template argument: kernels
 * of one type passed as values would share the static, and only the first would be raised */
template <auto Kernel, int LDS>
hipError_t apus_i8_lds_limit() {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    return attr;
}

template <class B>
hipError_t apus_launch_i8_block(const ApusI8Args &a, hipStream_t st) {
    auto go = [&](auto yb) {
        constexpr auto kernel = &apus_i8_block_kernel<B, decltype(yb)::value>;
        const hipError_t attr = apus_i8_lds_limit<kernel, B::LDS>();
        if (attr != hipSuccess) return attr;
        const size_t tiles = ((size_t)a.M + B::BM - 1) / B::BM * (((size_t)a.O + B::BN - 1) / B::BN);
        if (tiles > 0xffffffffu / (64 * B::NW)) return hipErrorInvalidValue;
        hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(64 * B::NW), B::LDS, st, a);
        return hipGetLastError();
    };
    return a.y_bf16 ? go(std::true_type{}) : go(std::false_type{});
}

/*
 * Narrow schedule, for some tens of rows: a workgroup owns 16 TN weight rows and 16 TM
 * activation rows (HALF: at most 8 rows, half a tile's loads);
 * its NW waves split K, each bringing both operands through a ring of its own in
 * LDS, PD steps of 128 bytes deep: no barrier in the loop. The waves' integer sums
 * meet in LDS. 8 rows, 4096 x 8192: 8.0 us (33.5 MB at 4.2 TB/s; 5 us of them at the rate of
 * a long stream), the rest launch, ramp and the sums; up to 64 rows 12.4, where 256
 * workgroups read 134 MB of activations from L2.
 */
template <int TM, int TN, int NW, int PD, bool HALF, bool YB>
__global__ __launch_bounds__(64 * NW) void apus_i8_narrow_kernel(ApusI8Args a) {
    constexpr int LX = HALF ? 1 : 2 * TM, NL = LX + 2 * TN, SLOT = NL * 1024;
    static_assert((PD - 1) * NL < 64 && PD >= 2 && PD <= 4, "vmcnt");
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4, K = a.K, nq = (K + 127) >> 7, tail = K & 127;
    const int mt = (a.M + 16 * TM - 1) / (16 * TM), nt = (a.O + 16 * TN - 1) / (16 * TN);
    const unsigned t0 = apus_i8_band(blockIdx.x, (unsigned)mt * nt);     /* the row blocks of a column block in turn */
    const int n0 = (int)(t0 / mt) * 16 * TN, m0 = (int)(t0 % mt) * 16 * TM;
    const int q0 = (int)((size_t)nq * wave / NW), q1 = (int)((size_t)nq * (wave + 1) / NW);
    uint8_t *ring = lds + wave * PD * SLOT;
    const unsigned rbase = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)ring);
    const uint8_t *xb = (const uint8_t *)a.a + (size_t)m0 * K, *wb = (const uint8_t *)a.w + (size_t)n0 * K;
    unsigned off[NL];
    int chunk[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) chunk[h] = (lane & 7) ^ ((4 * h + (lane >> 4)) & 7);
#pragma unroll
    for (int u = 0; u < NL; ++u) {
        const int j = u < LX ? u : u - LX, i = 8 * j + (lane >> 3);
        off[u] = (unsigned)min(i, (u < LX ? a.M - m0 : a.O - n0) - 1) * (unsigned)K + chunk[j & 1] * 16;
    }
    auto issue = [&](int q, int slot) {
        const bool last = tail && q == nq - 1;
#pragma unroll
        for (int u = 0; u < NL; ++u) {
            unsigned o = off[u];
            if (last) o -= max(0, chunk[(u < LX ? u : u - LX) & 1] * 16 - (tail - 16));
            asm("" : "+v"(o));
            apus_g2lds16((u < LX ? xb : wb) + (size_t)q * 128 + o, rbase + slot * SLOT + u * 1024);
        }
    };
    apus_v4i acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[i][t] = apus_v4i{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < PD; ++d)
        if (q0 + d < q1) issue(q0 + d, d);
    const int sw = (r >> 1) & 7;
    int slot = 0;
    for (int q = q0; q < q1; ++q) {
        const int later = min(q1 - 1 - q, PD - 1);
        if (PD > 3 && later >= 3)      apus_wait_vm<3 * NL>();
        else if (PD > 2 && later >= 2) apus_wait_vm<2 * NL>();
        else if (later >= 1)           apus_wait_vm<NL>();
        else                           apus_wait_vm<0>();
        uint8_t *stg = ring + slot * SLOT;
        if (tail && q == nq - 1) {
#pragma unroll
            for (int u = 0; u < LX; ++u)
                if (chunk[u & 1] * 16 >= tail)
                    *reinterpret_cast<apus_v4i *>(stg + u * 1024 + lane * 16) = apus_v4i{0, 0, 0, 0};
            asm volatile("" ::: "memory");
        }
        apus_v4i w[TN][2], x[TM][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = ((4 * h + g) ^ sw) << 4;
#pragma unroll
            for (int i = 0; i < TN; ++i)
                w[i][h] = *reinterpret_cast<const apus_v4i *>(stg + LX * 1024 + (16 * i + r) * 128 + c);
            /* HALF: rows 8..15 read rows 0..7 again; their columns are not stored */
#pragma unroll
            for (int t = 0; t < TM; ++t)
                x[t][h] = *reinterpret_cast<const apus_v4i *>(stg + (HALF ? r & 7 : 16 * t + r) * 128 + (HALF ? ((4 * h + g) ^ ((r & 7) >> 1)) << 4 : c));
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      /* slot read before its refill */
        if (q + PD < q1) issue(q + PD, slot);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int t = 0; t < TM; ++t)
                    acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i][h], x[t][h], acc[i][t], 0, 0, 0);
        slot = slot + 1 == PD ? 0 : slot + 1;
    }
    /* lane: activation row 16 t + r, weight rows n0 + 16 i + 4 g + k */
    apus_v4i *red = reinterpret_cast<apus_v4i *>(lds);
    if constexpr (NW > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int t = 0; t < TM; ++t) red[(wave * TN * TM + i * TM + t) * 64 + lane] = acc[i][t];
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < TN * TM; ++u) {
        if (NW > 1 && u % NW != wave) continue;
        const int i = u / TM, t = u % TM, m = m0 + 16 * t + r, o = n0 + 16 * i + 4 * g;
        apus_v4i v = NW > 1 ? red[u * 64 + lane] : acc[i][t];
#pragma unroll
        for (int k = 1; k < NW; ++k) v += red[(k * TN * TM + u) * 64 + lane];
        if (m < a.M) i8_store4<YB>(a, m, o, v);
    }
}

template <int TM, int TN, int NW, int PD, bool HALF>
hipError_t apus_launch_i8_narrow(const ApusI8Args &a, hipStream_t st) {
    constexpr int ring = NW * PD * ((HALF ? 1 : 2 * TM) + 2 * TN) * 1024, sums = NW * TM * TN * 1024;
    constexpr int lds = ring > sums ? ring : sums;
    static_assert(lds <= 160 * 1024, "LDS");
    auto go = [&](auto yb) {
        constexpr auto kernel = &apus_i8_narrow_kernel<TM, TN, NW, PD, HALF, decltype(yb)::value>;
        const hipError_t attr = apus_i8_lds_limit<kernel, lds>();
        if (attr != hipSuccess) return attr;
        const size_t wgs = ((size_t)a.O + 16 * TN - 1) / (16 * TN) * (((size_t)a.M + 16 * TM - 1) / (16 * TM));
        if (wgs > 0xffffffffu / (64 * NW)) return hipErrorInvalidValue;
        hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(64 * NW), lds, st, a);
        return hipGetLastError();
    };
    return a.y_bf16 ? go(std::true_type{}) : go(std::false_type{});
}

/*
 * One row: dot products on the vector units. A wave takes R weight rows, U chunks of
 * 1 KB (16 bytes a lane) of each under way at once; sums over the lanes by a
 * reduce-scatter. XS: the activations are codes (0), or an fp32 (1) or BF16 (2) row
 * that every workgroup quantises for itself into LDS while its first weights come.
 */
template <int R, int U, int XS, bool YB>
__global__ __launch_bounds__(256) void apus_i8_gemv_kernel(ApusI8Args a) {
    extern __shared__ __align__(16) uint8_t lds[];               /* XS: the row's codes */
    __shared__ unsigned lmax[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int K = a.K, nc = (K + 1023) >> 10, n0 = (blockIdx.x * 4 + wave) * R;
    const uint8_t *wr[R];
#pragma unroll
    for (int i = 0; i < R; ++i) wr[i] = (const uint8_t *)a.w + (size_t)min(n0 + i, a.O - 1) * K;
    apus_v4i w[U][R];
    auto load_w = [&](int c0) {                                  /* past K: the row's last bytes again */
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < R; ++i)
                w[u][i] = __builtin_bit_cast(apus_v4i, apus_ld16_stream(wr[i] + min((c0 + u) * 1024 + lane * 16, K - 16)));
    };
    load_w(0);
    float sa;
    if constexpr (XS != 0) {
        __builtin_amdgcn_sched_barrier(0);                       /* the weights are under way first */
        auto ldx = [&](int k, float (&v)[4]) {
            if constexpr (XS == 1) {
                const float4 f = apus_gld<float4>((const float *)a.x + k);
                v[0] = apus_bf16_rne(f.x); v[1] = apus_bf16_rne(f.y); v[2] = apus_bf16_rne(f.z); v[3] = apus_bf16_rne(f.w);
            } else {
                const uint64_t f = apus_gld<uint64_t>((const uint16_t *)a.x + k);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = apus_u2f((uint32_t)(f >> (16 * j)) << 16);
            }
        };
        unsigned top = 0;
        for (int k = threadIdx.x * 4; k < K; k += 1024) {
            float v[4];
            ldx(k, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, apus_f2u(v[j]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
        if (lane == 0) lmax[wave] = top;
        apus_lds_barrier();
        float inv;
        apus_i8_scale(apus_u2f(max(max(lmax[0], lmax[1]), max(lmax[2], lmax[3]))), sa, inv);
        for (int k = threadIdx.x * 4; k < K; k += 1024) {
            float v[4];
            ldx(k, v);
            unsigned c = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) c |= (unsigned)(apus_i8_code(v[j], inv) & 0xff) << (8 * j);
            *reinterpret_cast<unsigned *>(lds + k) = c;
        }
        apus_lds_barrier();
    } else {
        sa = a.as[0];
    }
    int v[R] = {};
    for (int c0 = 0; c0 < nc; c0 += U) {
        if (c0) load_w(c0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (c0 + u) * 1024 + lane * 16, kk = min(k, K - 16);
            apus_v4i x;
            if constexpr (XS != 0) x = *reinterpret_cast<const apus_v4i *>(lds + kk);
            else                   x = apus_gld<apus_v4i>(a.a + kk);
            if (k >= K) x = apus_v4i{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i] = __builtin_amdgcn_sdot4(w[u][i][j], x[j], v[i], false);
        }
    }
    /* reduce-scatter: lane l ends up with row l's sum, its low bits in reverse */
#pragma unroll
    for (int off = 1, n = R; off <= 32; off <<= 1, n = n > 1 ? n >> 1 : 1) {
        const bool up = lane & off;
        if (n == 1) {
            v[0] += __shfl_xor(v[0], off, 64);
            continue;
        }
#pragma unroll
        for (int j = 0; j < n / 2; ++j) {
            const int keep = up ? v[n / 2 + j] : v[j], send = up ? v[j] : v[n / 2 + j];
            v[j] = keep + __shfl_xor(send, off, 64);
        }
    }
    static_assert(R == 1 || R == 2 || R == 4, "rows of a wave");
    const int o = n0 + (R == 4 ? (lane & 1) * 2 + (lane >> 1) : lane);
    if (lane < R && o < a.O) i8_store<YB>(a.out, o, v[0], sa, a.ws[o], a.round_out);
}

template <int R, int U, int XS>
hipError_t apus_launch_i8_gemv(const ApusI8Args &a, hipStream_t st) {
    auto go = [&](auto kernel) {
        const size_t wgs = ((size_t)a.O + 4 * R - 1) / (4 * R);
        if (wgs > 0xffffffffu / 256) return hipErrorInvalidValue;
        hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(256), XS ? (a.K + 15) & ~15 : 0, st, a);
        return hipGetLastError();
    };
    return a.y_bf16 ? go(&apus_i8_gemv_kernel<R, U, XS, true>) : go(&apus_i8_gemv_kernel<R, U, XS, false>);
}

namespace {

/* a launch holds fewer than 2^32 threads */
constexpr size_t THREADS_MAX = 0xffffffffu;

/* Rows and chunks a wave: about 4 KB of weights under way in each, from as many rows as
 * that takes (us, 1 x 4 / 2 x 2 / 4 x 1: K 8192, 4096 channels 7.1 / 7.6 / 8.8; K 4096, 1024
 * channels 2.8 / 3.4 / 4.5, 129280 74 / 75 / 79 (7.1 TB/s); K 2048, 4096 channels 3.8 / 3.4 /
 * 3.7; K 1024, 32768 channels 12.5 / 8.0 / 7.0; more of a row or more rows at once are
 * slower everywhere). Bound by HBM, or by the launch and one pass of latency. */
int gemv_rows(int K) { return K > 2048 ? 1 : K > 1024 ? 2 : 4; }
/* whether the one-row schedule's grid holds O channels */
bool gemv_fits(int O, int K) {
    return O <= 1 << 26 && ((size_t)O + 4 * gemv_rows(K) - 1) / (4 * gemv_rows(K)) <= THREADS_MAX / 256;
}

}  // namespace

template <int XS>
hipError_t apus_launch_i8_gemv_x(const ApusI8Args &a, hipStream_t st) {
    const int rows = gemv_rows(a.K);
    return rows == 1 ? apus_launch_i8_gemv<1, 4, XS>(a, st) : rows == 2 ? apus_launch_i8_gemv<2, 2, XS>(a, st)
                                                                        : apus_launch_i8_gemv<4, 1, XS>(a, st);
}

namespace {

struct Sched {
    hipError_t (*launch)(const ApusI8Args &, hipStream_t);
    ApusI8Shape shape;
    float c, e, t, c2, e2;                /* the modelled time, in us */
};
template <int TM, int TN, int NW, int PD, bool HALF>
constexpr Sched narrow_sched(float c, float e, float t, float c2, float e2) {
    return {apus_launch_i8_narrow<TM, TN, NW, PD, HALF>, {HALF ? 8 : 16 * TM, 16 * TN, NW, PD, 64 * NW}, c, e, t, c2, e2};
}
template <class B>
constexpr Sched block_sched(float c, float e, float t, float c2, float e2) {
    return {apus_launch_i8_block<B>, {B::BM, B::BN, 1, B::NST, 64 * B::NW}, c, e, t, c2, e2};
}
constexpr Sched FEW[] = {narrow_sched<1, 1, 4, 4, true>(0, 0, 0, 0, 0), narrow_sched<1, 2, 2, 4, true>(0, 0, 0, 0, 0)};
/* Fitted to every other of 228 measured shapes (9 to 4096 rows, 256 to 32768 channels, K 512
 * to 8192; mean error 6 to 11 % a schedule); on the rest the choice is 0.7 % behind the
 * fastest of all in the geometric mean, 12 % at worst. Without 256 x 128 it is 0.8 %, 23 % at
 * worst; without any other, 1.0 to 8.2 %. */
constexpr Sched MORE[] = {
    narrow_sched<1, 1, 4, 4, false>(0.046f, 1.04f, 1.46f, 0.105f, 0.99f),
    narrow_sched<2, 2, 2, 4, false>(0.129f, 0.54f, 2.31f, 0.0f, 0.0f),
    narrow_sched<4, 2, 4, 2, false>(0.159f, 2.23f, 0.81f, 0.0f, 0.0f),
    block_sched<ApusI8Blk<64, 64, 4, 2, 4>>(0.216f, 1.00f, 2.48f, 0.419f, 2.42f),
    block_sched<ApusI8Blk<64, 128, 2, 4, 4>>(0.352f, 3.24f, 0.55f, 0.0f, 0.0f),
    block_sched<ApusI8Blk<128, 128, 2, 4, 4>>(0.481f, 5.69f, -1.01f, 0.0f, 0.0f),
    block_sched<ApusI8Blk<128, 128, 2, 4, 2>>(0.779f, 0.12f, 3.03f, 1.020f, 4.95f),
    block_sched<ApusI8Blk<256, 128, 4, 2, 3>>(0.797f, 7.71f, -0.71f, 0.0f, 0.0f),
    block_sched<ApusI8Blk<256, 256, 2, 4, 2>>(1.403f, 13.47f, -3.17f, 0.0f, 0.0f),
};

size_t tiles_of(const ApusI8Shape &s, int M, int O) { return ((size_t)M + s.rows - 1) / s.rows * (((size_t)O + s.cols - 1) / s.cols); }

/* The schedule of 2 rows and more with 16-byte pieces; null where no grid holds the tiles. */
const Sched *choose(int M, int O, int K) {
    if (O > 1 << 26) return nullptr;
    if (M <= 8)
        /* Short rows of many channels: twice the channels a workgroup and half the waves
         * (16 x 4 / 32 x 2, 8 rows, us: K 1024, 8192 / 16384 / 32768 channels 3.7 / 6.5 / 10.0
         * against 3.8 / 5.9 / 8.5; K 2048, 12288 channels 6.8 against 7.6; K 4096, 32768 25.8
         * against 28.6; 4096 x 8192 8.0 against 10.5) */
        return &FEW[K <= 1024 && O > 8192];
    /* More rows: the schedule whose modelled time is least. n workgroups of `steps`
     * steps of 128 bytes of K take, in us, rounds of 256 CUs times (c steps + e); where
     * two workgroups fit a CU, rounds of 512 times (c2 steps + e2), a last one of up to
     * 256 the former; + t. */
    const float steps = (float)((K + 127) / 128);
    const Sched *best = nullptr;
    float least = 0.0f;
    for (const Sched &c : MORE) {
        const size_t n = tiles_of(c.shape, M, O), left = n % 512;
        if (n > THREADS_MAX / c.shape.threads) continue;
        const float one = c.c * steps + c.e, two = c.c2 * steps + c.e2;
        const float us = c.c2 == 0.0f ? (float)((n + 255) / 256) * one + c.t
                                      : (float)(n / 512) * two + (left == 0 ? 0.0f : left <= 256 ? one : two) + c.t;
        if (!best || us < least) {
            best = &c;
            least = us;
        }
    }
    return best;
}

}  // namespace

ApusI8Shape apus_i8_schedule(int M, int O, int K) {
    if (M == 1) return gemv_fits(O, K) ? ApusI8Shape{1, 4 * gemv_rows(K), 1, 1, 256} : ApusI8Shape{};
    const Sched *s = choose(M, O, K);
    return s ? s->shape : ApusI8Shape{};
}

/* one row, fp32 or BF16 in: quantised inside the product's launch */
bool apus_i8_fused_ok(const ApusI8Args *a) {
    return a->M == 1 && gemv_fits(a->O, a->K) && a->K % 16 == 0 && a->K <= 32768 && (((uintptr_t)a->x | (uintptr_t)a->w) & 15) == 0;
}

hipError_t apus_launch_i8_gemm(const ApusI8Args *a, hipStream_t st) {
    if (a->M <= 0) return hipSuccess;
    if (a->x) return a->x_bf16 ? apus_launch_i8_gemv_x<2>(*a, st) : apus_launch_i8_gemv_x<1>(*a, st);
    if (a->K % 16 == 0 && (((uintptr_t)a->a | (uintptr_t)a->w) & 15) == 0) {
        if (a->M == 1) {
            if (gemv_fits(a->O, a->K)) return apus_launch_i8_gemv_x<0>(*a, st);
        } else if (const Sched *s = choose(a->M, a->O, a->K)) {
            return s->launch(*a, st);
        }
        /* more channels or tiles than a launch has workgroups for: the loops of the last kernel */
    }
    const size_t tiles = ((size_t)a->M + 63) / 64 * (((size_t)a->O + 63) / 64);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(tiles, (size_t)1 << 20)), dim3(256), 0, st, *a);
        return hipGetLastError();
    };
    return a->y_bf16 ? go(apus_i8_any_kernel<true>) : go(apus_i8_any_kernel<false>);
}
