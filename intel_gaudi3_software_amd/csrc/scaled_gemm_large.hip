// scaled_gemm_large.hip -- the scaled product with tiles of 256 x 256 outputs, for products with enough of them: bound by the matrix
// cores (and by the power that they and the operands' way to them draw).
//
// The plan is the one of the fp8 contraction's large-tile kernel (gemm_large_tile_impl.hpp): eight wavefronts, 2 x 4 over the tile,
// 128 x 64 outputs each in 128 accumulator registers; a ring of four stages of 64 k (32 KiB each) filled by direct copies from
// memory to LDS; a stage's fragments are read while the previous stage is multiplied, each register refilled right after its last
// use, so a slot is free again one step before its stage is multiplied and three stages are in flight behind the one being
// read; one barrier per stage; 16-byte chunks of the 64-byte rows swizzled by (row >> 2) & 3, which keeps the fragment reads free of bank
// conflicts.  New here: int8 (two 32-k instructions where fp8 has one of 64 k), rows of any count on both sides (the copies of a
// partial tile read its last row again, its stores are predicated), K of any length from 256 on (what is left behind the last whole
// stage is multiplied from registers), and an epilogue with a scale per row and per column.  Measured: int8 4096^3 with a bias 64 us
// (2150 TOP/s), fp8 57 us; four products of 2048 x 14336 x 4096 in fp8 425 us (2260 TFLOP/s), in int8 455; 8192 x 4096 x 256, whose time
// is the stores', 25 us.
#include "scaled_gemm_common.hpp"

namespace mme
{
namespace
{
constexpr int TM = 256, TN = 256, BK = 64, NST = 4, STAGE = (TM + TN) * BK;
constexpr int LDS_BYTES = NST * STAGE; // 128 KiB
#define FENCE __builtin_amdgcn_sched_barrier(0)
// at most n of the wavefront's requests outstanding, and none of its LDS reads
constexpr int landed_and_read(int n) { return vm_wait(n) & ~0x0F00; }

__device__ __forceinline__ s_v8i read_frag(const char* st, int row0, int lane)
{
    const int r = row0 + (lane & 31), c0 = 2 * (lane >> 5), z = (r >> 2) & 3;
    return join(*(const s_v4i*) (st + (r * 4 + (c0 ^ z)) * 16), *(const s_v4i*) (st + (r * 4 + ((c0 + 1) ^ z)) * 16));
}

typedef uint32_t any_v4u __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t lds_v4u __attribute__((ext_vector_type(4)));

template<int OPS>
__global__ __launch_bounds__(512, 2) void scaled_gemm_large_kernel(const ScaledGemmArgs a)
{
    typedef typename Sums<OPS>::v16 v16;
    typedef typename Sums<OPS>::one one;
    constexpr int NI = 4, NJ = 2, WC = 64, WR = 128, NREQ = 4;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const int tiles_m = (a.M + TM - 1) / TM, tiles_n = (a.N + TN - 1) / TN;
    // consecutive tiles go to one XCD (workgroups are dealt out to the eight in turn); within that order, bands of eight tile rows are
    // walked column by column, so that the tiles an XCD works on at a time share eight panels of x and a few of w
    const int total = (int) gridDim.x, xcd = (int) blockIdx.x & 7;
    const int L = xcd * (total >> 3) + min(xcd, total & 7) + ((int) blockIdx.x >> 3);
    const int band = L / (8 * tiles_n), in_band = L - band * 8 * tiles_n, height = min(8, tiles_m - band * 8);
    const int m0 = (band * 8 + in_band % height) * TM, n0 = (in_band / height) * TN;
    const BatchOffsets o = batch_offsets(a, blockIdx.y);
    const uint8_t*     X = a.x + o.x;
    const uint8_t*     W = a.w + o.w;
    const uint32_t     lds_base = (uint32_t) (uintptr_t) lds;

    const uint8_t* gx[2];
    const uint8_t* gw[2];
#pragma unroll
    for (int u = 0; u < 2; u++)
    {
        const int r = (wave * 2 + u) * 16 + (lane >> 2), c = (lane & 3) ^ ((r >> 2) & 3);
        gx[u] = X + (long long) min(m0 + r, a.M - 1) * a.x_ld + c * 16;
        gw[u] = W + (long long) min(n0 + r, a.N - 1) * a.w_ld + c * 16;
    }
    auto issue_x = [&](int u, int stage, int slot) __attribute__((always_inline)) { dma16(gx[u] + (size_t) stage * BK, lds_base + slot * STAGE + (wave * 2 + u) * 1024); };
    auto issue_w = [&](int u, int stage, int slot) __attribute__((always_inline)) { dma16(gw[u] + (size_t) stage * BK, lds_base + slot * STAGE + TM * BK + (wave * 2 + u) * 1024); };

    v16 acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[i][j][v] = 0;

    const int nk = a.K >> 6; // whole stages, at least NST
    for (int t = 0; t < NST; t++)
    {
        issue_x(0, t, t);
        issue_x(1, t, t);
        issue_w(0, t, t);
        issue_w(1, t, t);
    }
    __builtin_amdgcn_s_waitcnt(vm_wait((NST - 1) * NREQ));
    __syncthreads();
    s_v8i fx[NI], fw[NJ];
#pragma unroll
    for (int i = 0; i < NI; i++) fx[i] = read_frag(lds, wm * WR + i * 32, lane);
#pragma unroll
    for (int j = 0; j < NJ; j++) fw[j] = read_frag(lds + TM * BK, wn * WC + j * 32, lane);

    // One stage: the products of stage t; behind the first, a wait until stage t + 1 has landed for every wavefront, then its
    // fragments, each right after the last use of the register it goes to, and the requests of stage t + 4 into the slot of stage t.
    // The wait is for this wavefront's reads of that slot as well: the last of them were issued at the end of the step before, and a
    // barrier does not wait for them, while the requests behind it come from other wavefronts.  (The second product needs them anyway: no
    // time is lost.  int8 4096^3 64.0 us, four products of fp8 2048 x 14336 x 4096 420.1, wait and barrier behind the second product 64.0 and 419.9.)
    auto step = [&](int t, auto waitc, auto loads, auto readnext) __attribute__((always_inline))
    {
        constexpr int  WAITC = decltype(waitc)::value;
        constexpr bool LOADS = decltype(loads)::value, RN = decltype(readnext)::value;
        const int      slot = t & 3;
        const char*    st = lds + ((t + 1) & 3) * STAGE;
        auto           mma = [&](int i, int j) __attribute__((always_inline)) { acc[i][j] = mma32<OPS>(fw[j], fx[i], acc[i][j]); };
        auto           rx = [&](int i) __attribute__((always_inline)) { if (RN) fx[i] = read_frag(st, wm * WR + i * 32, lane); };
        auto           rw = [&](int j) __attribute__((always_inline)) { if (RN) fw[j] = read_frag(st + TM * BK, wn * WC + j * 32, lane); };
        mma(0, 0);
        FENCE;
        if (RN)
        {
            __builtin_amdgcn_s_waitcnt(WAITC);
            __builtin_amdgcn_s_barrier();
        }
        FENCE;
        mma(0, 1);
        FENCE;
        rx(0);
        if (LOADS) issue_x(0, t + NST, slot);
        mma(1, 0);
        FENCE;
        mma(1, 1);
        FENCE;
        rx(1);
        if (LOADS) issue_x(1, t + NST, slot);
        mma(2, 0);
        FENCE;
        mma(2, 1);
        FENCE;
        rx(2);
        if (LOADS) issue_w(0, t + NST, slot);
        mma(3, 0);
        FENCE;
        rw(0);
        if (LOADS) issue_w(1, t + NST, slot);
        mma(3, 1);
        FENCE;
        rx(3);
        rw(1);
        FENCE;
    };
    using WM = std::integral_constant<int, landed_and_read((NST - 2) * NREQ)>;
    using T = std::true_type;
    using F = std::false_type;
    int t = 0;
    for (; t + NST + 1 < nk; t += 2)
    {
        step(t, WM {}, T {}, T {});
        step(t + 1, WM {}, T {}, T {});
    }
    if (t + NST < nk)
    {
        step(t, WM {}, T {}, T {});
        t++;
    }
    step(t, std::integral_constant<int, landed_and_read(2 * NREQ)> {}, F {}, T {});
    step(t + 1, std::integral_constant<int, landed_and_read(NREQ)> {}, F {}, T {});
    step(t + 2, std::integral_constant<int, landed_and_read(0)> {}, F {}, T {});
    step(t + 3, std::integral_constant<int, landed_and_read(0)> {}, F {}, F {});
    if (nk * BK < a.K)
    {
        // the codes behind the last whole stage, from registers
        const int k = nk * BK + (lane >> 5) * 32;
#pragma unroll
        for (int j = 0; j < NJ; j++)
        {
            const uint8_t* p = W + (long long) min(n0 + wn * WC + j * 32 + (lane & 31), a.N - 1) * a.w_ld;
            fw[j] = join(load16(p, k, a.K), load16(p, k + 16, a.K));
        }
#pragma unroll
        for (int i = 0; i < NI; i++)
        {
            const uint8_t* p = X + (long long) min(m0 + wm * WR + i * 32 + (lane & 31), a.M - 1) * a.x_ld;
            fx[i] = join(load16(p, k, a.K), load16(p, k + 16, a.K));
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[i][j] = mma32<OPS>(fw[j], fx[i], acc[i][j]);
        }
    }

    // ---- epilogue.  Accumulator register v of lane l is column 8 (v / 4) + 4 (l / 32) + v % 4 of row l % 32 of its block: one lane swap
    // per register pair leaves every lane with 16 consecutive columns of one row, and the rounded values pass through LDS (32 rows of 64
    // columns per wavefront, chunks swizzled by row), so that a store instruction writes whole lines.
    const int kg = lane >> 5, row = lane & 31;
    __syncthreads(); // the ring is idle
    float* sw_s = (float*) (lds + 64 * 1024);
    float* bias_s = sw_s + TN;
    if (threadIdx.x < TN)
    {
        const int n = min(n0 + (int) threadIdx.x, a.N - 1);
        sw_s[threadIdx.x] = a.sw ? a.sw[o.sw + n] : 1.0f;
        bias_s[threadIdx.x] = a.bias ? a.bias[o.sw + n] : 0.0f;
    }
    float sx[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) sx[i] = a.sx ? a.sx[o.sx + min(m0 + wm * WR + i * 32 + row, a.M - 1)] : 1.0f;
    __syncthreads();
    const bool has_bias = a.bias != nullptr;
    const float alpha = a.alpha;
    auto        walk = [&](auto esz_c, auto convert) __attribute__((always_inline))
    {
        constexpr int ESZ = decltype(esz_c)::value, RB = 64 * ESZ, CPR = RB / 16, NRD = RB / 32;
        char*         stg = lds + wave * (32 * RB);
        const int     swz = row & 7;
        uint8_t*      out = (uint8_t*) a.out + (o.out + (long long) (m0 + wm * WR) * a.out_ld + n0 + wn * WC) * ESZ;
#pragma unroll
        for (int i = 0; i < NI; i++)
        {
#pragma unroll
            for (int j = 0; j < NJ; j++)
            {
                one val[16];
#pragma unroll
                for (int q = 0; q < 2; q++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                    {
                        uint32_t lo, hi;
                        __builtin_memcpy(&lo, (const one[1]) {acc[i][j][4 * q + r]}, 4);
                        __builtin_memcpy(&hi, (const one[1]) {acc[i][j][8 + 4 * q + r]}, 4);
                        const auto s = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
                        const uint32_t s0 = s[0], s1 = s[1];
                        __builtin_memcpy(&val[8 * q + r], &s0, 4);
                        __builtin_memcpy(&val[8 * q + 4 + r], &s1, 4);
                    }
                uint32_t pk[4 * ESZ];
                convert(val, sx[i], sw_s + wn * WC + j * 32 + kg * 16, bias_s + wn * WC + j * 32 + kg * 16, pk);
#pragma unroll
                for (int h = 0; h < ESZ; h++)
                    *(lds_v4u*) (stg + row * RB + ((((j * 2 + kg) * ESZ + h) ^ swz) << 4)) = lds_v4u {pk[4 * h], pk[4 * h + 1], pk[4 * h + 2], pk[4 * h + 3]};
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int r = 0; r < NRD; r++)
            {
                const int     q = r * 64 + lane, rr = q / CPR, lc = q % CPR;
                const lds_v4u v = *(const lds_v4u*) (stg + rr * RB + ((lc ^ (rr & 7)) << 4));
                const int     left = a.N - (n0 + wn * WC + lc * (16 / ESZ)); // outputs of this chunk that exist
                if (m0 + wm * WR + i * 32 + rr < a.M && left > 0)
                {
                    uint8_t* p = out + (long long) (i * 32 + rr) * a.out_ld * ESZ + lc * 16;
                    if (left >= 16 / ESZ) __builtin_nontemporal_store(v, (any_v4u*) p);
                    else
                    {
                        for (int e = 0; e < left; e++)
                        {
                            const uint32_t word = v[e * ESZ / 4];
                            if constexpr (ESZ == 4) ((uint32_t*) p)[e] = word;
                            else
                                ((uint16_t*) p)[e] = (uint16_t) (word >> (16 * (e & 1)));
                        }
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    auto scaled = [&](const one (&val)[16], float s, const float* sw, const float* bias, float (&v)[16]) __attribute__((always_inline))
    {
#pragma unroll
        for (int c = 0; c < 16; c++) v[c] = scaled_value(val[c], alpha, s, sw[c], bias[c], has_bias);
    };
    typedef float e_v2f __attribute__((ext_vector_type(2)));
    if (a.out_type == SCALED_OUT_BF16)
        walk(std::integral_constant<int, 2>(), [&](const one(&val)[16], float s, const float* sw, const float* bias, uint32_t(&pk)[8]) __attribute__((always_inline)) {
            float v[16];
            scaled(val, s, sw, bias, v);
#pragma unroll
            for (int c = 0; c < 8; c++)
            {
                typedef __bf16 b2 __attribute__((ext_vector_type(2)));
                const b2       h = __builtin_convertvector(e_v2f {v[2 * c], v[2 * c + 1]}, b2);
                __builtin_memcpy(&pk[c], &h, 4);
            }
        });
    else if (a.out_type == SCALED_OUT_FP16)
        walk(std::integral_constant<int, 2>(), [&](const one(&val)[16], float s, const float* sw, const float* bias, uint32_t(&pk)[8]) __attribute__((always_inline)) {
            float v[16];
            scaled(val, s, sw, bias, v);
#pragma unroll
            for (int c = 0; c < 8; c++)
            {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2         h = __builtin_convertvector(e_v2f {v[2 * c], v[2 * c + 1]}, h2);
                __builtin_memcpy(&pk[c], &h, 4);
            }
        });
    else if constexpr (OPS < 0) // (fp8 operands have 16-bit outputs)
    {
        const bool raw = a.out_type == SCALED_OUT_INT32;
        walk(std::integral_constant<int, 4>(), [&](const one(&val)[16], float s, const float* sw, const float* bias, uint32_t(&pk)[16]) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < 16; c++) pk[c] = raw ? (uint32_t) val[c] : __float_as_uint(scaled_value(val[c], alpha, s, sw[c], bias[c], has_bias));
        });
    }
}

template<int OPS>
hipError_t start(const ScaledGemmArgs& a, hipStream_t s)
{
    if (hipError_t e = allow_lds((const void*) scaled_gemm_large_kernel<OPS>, LDS_BYTES)) return e;
    const dim3 grid((unsigned) (((a.M + TM - 1) / TM) * ((a.N + TN - 1) / TN)), (unsigned) (a.batch[0] * a.batch[1] * a.batch[2]));
    hipLaunchKernelGGL((scaled_gemm_large_kernel<OPS>), grid, dim3(512), LDS_BYTES, s, a);
    return hipGetLastError();
}
} // namespace

hipError_t launch_scaled_gemm_large(const ScaledGemmArgs& a, hipStream_t s)
{
    if (a.int8) return start<-1>(a, s);
    switch (a.fmt)
    {
        case 0: return start<0>(a, s);
        case 1: return start<1>(a, s);
        case 2: return start<2>(a, s);
        default: return start<3>(a, s);
    }
}
} // namespace mme
