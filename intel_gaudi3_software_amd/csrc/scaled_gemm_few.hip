// scaled_gemm_few.hip -- the scaled product for few rows of x (tokens being generated), or few outputs in all.
//
// Bound by reading w once.  A workgroup owns 16 NT rows of w and 8, 16 or 32 rows of x; its wavefronts share out the reduction, 128 k at a
// time in turn, and share nothing until the end, when their partial sums meet in LDS and are added in the order of the wavefronts.
//
// The 16 x 16 matrix instructions want neighbouring lanes on neighbouring rows.  Loaded that way from memory every lane is a line
// of its own and a compute unit takes in 17 bytes a clock; so a wavefront brings a stage (128 k of every row) into a ring of its
// own in LDS, eight neighbouring lanes on the eight 16-byte chunks of a line, and reads it back in the instructions' layout (chunk c
// of row r lies at position c ^ (r / 2 & 7): the sixteen rows of a read meet every bank once).  Sixteen tokens, 4096 x 14336: 11.9 us,
// 4.9 TB/s of w and x (loaded straight into the instructions' layout: 15.2); 14336 x 4096: 12.5 us, 4.7 TB/s; one token, 4096 x 4096:
// 5.6 us, most of it the launch.  Where all rows are 16-byte aligned the copies are direct, memory to LDS, and D stages are in
// flight; elsewhere they pass through registers.  The last K % 128 codes are loaded by hand.
#include "scaled_gemm_common.hpp"

namespace mme
{
namespace
{
// NT: 16-row tiles of w; XR: rows of x (8, 16 or 32); D: stages of a wavefront's ring
template<int OPS, int NT, int XR, int WAVES, int D, bool ALIGNED>
__global__ __launch_bounds__(WAVES * 64) void scaled_gemm_few_kernel(const ScaledGemmArgs a)
{
    typedef typename Sums<OPS>::v4  v4;
    typedef typename Sums<OPS>::one one;
    constexpr int MT = XR <= 16 ? 1 : XR / 16; // 16-row tiles of x
    constexpr int QW = 2 * NT, QX = XR / 8, Q = QW + QX; // requests per stage: eight rows of 128 bytes each
    constexpr int STAGE = Q * 1024;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int          lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // consecutive tiles go to one XCD (workgroups are dealt out to the eight in turn), those over one panel of w next to each other
    const int tiles_m = (a.M + XR - 1) / XR, total = (int) gridDim.x, xcd = (int) blockIdx.x & 7;
    const int tile = xcd * (total >> 3) + min(xcd, total & 7) + ((int) blockIdx.x >> 3);
    const int m0 = (tile % tiles_m) * XR, n0 = (tile / tiles_m) * (16 * NT);
    const BatchOffsets o = batch_offsets(a, blockIdx.y);
    const int          row8 = lane >> 3; // request side: row of eight
    auto chunk = [&](int q) __attribute__((always_inline)) { return (lane & 7) ^ swizzle(q * 8 + row8); }; // and the 16-byte chunk of its line
    char*              ring = lds + wave * (D * STAGE);
    const uint32_t     ring_off = (uint32_t) (uintptr_t) lds + wave * (D * STAGE);
    const uint8_t*     w = a.w + o.w;
    const uint8_t*     x = a.x + o.x;
    // (rows beyond the last read the last: their outputs are not stored)
    const uint8_t* src[Q];
#pragma unroll
    for (int q = 0; q < QW; q++) src[q] = w + (long long) min(n0 + q * 8 + row8, a.N - 1) * a.w_ld + chunk(q) * 16 + wave * 128;
#pragma unroll
    for (int q = 0; q < QX; q++) src[QW + q] = x + (long long) min(m0 + q * 8 + row8, a.M - 1) * a.x_ld + chunk(q) * 16 + wave * 128;

    v4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int v = 0; v < 4; v++) acc[i][j][v] = 0;

    const int  whole = a.K >> 7;                                                 // whole stages of the reduction
    const int  mine = whole > wave ? (whole - wave + WAVES - 1) / WAVES : 0;     // this wavefront's
    const int  r = lane & 15, g = lane >> 4;
    auto       multiply = [&](const char* st) __attribute__((always_inline))
    {
        // k order within a stage: chunk g, then chunk g + 4, the same for both operands
        auto frag = [&](int row) __attribute__((always_inline))
        {
            const char* p = st + row * 128;
            return join(*(const s_v4i*) (p + ((g ^ swizzle(row)) << 4)), *(const s_v4i*) (p + (((g + 4) ^ swizzle(row)) << 4)));
        };
        s_v8i fw[NT], fx[MT];
#pragma unroll
        for (int j = 0; j < NT; j++) fw[j] = frag(j * 16 + r);
#pragma unroll
        for (int i = 0; i < MT; i++) fx[i] = frag(16 * NT + i * 16 + (XR == 8 ? r & 7 : r));
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = mma16<OPS>(fw[j], fx[i], acc[i][j]);
    };
    if constexpr (ALIGNED)
    {
        auto issue = [&](int t, int slot) __attribute__((always_inline))
        {
#pragma unroll
            for (int q = 0; q < Q; q++) dma16(src[q] + (size_t) t * (WAVES * 128), ring_off + slot * STAGE + q * 1024);
        };
        // (every stage of the ring is requested and waited for in turn; stages beyond the last are requests of the last one again, so
        // that the count of requests in flight is always the same)
        if (mine > 0)
        {
#pragma unroll
            for (int t = 0; t < D; t++) issue(min(t, mine - 1), t);
            int slot = 0;
#pragma unroll 1
            for (int t = 0; t < mine; t++)
            {
                __builtin_amdgcn_s_waitcnt(vm_wait((D - 1) * Q));
                asm volatile("" ::: "memory");
                multiply(ring + slot * STAGE);
                // the fragments are in registers before their slot is written again
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (t + D < mine) issue(t + D, slot);
                else
                    issue(mine - 1, slot);
                slot = slot + 1 == D ? 0 : slot + 1;
            }
            __builtin_amdgcn_s_waitcnt(vm_wait(0)); // (the ring is used for the sums below)
        }
    }
    else
    {
        s_v4i  held[D][Q];
        auto   load = [&](int t, int d) __attribute__((always_inline))
        {
#pragma unroll
            for (int q = 0; q < Q; q++)
            {
                const u128_any u = *(const u128_any*) (src[q] + (size_t) t * (WAVES * 128));
                held[d][q] = s_v4i {(int) u.v[0], (int) u.v[1], (int) u.v[2], (int) u.v[3]};
            }
        };
#pragma unroll
        for (int d = 0; d < D; d++)
            if (d < mine) load(d, d);
#pragma unroll 1
        for (int t0 = 0; t0 < mine; t0 += D)
#pragma unroll
            for (int d = 0; d < D; d++)
                if (t0 + d < mine)
                {
#pragma unroll
                    for (int q = 0; q < Q; q++) *(s_v4i*) (ring + d * STAGE + q * 1024 + lane * 16) = held[d][q];
                    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                    if (t0 + D + d < mine) load(t0 + D + d, d);
                    multiply(ring + d * STAGE);
                }
    }
    const int rest = whole * 128;
    if (rest < a.K && wave == whole % WAVES)
    {
        const int k = rest + g * 16;
        s_v8i     fx[MT];
#pragma unroll
        for (int i = 0; i < MT; i++)
        {
            const uint8_t* p = x + (long long) min(m0 + i * 16 + r, a.M - 1) * a.x_ld;
            fx[i] = join(load16(p, k, a.K), load16(p, k + 64, a.K));
        }
#pragma unroll
        for (int j = 0; j < NT; j++)
        {
            const uint8_t* p = w + (long long) min(n0 + j * 16 + r, a.N - 1) * a.w_ld;
            const s_v8i    fw = join(load16(p, k, a.K), load16(p, k + 64, a.K));
#pragma unroll
            for (int i = 0; i < MT; i++) acc[i][j] = mma16<OPS>(fw, fx[i], acc[i][j]);
        }
    }
    __syncthreads();
    one* part = (one*) lds; // [wave][tile][lane][4]
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) *(v4*) (part + ((wave * MT * NT + i * NT + j) * 64 + lane) * 4) = acc[i][j];
    __syncthreads();
    // consecutive lanes on consecutive groups of four columns of a row
    for (int t = threadIdx.x; t < MT * NT * 64; t += WAVES * 64)
    {
        const int row = t / (4 * NT), group = t % (4 * NT), l = (group & 3) * 16 + (row & 15), block = (row >> 4) * NT + (group >> 2);
        const int m = m0 + row, n = n0 + group * 4;
        if (m >= a.M || n >= a.N) continue;
        const float   sx = scale_of_row(a, o, m);
        const Columns c = columns_of(a, o, n);
        v4            sum = *(const v4*) (part + (block * 64 + l) * 4);
#pragma unroll
        for (int q = 1; q < WAVES; q++) sum += *(const v4*) (part + ((q * MT * NT + block) * 64 + l) * 4);
        const one s[4] = {sum[0], sum[1], sum[2], sum[3]};
        store_scaled4(a, o, m, n, sx, c, s);
    }
}

template<int OPS, int NT, int XR, int WAVES, int D, bool ALIGNED>
hipError_t start(const ScaledGemmArgs& a, hipStream_t s)
{
    constexpr int MT = XR <= 16 ? 1 : XR / 16;
    constexpr int ring = WAVES * D * (16 * NT + XR) * 128, sums = WAVES * MT * NT * 1024, lds = ring > sums ? ring : sums;
    static_assert(lds <= 160 * 1024, "LDS of a compute unit");
    if (hipError_t e = allow_lds((const void*) scaled_gemm_few_kernel<OPS, NT, XR, WAVES, D, ALIGNED>, lds)) return e;
    const dim3 grid((unsigned) (((a.M + XR - 1) / XR) * ((a.N + 16 * NT - 1) / (16 * NT))), (unsigned) (a.batch[0] * a.batch[1] * a.batch[2]));
    hipLaunchKernelGGL((scaled_gemm_few_kernel<OPS, NT, XR, WAVES, D, ALIGNED>), grid, dim3(WAVES * 64), lds, s, a);
    return hipGetLastError();
}

template<int OPS>
hipError_t start_shaped(const ScaledGemmArgs& a, hipStream_t s)
{
    if (!a.aligned)
    {
        if (a.tile_m == 8) return start<OPS, 1, 8, 8, 4, false>(a, s);
        return a.tile_m == 16 ? start<OPS, 1, 16, 8, 3, false>(a, s) : start<OPS, 1, 32, 8, 2, false>(a, s);
    }
    if (a.tile_m == 8) return a.tile_n == 1 ? start<OPS, 1, 8, 8, 6, true>(a, s) : a.tile_n == 2 ? start<OPS, 2, 8, 8, 4, true>(a, s) : start<OPS, 4, 8, 4, 4, true>(a, s);
    if (a.tile_m == 16) return a.tile_n == 1 ? start<OPS, 1, 16, 8, 4, true>(a, s) : a.tile_n == 2 ? start<OPS, 2, 16, 8, 3, true>(a, s) : start<OPS, 4, 16, 4, 4, true>(a, s);
    return a.tile_n == 1 ? start<OPS, 1, 32, 8, 3, true>(a, s) : a.tile_n == 2 ? start<OPS, 2, 32, 4, 5, true>(a, s) : start<OPS, 4, 32, 4, 3, true>(a, s);
}
} // namespace

hipError_t launch_scaled_gemm_few(const ScaledGemmArgs& a, hipStream_t s)
{
    if (a.int8) return start_shaped<-1>(a, s);
    switch (a.fmt)
    {
        case 0: return start_shaped<0>(a, s);
        case 1: return start_shaped<1>(a, s);
        case 2: return start_shaped<2>(a, s);
        default: return start_shaped<3>(a, s);
    }
}
} // namespace mme
