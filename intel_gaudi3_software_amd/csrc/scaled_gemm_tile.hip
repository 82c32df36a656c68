// scaled_gemm_tile.hip -- the scaled product with tiles of 64 x 64 or 128 x 128 outputs.
//
// For products whose outputs are too few for the 256 x 256 tiles: bound by bringing operands into LDS (a compute unit takes in about
// 80 GB/s when all of them do, 57 bytes a clock when few do).  Four wavefronts multiply, 2 x 2 over the tile, and four others do
// nothing but request: a request holds its wavefront up for as long as the products of half a stage take, and with both in one
// wavefront, requests in a row or spread between the products, 32 stages of the 128 x 128 tile took 15.6 us or more; apart 13.9
// (reading and multiplying alone 10.7, requesting alone 8.8).
// A stage is 128 k of every row of the tile, eight neighbouring lanes on a line (chunk c of row r lies at position c ^ (r / 2 & 7)); NST
// stages form a ring.  A stage is multiplied in two halves, each while the fragments of the next are read; one barrier per stage, in its
// middle: behind it the next stage has landed, and everybody has the rest of this one in registers, so its slot is requested
// again.  Where all rows are 16-byte aligned the copies go directly from memory to LDS; elsewhere they pass through registers, up to
// four stages of loads ahead (1000 x 4096 x 4097 35.2 us, 1000 x 4096 x 4096 24).
// Wavefronts that share out a stage's k instead of the tile's outputs (each byte of LDS is then read once, not twice) were slower: 64 x 64,
// 250 x 4096 x 14336 25.4 -> 26.1 us, 512 x 4096 x 4096 15.7 -> 19.8 (one workgroup per compute unit for the longer stages).
// No split of the reduction: its partial sums and second kernel cost 8 us and more, and where few tiles have a long reduction the
// form for few rows, whose wavefronts share it out, is faster at any number of rows.
#include "scaled_gemm_common.hpp"

namespace mme
{
namespace
{
constexpr int COPIERS = 4; // wavefronts that request the operands

template<int OPS, int NI, int NJ, int NST, bool ALIGNED>
__global__ __launch_bounds__((4 + COPIERS) * 64) void scaled_gemm_tile_kernel(const ScaledGemmArgs a)
{
    constexpr int WM = 2, WN = 2, WAVES = WM * WN, TM = WM * NI * 32, TN = WN * NJ * 32, ROWS = TM + TN;
    constexpr int STAGE = ROWS * 128, Q = ROWS / 8 / COPIERS; // requests per copying wavefront and stage: eight rows each
    constexpr int P = 16 / Q; // stages that pass through registers at a time
    static_assert(Q * 8 * COPIERS == ROWS, "whole requests");
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    typedef typename Sums<OPS>::v16 v16;
    typedef typename Sums<OPS>::one one;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    const int tiles_m = (a.M + TM - 1) / TM;
    // consecutive tiles go to one XCD (workgroups are dealt out to the eight in turn), the tiles over one panel of w next to each other
    const int total = (int) gridDim.x, xcd = (int) blockIdx.x & 7, per = total >> 3, extra = total & 7;
    const int L = xcd * per + min(xcd, extra) + ((int) blockIdx.x >> 3);
    const int          m0 = (L % tiles_m) * TM, n0 = (L / tiles_m) * TN;
    const BatchOffsets o = batch_offsets(a, blockIdx.y);
    const int whole = a.K >> 7, nk = (a.K + 127) >> 7; // stages: whole ones, and all (codes behind a row's end are zeros)
    v16       acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) acc[i][j][v] = 0;
    // Both kinds of wavefronts meet nk + 1 barriers: before stage 0 and in the middle of every stage.
    if (nk > 0 && wave >= WAVES)
    {
        const int      copier = wave - WAVES, row8 = lane >> 3;
        const uint32_t lds_off = (uint32_t) (uintptr_t) lds;
        const uint8_t* src[Q]; // this lane's chunk of stage 0
        int            c16[Q]; // where it lies in its row
#pragma unroll
        for (int q = 0; q < Q; q++)
        {
            const int r = (q * COPIERS + copier) * 8 + row8; // row of the stage: x first
            c16[q] = ((lane & 7) ^ swizzle(r)) * 16;
            src[q] = c16[q] + (r < TM ? a.x + o.x + (long long) min(m0 + r, a.M - 1) * a.x_ld : a.w + o.w + (long long) min(n0 + r - TM, a.N - 1) * a.w_ld);
        }
        // 16 codes of stage t on their way through registers: a chunk that crosses the row's end is loaded as the row's last sixteen
        // codes and moved into place only when it is put into LDS, so that the loads behind it stay in flight
        auto load = [&](int t, int q) __attribute__((always_inline))
        {
            const u128_any u = *(const u128_any*) (src[q] + min(t * 128, a.K - 16 - c16[q]));
            return s_v4i {(int) u.v[0], (int) u.v[1], (int) u.v[2], (int) u.v[3]};
        };
        auto in_place = [&](s_v4i v, int t, int q) __attribute__((always_inline)) { return moved_down(v, t * 128 + c16[q] - (a.K - 16)); };
        auto put = [&](s_v4i v, int slot, int q) __attribute__((always_inline)) { *(s_v4i*) (lds + slot * STAGE + (q * COPIERS + copier) * 1024 + lane * 16) = v; };
        if constexpr (ALIGNED)
        {
            auto issue = [&](int t, int slot) __attribute__((always_inline))
            {
#pragma unroll
                for (int q = 0; q < Q; q++) dma16(src[q] + (size_t) t * 128, lds_off + slot * STAGE + (q * COPIERS + copier) * 1024);
            };
            // a last stage that K cuts off
            auto last_stage = [&](int slot) __attribute__((always_inline))
            {
                s_v4i v[Q];
#pragma unroll
                for (int q = 0; q < Q; q++) v[q] = load(whole, q);
#pragma unroll
                for (int q = 0; q < Q; q++) put(in_place(v[q], whole, q), slot, q);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            };
            // stage t has landed once at most the requests of the whole stages behind it, up to `last`, are outstanding
            auto landed = [&](int t, int last) __attribute__((always_inline))
            {
                const int behind = min(last, whole - 1) - t;
                if (NST > 3 && behind >= 3) __builtin_amdgcn_s_waitcnt(vm_wait(3 * Q));
                else if (NST > 2 && behind >= 2)
                    __builtin_amdgcn_s_waitcnt(vm_wait(2 * Q));
                else if (behind >= 1)
                    __builtin_amdgcn_s_waitcnt(vm_wait(Q));
                else
                    __builtin_amdgcn_s_waitcnt(vm_wait(0));
            };
#pragma unroll
            for (int t = 0; t < NST; t++)
                if (t < whole) issue(t, t);
            if (whole < NST && whole < nk) last_stage(whole);
            landed(0, NST - 1);
            __builtin_amdgcn_s_barrier();
            int slot = 0;
#pragma unroll 1
            for (int t = 0; t < nk; t++)
            {
                landed(t + 1, t + NST - 1);
                __builtin_amdgcn_s_barrier(); // and the rest of stage t is in the others' registers: its slot is free
                if (t + NST < whole) issue(t + NST, slot);
                else if (t + NST < nk)
                    last_stage(slot);
                slot = slot + 1 == NST ? 0 : slot + 1;
            }
        }
        else
        {
            // P stages are held, a row of fewer than sixteen codes (one stage) only when it is put down
            s_v4i      held[P][Q];
            const bool sixteen = a.K >= 16;
            auto       take = [&](int t, int d) __attribute__((always_inline))
            {
#pragma unroll
                for (int q = 0; q < Q; q++) held[d][q] = load(t, q);
            };
            auto put_stage = [&](int t, int slot, int d) __attribute__((always_inline))
            {
                if (t == whole)
                {
#pragma unroll
                    for (int q = 0; q < Q; q++) held[d][q] = sixteen ? in_place(held[d][q], t, q) : load16(src[q] - c16[q], c16[q], a.K);
                }
#pragma unroll
                for (int q = 0; q < Q; q++) put(held[d][q], slot, q);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            };
            if (sixteen)
            {
#pragma unroll
                for (int d = 0; d < P; d++) take(d, d);
            }
            put_stage(0, 0, 0);
            if (sixteen) take(P, 0);
            __builtin_amdgcn_s_barrier();
            int slot = 0;
            // stage t + 1 is held in set (t + 1) % P
#pragma unroll 1
            for (int t0 = 0; t0 < nk; t0 += P)
#pragma unroll
                for (int d = 0; d < P; d++)
                    if (t0 + d < nk)
                    {
                        slot = slot + 1 == NST ? 0 : slot + 1;
                        put_stage(t0 + d + 1, slot, (d + 1) % P);
                        if (sixteen) take(t0 + d + 1 + P, (d + 1) % P);
                        __builtin_amdgcn_s_barrier();
                    }
        }
    }
    else if (nk > 0)
    {
        auto read = [&](s_v8i(&fx)[NI], s_v8i(&fw)[NJ], const char* st, int half) __attribute__((always_inline))
        {
            auto frag = [&](int row) __attribute__((always_inline))
            {
                const char* p = st + row * 128;
                const int   c = half * 4 + 2 * (lane >> 5);
                return join(*(const s_v4i*) (p + ((c ^ swizzle(row)) << 4)), *(const s_v4i*) (p + (((c + 1) ^ swizzle(row)) << 4)));
            };
#pragma unroll
            for (int i = 0; i < NI; i++) fx[i] = frag((wm * NI + i) * 32 + (lane & 31));
#pragma unroll
            for (int j = 0; j < NJ; j++) fw[j] = frag(TM + (wn * NJ + j) * 32 + (lane & 31));
        };
        auto multiply = [&](const s_v8i(&fx)[NI], const s_v8i(&fw)[NJ]) __attribute__((always_inline))
        {
#pragma unroll
            for (int i = 0; i < NI; i++)
#pragma unroll
                for (int j = 0; j < NJ; j++) acc[i][j] = mma32<OPS>(fw[j], fx[i], acc[i][j]);
        };
        // the halves of a stage in turn: one is multiplied while the fragments of the next are on their way from LDS
        s_v8i fx0[NI], fw0[NJ], fx1[NI], fw1[NJ];
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read(fx0, fw0, lds, 0);
        int slot = 0;
#pragma unroll 1
        for (int t = 0; t < nk; t++)
        {
            const int next = slot + 1 == NST ? 0 : slot + 1;
            read(fx1, fw1, lds + slot * STAGE, 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(fx0, fw0);
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            read(fx0, fw0, lds + next * STAGE, 0); // (behind the last stage: that stage again, not used)
            __builtin_amdgcn_sched_barrier(0);
            multiply(fx1, fw1);
            __builtin_amdgcn_sched_barrier(0);
            slot = next;
        }
    }
    // the sums pass through LDS, half of the tile's rows at a time, so that consecutive lanes store consecutive groups of four columns
    // of a row (the pitch puts rows that are stored together into different banks)
    typedef typename Sums<OPS>::v4 v4;
    constexpr int PITCH = TN + 4, HALF = TM / 2, LANES_N = TN / 4, ROWS_AT_A_TIME = (WAVES + COPIERS) * 64 / LANES_N;
    static_assert(HALF * PITCH * 4 <= NST * STAGE, "half of the sums fit the ring");
    one*          sums = (one*) lds;
    const int     n = n0 + ((int) threadIdx.x % LANES_N) * 4;
    const Columns cols = columns_of(a, o, n);
    float         sx[TM / ROWS_AT_A_TIME];
#pragma unroll
    for (int q = 0; q < TM / ROWS_AT_A_TIME; q++) sx[q] = scale_of_row(a, o, m0 + q * ROWS_AT_A_TIME + (int) threadIdx.x / LANES_N);
#pragma unroll
    for (int h = 0; h < 2; h++)
    {
        __syncthreads();
        if (wave < WAVES && wm == h)
#pragma unroll
            for (int i = 0; i < NI; i++)
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        *(v4*) (sums + (i * 32 + (lane & 31)) * PITCH + (wn * NJ + j) * 32 + 8 * g + 4 * (lane >> 5)) =
                            v4 {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        __syncthreads();
#pragma unroll
        for (int q = 0; q < HALF / ROWS_AT_A_TIME; q++)
        {
            const int row = q * ROWS_AT_A_TIME + (int) threadIdx.x / LANES_N, m = m0 + h * HALF + row;
            if (m >= a.M || n >= a.N) continue;
            const v4  v = *(const v4*) (sums + row * PITCH + n - n0);
            const one s[4] = {v[0], v[1], v[2], v[3]};
            store_scaled4(a, o, m, n, sx[h * (HALF / ROWS_AT_A_TIME) + q], cols, s);
        }
    }
}

template<int OPS, int NI, int NJ, int NST, bool ALIGNED>
hipError_t start(const ScaledGemmArgs& a, hipStream_t s)
{
    constexpr int TM = NI * 64, TN = NJ * 64, lds = NST * (TM + TN) * 128;
    static_assert(lds <= 160 * 1024, "LDS of a compute unit");
    if (hipError_t e = allow_lds((const void*) scaled_gemm_tile_kernel<OPS, NI, NJ, NST, ALIGNED>, lds)) return e;
    const dim3 grid((unsigned) (((a.M + TM - 1) / TM) * ((a.N + TN - 1) / TN)), (unsigned) (a.batch[0] * a.batch[1] * a.batch[2]));
    hipLaunchKernelGGL((scaled_gemm_tile_kernel<OPS, NI, NJ, NST, ALIGNED>), grid, dim3((4 + COPIERS) * 64), lds, s, a);
    return hipGetLastError();
}

template<int OPS>
hipError_t start_shaped(const ScaledGemmArgs& a, hipStream_t s)
{
    const bool direct = a.aligned && a.K >= 16;
    if (a.tile_m == 64) return direct ? start<OPS, 1, 1, 4, true>(a, s) : start<OPS, 1, 1, 4, false>(a, s);
    return direct ? start<OPS, 2, 2, 4, true>(a, s) : start<OPS, 2, 2, 4, false>(a, s);
}
} // namespace

hipError_t launch_scaled_gemm_tile(const ScaledGemmArgs& a, hipStream_t s)
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
