// scaled_gemm.hip -- the scaled product: the choice of the kernel form, and the general form, which takes every size, stride and
// alignment.
//
// General form: 64 x 64 outputs per workgroup of four wavefronts (2 x 2, 32 x 32 each), 64 k per step.  Operands go through
// registers into LDS (rows of 64 codes on a pitch of 80 bytes), loaded 16 bytes at a time at any alignment; codes beyond K are
// replaced by zeros in both operands, so that nothing behind a row's end reaches a sum.
#include <mutex>
#include <utility>
#include <vector>

#include "scaled_gemm_common.hpp"

namespace mme
{
namespace
{
constexpr int GT = 64, GK = 64, GP = 80;

template<int OPS>
__global__ __launch_bounds__(256) void scaled_gemm_general_kernel(const ScaledGemmArgs a)
{
    __shared__ __attribute__((aligned(16))) char lds[2][GT * GP];
    const int          tiles_n = (a.N + GT - 1) / GT;
    const int          m0 = (int) (blockIdx.x / tiles_n) * GT, n0 = (int) (blockIdx.x % tiles_n) * GT;
    const BatchOffsets o = batch_offsets(a, blockIdx.y);
    const int          lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
    // each lane brings 16 codes of one row of each operand per step (a row beyond the last reads the last: its outputs are not stored)
    const int      r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
    const uint8_t* xr = a.x + o.x + (long long) min(m0 + r, a.M - 1) * a.x_ld;
    const uint8_t* wr = a.w + o.w + (long long) min(n0 + r, a.N - 1) * a.w_ld;
    typename Sums<OPS>::v16 acc;
#pragma unroll
    for (int v = 0; v < 16; v++) acc[v] = 0;
    s_v4i xv = load16(xr, c, a.K), wv = load16(wr, c, a.K);
    for (int k0 = 0; k0 < a.K; k0 += GK)
    {
        *(s_v4i*) (lds[0] + r * GP + c) = xv;
        *(s_v4i*) (lds[1] + r * GP + c) = wv;
        __syncthreads();
        if (k0 + GK < a.K)
        {
            xv = load16(xr, k0 + GK + c, a.K);
            wv = load16(wr, k0 + GK + c, a.K);
        }
        auto frag = [&](const char* base, int row) __attribute__((always_inline))
        {
            const char* p = base + (row + (lane & 31)) * GP + (lane >> 5) * 32;
            return join(*(const s_v4i*) p, *(const s_v4i*) (p + 16));
        };
        acc = mma32<OPS>(frag(lds[1], wn * 32), frag(lds[0], wm * 32), acc);
        __syncthreads();
    }
    const int m = m0 + wm * 32 + (lane & 31);
    if (m >= a.M) return;
#pragma unroll
    for (int g = 0; g < 4; g++)
    {
        const int n = n0 + wn * 32 + 8 * g + 4 * (lane >> 5);
        const typename Sums<OPS>::one sum[4] = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
        if (n < a.N) store_scaled4(a, o, m, n, sum);
    }
}
} // namespace

hipError_t allow_lds(const void* kernel, int bytes)
{
    static std::mutex                               mutex;
    static std::vector<std::pair<const void*, int>> done;
    int                                             device = 0;
    if (hipError_t e = hipGetDevice(&device)) return e;
    const std::lock_guard<std::mutex> lock(mutex);
    for (const auto& d : done)
        if (d.first == kernel && d.second == device) return hipSuccess;
    if (hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
    done.emplace_back(kernel, device);
    return hipSuccess;
}

void plan_scaled_gemm(ScaledGemmArgs& a, int num_cus, int (&figures)[4])
{
    a.form = SCALED_FORM_GENERAL;
    a.split_k = 1;
    figures[0] = 0, figures[1] = GT, figures[2] = 1, figures[3] = 4;
    bool aligned = (uintptr_t) a.x % 16 == 0 && (uintptr_t) a.w % 16 == 0 && (a.M == 1 || a.x_ld % 16 == 0) && (a.N == 1 || a.w_ld % 16 == 0);
    for (int d = 0; d < 3; d++) aligned = aligned && a.x_bs[d] % 16 == 0 && a.w_bs[d] % 16 == 0;
    a.aligned = aligned;
    if (a.M <= 32)
    {
        a.form = SCALED_FORM_FEW;
        scaled_gemm_few_shape(a, num_cus);
        figures[0] = 3, figures[1] = a.tile_m, figures[3] = a.waves;
    }
}

size_t scaled_gemm_partial_bytes(const ScaledGemmArgs& a)
{
    return a.split_k > 1 ? (size_t) a.split_k * a.batch[0] * a.batch[1] * a.batch[2] * a.M * a.N * 4 : 0;
}

hipError_t launch_scaled_gemm(const ScaledGemmArgs& a, hipStream_t s)
{
    if (a.form == SCALED_FORM_FEW) return launch_scaled_gemm_few(a, s);
    const dim3 grid((unsigned) (((a.M + GT - 1) / GT) * ((a.N + GT - 1) / GT)), (unsigned) (a.batch[0] * a.batch[1] * a.batch[2]));
    auto       go = [&](auto ops) { hipLaunchKernelGGL((scaled_gemm_general_kernel<decltype(ops)::value>), grid, dim3(256), 0, s, a); };
    if (a.int8) go(std::integral_constant<int, -1>());
    else if (a.fmt == 0)
        go(std::integral_constant<int, 0>());
    else if (a.fmt == 1)
        go(std::integral_constant<int, 1>());
    else if (a.fmt == 2)
        go(std::integral_constant<int, 2>());
    else
        go(std::integral_constant<int, 3>());
    return hipGetLastError();
}
} // namespace mme
