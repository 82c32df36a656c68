// scaled_gemm.hip -- the scaled product: the choice of the kernel form.
#include <mutex>
#include <utility>
#include <vector>

#include "scaled_kernels.hpp"

namespace mme
{
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

// What a form is expected to take: 3 us for the call, and for every round of workgroups over the compute units a fixed part (the first
// operands' way, the sums' way out) and one per 1024 k.  The constants are fitted to 41 products, 64 x 14336 x 4096 to 16384 x 512 x
// 320, in every form that takes them; the estimates' order is the measured one except where the first two are within 5 %.  Measured
// in us (estimated), M x N x K, int8 -> bf16, the best form and the next:
//   64 x 1024 x 16384     32 x 16 11.5 (14.8), 32 x 32 13.9        512 x 4096 x 4096     64 x 64 16.6 (18.6), 128 x 128 21.5
//   250 x 4096 x 14336    64 x 64 26.3 (26.3), 32 x 64 36.7        600 x 8192 x 1024     64 x 64 16.0 (18.8), 256 x 256 17.7
//   1024 x 4096 x 4096    128 x 128 24.0 (23.6), 64 x 64 31.2      400 x 14336 x 4096    256 x 256 42.1 (44.0), 128 x 128 42.7
//   2048 x 4096 x 4096    256 x 256 43.9 (44.0), 128 x 128 49.4    8192 x 4096 x 256     256 x 256 26.1 (24.2), 128 x 128 50.3
//   1000 x 4096 x 4097    128 x 128 35.5 (33.0), 64 x 64 61.3      4096 x 4096 x 4096    256 x 256 64.7 (65.2), 128 x 128 103.8
void plan_scaled_gemm(ScaledGemmArgs& a, int num_cus, int (&figures)[4])
{
    bool aligned = (uintptr_t) a.x % 16 == 0 && (uintptr_t) a.w % 16 == 0 && (a.M == 1 || a.x_ld % 16 == 0) && (a.N == 1 || a.w_ld % 16 == 0);
    for (int d = 0; d < 3; d++) aligned = aligned && a.x_bs[d] % 16 == 0 && a.w_bs[d] % 16 == 0;
    a.aligned = aligned;
    double best = 0.0;
    a.form = -1;
    auto groups_of = [&](int rows_m, int rows_n) {
        return (double) (((long long) a.M + rows_m - 1) / rows_m) * (double) (((long long) a.N + rows_n - 1) / rows_n) * a.batch[0] * a.batch[1] * a.batch[2];
    };
    auto consider = [&](int form, int rows_m, int rows_n, int tile_n, int waves, double us_per_round, double us_per_1024) {
        const double groups = groups_of(rows_m, rows_n);
        const double us = 3.0 + __builtin_ceil(groups / num_cus) * (us_per_round + us_per_1024 * a.K / 1024.0);
        if (a.form >= 0 && us >= best) return;
        best = us;
        a.form = form;
        a.tile_m = rows_m;
        a.tile_n = tile_n;
        a.waves = waves;
    };
    const int few = a.M <= 8 ? 8 : a.M <= 16 ? 16 : 32;
    consider(SCALED_FORM_FEW, few, 16, 1, 8, 2.2, aligned ? 0.6 : 1.07);
    if (aligned)
    {
        consider(SCALED_FORM_FEW, few, 32, 2, few == 32 ? 4 : 8, 2.5, 0.73);
        consider(SCALED_FORM_FEW, few, 64, 4, 4, 3.4, 1.0);
    }
    if (a.M > 32)
    {
        consider(SCALED_FORM_TILE, 64, 64, 64, 8, aligned ? 1.6 : 1.8, aligned ? 1.55 : 3.4);
        consider(SCALED_FORM_TILE, 128, 128, 128, 8, aligned ? 5.6 : 6.0, aligned ? 3.75 : 6.0);
        // the largest tiles: what one compute unit needs for 1024 k by itself, or what the operands' way to all of them takes
        const double groups = groups_of(256, 256), fill = groups / (__builtin_ceil(groups / num_cus) * num_cus);
        if (aligned && a.K >= 256) consider(SCALED_FORM_LARGE, 256, 256, 256, 8, 7.8, __builtin_fmax(8.3, 13.6 * fill));
    }
    figures[0] = a.form == SCALED_FORM_FEW ? 3 : 1;
    figures[1] = a.tile_m;
    figures[2] = 1;
    figures[3] = a.waves;
}

hipError_t launch_scaled_gemm(const ScaledGemmArgs& a, hipStream_t s)
{
    switch (a.form)
    {
        case SCALED_FORM_FEW: return launch_scaled_gemm_few(a, s);
        case SCALED_FORM_TILE: return launch_scaled_gemm_tile(a, s);
        default: return launch_scaled_gemm_large(a, s);
    }
}
} // namespace mme
