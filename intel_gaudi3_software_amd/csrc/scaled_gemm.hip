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

// What a form is expected to take: a fixed part, and for every round of workgroups over the compute units the bytes that one of them
// brings into LDS, at the rate that a compute unit of that form was seen to reach.  Measured against the estimate, in us (M x N x K,
// int8 -> bf16): few rows, 32 x 32 outputs, 64 x 4096 x 4096: 7.7 (6.6); 32 x 16, 64 x 1024 x 16384: 11.4 (12.7); 64 x 64 tiles, 128 x 14336 x 4096:
// 17.2 (16.6), 250 x 4096 x 14336: 27.0 (26.4), 512 x 4096 x 4096: 17.5 (16.6); 128 x 128, 1024 x 4096 x 4096: 25.6 (25.5), 400 x 14336 x 4096: 44.7
// (43.0); 256 x 256, 2048 x 4096 x 4096: 43.9 (41.0).  The estimates' order is the measured one in all of these; the runner-up took 5 %
// (512 x 4096 x 4096 in 128 x 128 tiles: 21.6) to 112 % (64 x 1024 x 16384 in 64 x 64 tiles: 24.4) more.
void plan_scaled_gemm(ScaledGemmArgs& a, int num_cus, int (&figures)[4])
{
    bool aligned = (uintptr_t) a.x % 16 == 0 && (uintptr_t) a.w % 16 == 0 && (a.M == 1 || a.x_ld % 16 == 0) && (a.N == 1 || a.w_ld % 16 == 0);
    for (int d = 0; d < 3; d++) aligned = aligned && a.x_bs[d] % 16 == 0 && a.w_bs[d] % 16 == 0;
    a.aligned = aligned;
    double best = 0.0;
    a.form = -1;
    auto consider = [&](int form, int rows_m, int rows_n, int tile_n, int waves, double fixed_us, double gb_per_s) {
        const double groups = (double) (((long long) a.M + rows_m - 1) / rows_m) * (double) (((long long) a.N + rows_n - 1) / rows_n) * a.batch[0] * a.batch[1] * a.batch[2];
        const double rounds = __builtin_ceil(groups / num_cus);
        const double us = fixed_us + rounds * (rows_m + rows_n) * (double) a.K / (gb_per_s * 1e3);
        if (a.form >= 0 && us >= best) return;
        best = us;
        a.form = form;
        a.tile_m = rows_m;
        a.tile_n = tile_n;
        a.waves = waves;
    };
    const int few = a.M <= 8 ? 8 : a.M <= 16 ? 16 : 32;
    consider(SCALED_FORM_FEW, few, 16, 1, 8, 3.5, 85.0);
    if (aligned)
    {
        consider(SCALED_FORM_FEW, few, 32, 2, few == 32 ? 4 : 8, 3.5, 85.0);
        consider(SCALED_FORM_FEW, few, 64, 4, 4, 3.5, 85.0);
    }
    if (a.M > 32)
    {
        consider(SCALED_FORM_TILE, 64, 64, 64, 8, 3.5, 80.0);
        consider(SCALED_FORM_TILE, 128, 128, 128, 8, 8.0, 60.0);
        if (aligned && a.K >= 256) consider(SCALED_FORM_LARGE, 256, 256, 256, 8, 8.0, 64.0);
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
