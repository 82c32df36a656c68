// scaled_kernels.hpp -- internal interface between the C ABI layer and the kernels of the 8-bit linear layer: the row quantisers
// (row_quant.hip) and the product of 8-bit operands with a scale per row and column (scaled_gemm*.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mme
{
// ---- row quantisers ------------------------------------------------------------------------------------------------
enum : int
{
    ROWS_PLAIN = 0,     // v = x
    ROWS_GATED = 1,     // v = gate(second) * x
    ROWS_NORM = 2,      // v = x * gamma, scaled by 1 / rms(x)
    ROWS_NORM_ADD = 3   // the same of s = x + second, which is also written to sum
};
enum : int
{
    CODE_INT8 = 0,
    CODE_E4M3 = 1,
    CODE_E5M2 = 2
};
enum : int
{
    REAL_BF16 = 0,
    REAL_FP16 = 1,
    REAL_FP32 = 2
};

struct RowQuantArgs
{
    const void* x;
    const void* second;   // residual or gate
    const void* gamma;    // NULL: ones
    void*       sum;      // NULL: not written
    uint8_t*    codes;
    float*      scales;   // dense, one per row
    long long   x_stride[4], second_stride[4], sum_stride[4], codes_stride[4]; // elements, dims 1 .. 4
    uint32_t    n[3];     // sizes of dims 1 .. 3 (a row's index is decoded by them); n[0] == rows: one stride per tensor
    uint32_t    rows, width;
    int         kind;     // ROWS_*
    int         type;     // REAL_*: x, second, sum
    int         gamma_type;
    int         gelu;     // ROWS_GATED: 0 silu, 1 gelu (tanh form)
    int         code;     // CODE_*
    float       qmax;     // value of the largest code, exponent bias of the hardware's format
    double      fold;     // scales are multiplied by this power of two (another exponent bias)
    double      eps;
    // filled in by plan_row_quant
    uint32_t    lanes;        // lanes that share a row
    int         lanes_shared; // 16, 32, 64: several rows share a workgroup of 256; 0: a workgroup per row
    int         steps;        // eights of elements that a lane holds, 0: the row is gone over in memory
};
void       plan_row_quant(RowQuantArgs& a, int num_cus);
hipError_t launch_row_quant(const RowQuantArgs& a, hipStream_t s);

// ---- scaled product --------------------------------------------------------------------------------------------------
enum : int
{
    SCALED_OUT_BF16 = 0,
    SCALED_OUT_FP16 = 1,
    SCALED_OUT_FP32 = 2,
    SCALED_OUT_INT32 = 3 // the sums themselves
};

struct ScaledGemmArgs
{
    const uint8_t* x;       // M rows of K codes
    const uint8_t* w;       // N rows of K codes
    void*          out;     // M rows of N values
    const float*   sx;      // per row of x, NULL: ones
    const float*   sw;      // per row of w, NULL: ones
    const float*   bias;    // per row of w, NULL: zeros
    int            M, N, K;
    int            batch[3];
    long long      x_ld, w_ld, out_ld;                   // elements between rows
    long long      x_bs[3], w_bs[3], out_bs[3];          // elements between batch elements, 0 where an operand is broadcast
    long long      sx_bs[3], sw_bs[3];                   // the same for the scales (and the bias, which goes with w)
    int            int8;    // 1: int8 codes, 0: fp8
    int            fmt;     // fp8: bit 0 = x is e5m2, bit 1 = w is e5m2
    int            out_type;
    float          alpha;   // fp8: power of two of the exponent biases
    int            aligned; // every row of x and w starts at a multiple of 16 bytes
    int            form;    // SCALED_FORM_*, filled in by plan_scaled_gemm
    int            tile_m, tile_n; // shape of a workgroup's outputs, in the form's own units
    int            waves;   // wavefronts per workgroup
};

enum : int
{
    SCALED_FORM_FEW = 0,  // few rows of x, or few outputs (scaled_gemm_few.hip): tile_m rows of x x 16 tile_n rows of w
    SCALED_FORM_TILE = 1, // 64 x 64 or 128 x 128 outputs (scaled_gemm_tile.hip)
    SCALED_FORM_LARGE = 2 // 256 x 256 (scaled_gemm_large.hip)
};

// picks the kernel form for these operands; figures: what mme_hip_last_contraction_form reports
void plan_scaled_gemm(ScaledGemmArgs& a, int num_cus, int (&figures)[4]);
// lets a kernel have `bytes` of dynamic LDS on the current device (asked for once per kernel and device)
hipError_t allow_lds(const void* kernel, int bytes);
hipError_t launch_scaled_gemm_few(const ScaledGemmArgs& a, hipStream_t s);
hipError_t launch_scaled_gemm_tile(const ScaledGemmArgs& a, hipStream_t s);
hipError_t launch_scaled_gemm_large(const ScaledGemmArgs& a, hipStream_t s);
hipError_t launch_scaled_gemm(const ScaledGemmArgs& a, hipStream_t s);
} // namespace mme
