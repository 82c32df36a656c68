// row_quant.hip -- rows of activations (or weights) -> 8-bit codes with one scale per row.
//
//   v_i = x_i                             ROWS_PLAIN
//   v_i = gate(g_i) x_i                   ROWS_GATED      gate: silu or gelu (tanh form)
//   v_i = s_i gamma_i / rms               ROWS_NORM(_ADD) s = x (+ residual), rms = sqrt(mean(s^2) + eps)
//   scale = max|v| / qmax,   code_i = round to nearest even(v_i / scale)
//
// The norm's factor 1 / rms is the same for a whole row, so it cancels out of the codes: code_i = rne(u_i qmax / max|u|) with
// u = s gamma, and only the one scale of the row contains it.  The sum of squares and the maximum therefore come out of a single
// pass over the row, which then sits in registers: every input is read once and every output written once.  The bound is HBM.
//
// Arithmetic is fp32 (the scale, one number per row, is finished in fp64).  Rounded to fewer bits: the codes, and the
// residual sum in its own type; the norm works on the sum before that rounding.
// Rows whose values leave the comfortable middle of the fp32 range (squares or products that overflow, a maximum below 2^-64
// whose reciprocal would) are gone over once more with the values multiplied by 2^-96 or 2^96, exactly.  A row that holds an
// inf or NaN gets the scale NaN and codes 0; a row of zeros the scale 0 and codes 0.
#include "mme_numeric.hpp"
#include "scaled_kernels.hpp"

namespace mme
{
namespace
{
constexpr int VEC = 8; // elements per lane and step

// loads and stores at any element alignment (the compiler turns these into single wide accesses: the target allows unaligned ones)
struct __attribute__((packed, aligned(1))) u128_any
{
    uint32_t v[4];
};
struct __attribute__((packed, aligned(1))) u64_any
{
    uint32_t v[2];
};

template<int TYPE>
struct Raw // eight elements as they lie in memory
{
    uint32_t v[TYPE == REAL_FP32 ? 8 : 4];
};

template<int TYPE>
__device__ __forceinline__ Raw<TYPE> load8(const void* base, long long elem, int left)
{
    constexpr int ES = TYPE == REAL_FP32 ? 4 : 2;
    const char*   p = (const char*) base + elem * ES;
    Raw<TYPE>     r;
    if (left >= VEC)
    {
        const u128_any lo = *(const u128_any*) p;
#pragma unroll
        for (int i = 0; i < 4; i++) r.v[i] = lo.v[i];
        if constexpr (TYPE == REAL_FP32)
        {
            const u128_any hi = *(const u128_any*) (p + 16);
#pragma unroll
            for (int i = 0; i < 4; i++) r.v[4 + i] = hi.v[i];
        }
    }
    else
    {
#pragma unroll
        for (int i = 0; i < (int) (sizeof r.v / 4); i++) r.v[i] = 0u;
#pragma unroll
        for (int i = 0; i < VEC; i++)
            if (i < left)
            {
                if constexpr (TYPE == REAL_FP32) r.v[i] = ((const uint32_t*) p)[i];
                else
                    r.v[i / 2] |= (uint32_t) ((const uint16_t*) p)[i] << (16 * (i & 1));
            }
    }
    return r;
}

template<int TYPE>
__device__ __forceinline__ float value(const Raw<TYPE>& r, int i)
{
    if constexpr (TYPE == REAL_FP32) return __uint_as_float(r.v[i]);
    else if constexpr (TYPE == REAL_BF16)
        return __uint_as_float((i & 1) ? (r.v[i / 2] & 0xFFFF0000u) : (r.v[i / 2] << 16));
    else
    {
        _Float16 h[2];
        __builtin_memcpy(h, &r.v[i / 2], 4);
        return (float) h[i & 1];
    }
}

// eight fp32 -> eight elements of TYPE, round to nearest even
template<int TYPE>
__device__ __forceinline__ Raw<TYPE> rounded(const float (&s)[VEC])
{
    Raw<TYPE> r;
    if constexpr (TYPE == REAL_FP32)
    {
#pragma unroll
        for (int i = 0; i < VEC; i++) r.v[i] = __float_as_uint(s[i]);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < VEC / 2; i++)
        {
            typedef float f2 __attribute__((ext_vector_type(2)));
            if constexpr (TYPE == REAL_BF16)
            {
                typedef __bf16 b2 __attribute__((ext_vector_type(2)));
                const b2 h = __builtin_convertvector(f2 {s[2 * i], s[2 * i + 1]}, b2);
                __builtin_memcpy(&r.v[i], &h, 4);
            }
            else
            {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 h = __builtin_convertvector(f2 {s[2 * i], s[2 * i + 1]}, h2);
                __builtin_memcpy(&r.v[i], &h, 4);
            }
        }
    }
    return r;
}

template<int TYPE>
__device__ __forceinline__ void store8(void* base, long long elem, int left, const Raw<TYPE>& r)
{
    constexpr int ES = TYPE == REAL_FP32 ? 4 : 2;
    char*         p = (char*) base + elem * ES;
    if (left >= VEC)
    {
#pragma unroll
        for (int q = 0; q < (int) sizeof r.v / 16; q++) *(u128_any*) (p + 16 * q) = u128_any {{r.v[4 * q], r.v[4 * q + 1], r.v[4 * q + 2], r.v[4 * q + 3]}};
    }
    else
    {
#pragma unroll
        for (int i = 0; i < VEC; i++)
            if (i < left)
            {
                if constexpr (TYPE == REAL_FP32) ((uint32_t*) p)[i] = r.v[i];
                else
                    ((uint16_t*) p)[i] = (uint16_t) (r.v[i / 2] >> (16 * (i & 1)));
            }
    }
}

// e^x to about one unit in the last place: the rounding error of x log2(e), which the hardware's 2^t would magnify by |x|, is
// computed and put back to first order (x is clamped to where the result is neither 0 nor inf)
__device__ __forceinline__ float exp_accurate(float x)
{
    constexpr float L2E = 0x1.715476p+0f, L2E_LO = 0x1.4ae0bep-26f, LN2 = 0x1.62e43p-1f;
    x = __builtin_fminf(__builtin_fmaxf(x, -87.0f), 88.0f);
    const float t = x * L2E;
    const float r = __builtin_fmaf(x, L2E_LO, __builtin_fmaf(x, L2E, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e * LN2, r, e);
}
__device__ __forceinline__ float gate_of(float g, int gelu)
{
    // (g / (1 + e^-g) and g / (1 + e^-2c): the tanh form of gelu is g sigmoid(2 c); an inf or NaN gate gives what the
    // formula gives in the limit, NaN for NaN, inf for +inf and NaN (0 x inf) for -inf)
    float a = -g;
    if (gelu) a *= 2.0f * 0.7978845608028654f * __builtin_fmaf(0.044715f * g, g, 1.0f);
    return g / (1.0f + (a > 88.0f ? __uint_as_float(0x7F800000u) : exp_accurate(a)));
}

// sum and maximum (of bit patterns of magnitudes, whose order is the values' with NaN on top) over 64 lanes: within rows of 16
// by data-parallel moves, across them by the two lane swaps
template<int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x)
{
    return (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ void wave_reduce(float& sum, uint32_t& top)
{
    auto step = [&](auto ctrl) __attribute__((always_inline))
    {
        constexpr int C = decltype(ctrl)::value;
        sum += __uint_as_float(dpp<C>(__float_as_uint(sum)));
        top = max(top, dpp<C>(top));
    };
    step(std::integral_constant<int, 0xB1>());  // quad_perm 1, 0, 3, 2
    step(std::integral_constant<int, 0x4E>());  // quad_perm 2, 3, 0, 1
    step(std::integral_constant<int, 0x141>()); // row_half_mirror
    step(std::integral_constant<int, 0x140>()); // row_mirror
    auto s16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(s16[0]) + __uint_as_float(s16[1]);
    auto t16 = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    top = max(t16[0], t16[1]);
    auto s32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(s32[0]) + __uint_as_float(s32[1]);
    auto t32 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = max(t32[0], t32[1]);
}

constexpr uint32_t INF_BITS = 0x7F800000u, LOW_BITS = 0x1F800000u /* 2^-64 */;

// T lanes per row (64: four rows per workgroup, one per wavefront; else a workgroup per row), NV steps of T x 8 elements held in
// registers; NV 0: rows of any width, gone over again in memory for every pass.
template<int KIND, int TYPE, int T, int NV>
__global__ __launch_bounds__(T == 64 ? 256 : T) void row_quant_kernel(const RowQuantArgs a)
{
    constexpr bool NORM = KIND == ROWS_NORM || KIND == ROWS_NORM_ADD;
    constexpr bool TWO = KIND == ROWS_GATED || KIND == ROWS_NORM_ADD;
    constexpr int  WAVES = T / 64;
    __shared__ float    part_sum[2][WAVES > 1 ? WAVES : 1];
    __shared__ uint32_t part_top[2][WAVES > 1 ? WAVES : 1];
    const int      lane = T == 64 ? threadIdx.x & 63 : threadIdx.x;
    const uint32_t row = T == 64 ? blockIdx.x * 4u + (uint32_t) __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
    if (T == 64 && row >= a.rows) return; // (no barrier is met by these instances)
    uint32_t i0 = row, i1 = 0, i2 = 0, i3 = 0;
    if (a.n[0] != a.rows)
    {
        uint32_t r = row / a.n[0];
        i0 = row - r * a.n[0];
        i1 = r % a.n[1];
        r /= a.n[1];
        i2 = r % a.n[2];
        i3 = r / a.n[2];
    }
    auto at = [&](const long long (&st)[4]) __attribute__((always_inline)) { return i0 * st[0] + i1 * st[1] + i2 * st[2] + i3 * st[3]; };
    const long long x0 = at(a.x_stride), y0 = TWO ? at(a.second_stride) : 0;
    const int       width = (int) a.width;

    // s: what the norm squares (or x), u: what the codes stand for (elements behind the row's end are zeros in both)
    auto load_s = [&](int e, float (&s)[VEC]) __attribute__((always_inline))
    {
        const int  left = width - e;
        const auto x = load8<TYPE>(a.x, x0 + e, left);
        if constexpr (TWO)
        {
            const auto y = load8<TYPE>(a.second, y0 + e, left);
#pragma unroll
            for (int i = 0; i < VEC; i++) s[i] = KIND == ROWS_NORM_ADD ? value<TYPE>(x, i) + value<TYPE>(y, i) : gate_of(value<TYPE>(y, i), a.gelu) * value<TYPE>(x, i);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < VEC; i++) s[i] = value<TYPE>(x, i);
        }
    };
    auto load_gamma = [&](int e, float (&g)[VEC]) __attribute__((always_inline))
    {
        if (a.gamma_type == REAL_FP32)
        {
            const auto q = load8<REAL_FP32>(a.gamma, e, width - e);
#pragma unroll
            for (int i = 0; i < VEC; i++) g[i] = value<REAL_FP32>(q, i);
        }
        else
        {
            const auto q = load8<TYPE>(a.gamma, e, width - e);
#pragma unroll
            for (int i = 0; i < VEC; i++) g[i] = value<TYPE>(q, i);
        }
    };

    float s[NV ? NV : 1][VEC], u[NV ? NV : 1][VEC];
    // fills u of step n; fs, fu: powers of two that the squares' operands and u are multiplied by (1 but for rows gone over again)
    auto fill = [&](int n, int e, float fs, float fu, float& sum, uint32_t& top) __attribute__((always_inline))
    {
        if constexpr (NORM)
        {
            float g[VEC];
            if (a.gamma) load_gamma(e, g);
            else
            {
#pragma unroll
                for (int i = 0; i < VEC; i++) g[i] = 1.0f;
            }
            if (fu == 1.0f)
            {
#pragma unroll
                for (int i = 0; i < VEC; i++) u[n][i] = s[n][i] * g[i];
            }
            else
            {
                // the power goes to the factor that it takes towards one: nothing overflows or vanishes on the way
#pragma unroll
                for (int i = 0; i < VEC; i++)
                {
                    const bool small = __builtin_fabsf(s[n][i]) < 1.0f, to_s = small == (fu > 1.0f);
                    u[n][i] = (to_s ? s[n][i] * fu : s[n][i]) * (to_s ? g[i] : g[i] * fu);
                }
            }
#pragma unroll
            for (int i = 0; i < VEC; i++) sum = __builtin_fmaf(s[n][i] * fs, s[n][i] * fs, sum);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < VEC; i++) u[n][i] = s[n][i] * fu;
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) top = max(top, __float_as_uint(u[n][i]) & 0x7FFFFFFFu);
    };
    int  phase = 0;
    auto reduce = [&](float& sum, uint32_t& top) __attribute__((always_inline))
    {
        wave_reduce(sum, top);
        if constexpr (WAVES > 1)
        {
            // (two sets of cells used in turn: a second reduction does not overwrite what a slow wavefront still reads)
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) part_sum[phase][wave] = sum, part_top[phase][wave] = top;
            __syncthreads();
            const int w = threadIdx.x & 63;
            sum = w < WAVES ? part_sum[phase][w] : 0.0f;
            top = w < WAVES ? part_top[phase][w] : 0u;
            wave_reduce(sum, top);
            phase ^= 1;
        }
    };
    auto pass = [&](float fs, float fu, float& sum, uint32_t& top) __attribute__((always_inline))
    {
        sum = 0.0f;
        top = 0u;
        if constexpr (NV > 0)
        {
#pragma unroll
            for (int n = 0; n < NV; n++) fill(n, (n * T + lane) * VEC, fs, fu, sum, top);
        }
        else
        {
#pragma unroll 1
            for (int e = lane * VEC; e < width; e += T * VEC)
            {
                load_s(e, s[0]);
                fill(0, e, fs, fu, sum, top);
            }
        }
        reduce(sum, top);
    };

    if constexpr (NV > 0)
    {
#pragma unroll
        for (int n = 0; n < NV; n++)
        {
            const int e = (n * T + lane) * VEC;
            if (e < width) load_s(e, s[n]);
            else
            {
#pragma unroll
                for (int i = 0; i < VEC; i++) s[n][i] = 0.0f;
            }
        }
    }
    float    fs = 1.0f, fu = 1.0f, sum;
    uint32_t top;
    pass(fs, fu, sum, top);
    if (top >= INF_BITS || top < LOW_BITS || (NORM && !(sum < 0x1p+126f && sum > 0x1p-100f)))
    {
        // (the same in every lane of the row)
        fu = top >= INF_BITS ? 0x1p-96f : (top < LOW_BITS ? 0x1p+96f : 1.0f);
        if (NORM) fs = !(sum < 0x1p+126f) ? 0x1p-96f : (sum > 0x1p-100f ? 1.0f : 0x1p+96f);
        pass(fs, fu, sum, top);
    }
    // an inf or NaN among s shows in the squares' sum as well as in u unless gamma is zero there
    const bool  bad = top >= INF_BITS || (NORM && !(sum < __uint_as_float(INF_BITS)));
    const float most = __uint_as_float(top);
    // qmax / max|u| in two parts, f the quotient rounded to fp32, f_lo what that leaves out
    const float f = bad || top == 0u ? 0.0f : a.qmax / most;
    const float f_lo = bad || top == 0u ? 0.0f : __builtin_fmaf(-f, most, a.qmax) / most;

    const long long c0 = at(a.codes_stride);
    auto            put = [&](int n, int e) __attribute__((always_inline))
    {
        const int left = width - e;
        if constexpr (KIND == ROWS_NORM_ADD)
            if (a.sum) store8<TYPE>(a.sum, at(a.sum_stride) + e, left, rounded<TYPE>(s[n]));
        uint32_t c[2] = {0u, 0u};
        if (!bad)
        {
            float q[VEC];
            if (a.code != CODE_INT8)
#pragma unroll
                for (int i = 0; i < VEC; i++) q[i] = __builtin_amdgcn_fmed3f(__builtin_fmaf(u[n][i], f, u[n][i] * f_lo), -a.qmax, a.qmax);
            if (a.code == CODE_INT8)
            {
                // added to 1.5 x 2^23 the product is rounded once, to a whole number (127 for the largest: f is off by less than
                // 2^-24), whose two's complement stands in the low byte
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    uint32_t b[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) b[i] = __float_as_uint(__builtin_fmaf(u[n][4 * h + i], f, 12582912.0f));
                    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000C0Cu);
                    c[h] = lo | hi;
                }
            }
            else if (a.code == CODE_E4M3)
            {
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    int p = 0;
                    p = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], p, false);
                    c[h] = (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], p, true);
                }
            }
            else
            {
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    int p = 0;
                    p = __builtin_amdgcn_cvt_pk_bf8_f32(q[4 * h], q[4 * h + 1], p, false);
                    c[h] = (uint32_t) __builtin_amdgcn_cvt_pk_bf8_f32(q[4 * h + 2], q[4 * h + 3], p, true);
                }
            }
        }
        uint8_t* o = a.codes + c0 + e;
        if (left >= VEC) *(u64_any*) o = u64_any {{c[0], c[1]}};
        else
        {
#pragma unroll
            for (int i = 0; i < VEC; i++)
                if (i < left) o[i] = (uint8_t) (c[i / 4] >> (8 * (i & 3)));
        }
    };
    if constexpr (NV > 0)
    {
#pragma unroll
        for (int n = 0; n < NV; n++)
        {
            const int e = (n * T + lane) * VEC;
            if (e < width) put(n, e);
        }
    }
    else
    {
#pragma unroll 1
        for (int e = lane * VEC; e < width; e += T * VEC)
        {
            float    dummy_sum = 0.0f;
            uint32_t dummy_top = 0u;
            load_s(e, s[0]);
            fill(0, e, fs, fu, dummy_sum, dummy_top);
            put(0, e);
        }
    }
    if (lane == 0)
    {
        double sc = (double) most / (double) a.qmax * a.fold / (double) fu;
        if (NORM)
        {
            const double ms = (double) sum / ((double) fs * (double) fs) / (double) width;
            sc = top == 0u ? 0.0 : sc / sqrt(ms + a.eps);
        }
        a.scales[row] = bad ? __uint_as_float(0x7FC00000u) : (float) sc;
    }
}

template<int KIND, int TYPE, int T, int NV>
hipError_t start(const RowQuantArgs& a, hipStream_t s)
{
    const uint32_t groups = T == 64 ? (a.rows + 3) / 4 : a.rows;
    hipLaunchKernelGGL((row_quant_kernel<KIND, TYPE, T, NV>), dim3(groups), dim3(T == 64 ? 256 : T), 0, s, a);
    return hipGetLastError();
}

template<int KIND, int TYPE>
hipError_t start_sized(const RowQuantArgs& a, int num_cus, hipStream_t s)
{
    (void) num_cus;
    if (a.width <= 512) return start<KIND, TYPE, 64, 1>(a, s);
    if (a.width <= 1024) return start<KIND, TYPE, 64, 2>(a, s);
    if (a.width <= 4096) return start<KIND, TYPE, 256, 2>(a, s);
    if (a.width <= 8192) return start<KIND, TYPE, 512, 2>(a, s);
    if (a.width <= 16384) return start<KIND, TYPE, 1024, 2>(a, s);
    return start<KIND, TYPE, 1024, 0>(a, s);
}

template<int KIND>
hipError_t start_typed(const RowQuantArgs& a, int num_cus, hipStream_t s)
{
    switch (a.type)
    {
        case REAL_BF16: return start_sized<KIND, REAL_BF16>(a, num_cus, s);
        case REAL_FP16: return start_sized<KIND, REAL_FP16>(a, num_cus, s);
        default: return start_sized<KIND, REAL_FP32>(a, num_cus, s);
    }
}
} // namespace

hipError_t launch_row_quant(const RowQuantArgs& a, int num_cus, hipStream_t s)
{
    if (a.rows == 0 || a.width == 0) return hipSuccess;
    switch (a.kind)
    {
        case ROWS_PLAIN: return start_typed<ROWS_PLAIN>(a, num_cus, s);
        case ROWS_GATED: return start_typed<ROWS_GATED>(a, num_cus, s);
        case ROWS_NORM: return start_typed<ROWS_NORM>(a, num_cus, s);
        default: return start_typed<ROWS_NORM_ADD>(a, num_cus, s);
    }
}
} // namespace mme
