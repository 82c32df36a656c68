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
// Rows whose values leave the comfortable middle of the fp32 range (squares or products with gamma that overflow, a maximum below 2^-64
// whose reciprocal would) are gone over once more, with the squared values multiplied by 2^-96 or 2^96 and the products by 2^-132 or 2^144,
// exactly.  A row that holds an inf or NaN (a gated product that overflows is one) gets the scale NaN and codes 0; a row of zeros the scale
// 0 and codes 0.
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

// e^x for |x| <= 110 (0 where that is below 2^-126), to about one unit in the last place.  e^x is 2^t with t = x log2(e); the rounding of
// t, which the exponential would magnify by |x|, is computed and put back to first order.
__device__ __forceinline__ float exponential(float x)
{
    constexpr float L2E = 0x1.715476p+0f, L2E_LO = 0x1.4ae0bep-26f, LN2 = 0x1.62e43p-1f;
    const float     t = x * L2E;
    const float     r = __builtin_fmaf(x, L2E_LO, __builtin_fmaf(x, L2E, -t));
    const float     e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e * LN2, r, e);
}
// v_i = g_i / (1 + e^-g_i), or its like with 2 sqrt(2 / pi) (g + 0.044715 g^3) in the exponent: the tanh form of gelu is that.  NaN gives
// NaN, +inf gives inf and -inf NaN (inf x 0).  The quotient is g times the hardware's reciprocal, which is off by up to one unit in the last
// place; a step of Newton's behind it took the gated rows of 8192 x 14336 from 108.5 to 112.5 us and did not change how many codes
// differ from 64-bit arithmetic (92 of 117 million, 106 with it).
// From e^87 on the sum and its reciprocal would leave the range: there the rest of the exponential is a factor of its own, and the result
// vanishes where fp32 ends.  That is rare: one branch for eight elements.
__device__ __forceinline__ void gate_of(const float (&g)[VEC], int gelu, float (&v)[VEC])
{
    float x[VEC], most = 0.0f;
#pragma unroll
    for (int i = 0; i < VEC; i++)
    {
        x[i] = -g[i];
        if (gelu) x[i] *= 2.0f * 0.7978845608028654f * __builtin_fmaf(0.044715f * g[i], g[i], 1.0f);
        most = __builtin_fmaxf(most, x[i]);
        v[i] = g[i] * __builtin_amdgcn_rcpf(1.0f + exponential(__builtin_amdgcn_fmed3f(x[i], -87.0f, 87.0f)));
    }
    if (most > 87.0f)
    {
#pragma unroll
        for (int i = 0; i < VEC; i++)
            if (x[i] > 87.0f) v[i] *= exponential(__builtin_fmaxf(87.0f - x[i], -110.0f));
    }
}

// sum and maximum (of bit patterns of magnitudes, whose order is the values' with NaN on top) over groups of LANES = 16, 32 or 64 lanes:
// within rows of 16 by data-parallel moves, across them by the two lane swaps
template<int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x)
{
    return (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, CTRL, 0xF, 0xF, true);
}
template<int LANES>
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
    if constexpr (LANES > 16)
    {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
        sum = __uint_as_float(s[0]) + __uint_as_float(s[1]);
        const auto t = __builtin_amdgcn_permlane16_swap(top, top, false, false);
        top = max(t[0], t[1]);
    }
    if constexpr (LANES > 32)
    {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
        sum = __uint_as_float(s[0]) + __uint_as_float(s[1]);
        const auto t = __builtin_amdgcn_permlane32_swap(top, top, false, false);
        top = max(t[0], t[1]);
    }
}

constexpr uint32_t INF_BITS = 0x7F800000u, LOW_BITS = 0x1F800000u /* 2^-64 */;

// LANES per row: 16, 32 or 64, several rows per workgroup of 256; or 0, a workgroup per row.  Each lane holds NV times 8 elements of its
// row in registers, at every (lanes per row x 8)-th place; NV 0: rows of any width, gone over again in memory for every pass (places are
// unsigned there: the step behind the last one of a row of nearly 2^31 elements leaves the signed range).
template<int KIND, int TYPE, int LANES, int NV>
__global__ __launch_bounds__(LANES ? 256 : NV == 1 || NV == 4 ? 512 : 1024) void row_quant_kernel(const RowQuantArgs a)
{
    constexpr bool NORM = KIND == ROWS_NORM || KIND == ROWS_NORM_ADD;
    constexpr bool TWO = KIND == ROWS_GATED || KIND == ROWS_NORM_ADD;
    constexpr int  N = NV ? NV : 1;
    __shared__ float    part_sum[2][16];
    __shared__ uint32_t part_top[2][16];
    const int      lane = LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x, lanes = LANES ? LANES : (int) blockDim.x;
    const uint32_t row = LANES ? blockIdx.x * (256u / (LANES ? LANES : 1)) + threadIdx.x / (LANES ? LANES : 1) : blockIdx.x;
    const bool     live = row < a.rows; // (every lane takes part in the reductions)
    const int      width = live ? (int) a.width : 0;
    auto           at = [&](const long long(&st)[4], uint32_t row) __attribute__((always_inline)) -> long long
    {
        if (a.n[0] == a.rows) return row * st[0];
        uint32_t       r = row / a.n[0];
        const uint32_t i0 = row - r * a.n[0], i1 = r % a.n[1];
        r /= a.n[1];
        return i0 * st[0] + i1 * st[1] + (r % a.n[2]) * st[2] + (r / a.n[2]) * st[3];
    };
    auto load_gamma = [&](uint32_t e, float(&g)[VEC]) __attribute__((always_inline))
    {
        if (!a.gamma)
        {
#pragma unroll
            for (int i = 0; i < VEC; i++) g[i] = 1.0f;
        }
        else if (a.gamma_type == REAL_FP32)
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
    // s: what the norm squares, or what the codes stand for (elements behind the row's end are zeros)
    auto make_s = [&](const Raw<TYPE>& x, const Raw<TYPE>& y, float(&s)[VEC]) __attribute__((always_inline))
    {
        if constexpr (KIND == ROWS_GATED)
        {
            float g[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) g[i] = value<TYPE>(y, i);
            gate_of(g, a.gelu, s);
#pragma unroll
            for (int i = 0; i < VEC; i++) s[i] *= value<TYPE>(x, i);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < VEC; i++) s[i] = KIND == ROWS_NORM_ADD ? value<TYPE>(x, i) + value<TYPE>(y, i) : value<TYPE>(x, i);
        }
    };
    // u: what the codes stand for up to a factor of the row; hu: a power of two that it is multiplied by twice (1 but for rows gone over again)
    auto make_u = [&](const float(&s)[VEC], const float(&g)[VEC], float hu, float(&u)[VEC]) __attribute__((always_inline))
    {
        if (hu == 1.0f)
        {
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] = NORM ? s[i] * g[i] : s[i];
        }
        else if (NORM)
        {
            // the powers go to the smaller factor where they enlarge, to the larger one where they diminish: with 2^144 (all products
            // below 2^-64, so the smaller factor below 2^-32) and 2^-132 (the largest product at least 2^128) nothing overflows on the
            // way, and what vanishes is nothing beside the largest
#pragma unroll
            for (int i = 0; i < VEC; i++)
            {
                const bool to_s = (__builtin_fabsf(s[i]) < __builtin_fabsf(g[i])) == (hu > 1.0f);
                u[i] = (to_s ? s[i] : g[i]) * hu * hu * (to_s ? g[i] : s[i]);
            }
        }
        else
        {
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] = s[i] * hu * hu;
        }
    };
    auto gather = [&](const float(&s)[VEC], const float(&g)[VEC], float fs, float hu, float& sum, uint32_t& top) __attribute__((always_inline))
    {
        float u[VEC];
        make_u(s, g, hu, u);
        if constexpr (NORM)
        {
#pragma unroll
            for (int i = 0; i < VEC; i++) sum = __builtin_fmaf(s[i] * fs, s[i] * fs, sum);
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) top = max(top, __float_as_uint(u[i]) & 0x7FFFFFFFu);
    };
    int  phase = 0;
    auto reduce = [&](float& sum, uint32_t& top) __attribute__((always_inline))
    {
        wave_reduce<LANES ? LANES : 64>(sum, top);
        if constexpr (LANES == 0)
        {
            // (two sets of cells used in turn: the second reduction does not overwrite what a slow wavefront still reads of the first)
            const int wave = threadIdx.x >> 6, w = threadIdx.x & 15, waves = (int) blockDim.x >> 6;
            if ((threadIdx.x & 63) == 0) part_sum[phase][wave] = sum, part_top[phase][wave] = top;
            __syncthreads();
            sum = w < waves ? part_sum[phase][w] : 0.0f;
            top = w < waves ? part_top[phase][w] : 0u;
            wave_reduce<16>(sum, top);
            phase ^= 1;
        }
    };

    float           gamma[N][VEC], s[N][VEC];
    const long long x0 = at(a.x_stride, row), y0 = TWO ? at(a.second_stride, row) : 0, c0 = at(a.codes_stride, row), r0 = KIND == ROWS_NORM_ADD ? at(a.sum_stride, row) : 0;
    if constexpr (NV > 0)
    {
        Raw<TYPE> x[N], y[N];
#pragma unroll
        for (int n = 0; n < NV; n++)
        {
            const int e = (n * lanes + lane) * VEC;
            x[n] = load8<TYPE>(a.x, x0 + e, width - e);
            if constexpr (TWO) y[n] = load8<TYPE>(a.second, y0 + e, width - e);
        }
        if constexpr (NORM)
        {
#pragma unroll
            for (int n = 0; n < NV; n++) load_gamma((n * lanes + lane) * VEC, gamma[n]);
        }
#pragma unroll
        for (int n = 0; n < NV; n++) make_s(x[n], y[n], s[n]);
    }
    auto pass = [&](float fs, float hu, float& sum, uint32_t& top) __attribute__((always_inline))
    {
        sum = 0.0f;
        top = 0u;
        if constexpr (NV > 0)
        {
#pragma unroll
            for (int n = 0; n < NV; n++) gather(s[n], gamma[n], fs, hu, sum, top);
        }
        else
        {
#pragma unroll 1
            for (uint32_t e = lane * VEC; e < (uint32_t) width; e += lanes * VEC)
            {
                const auto xe = load8<TYPE>(a.x, x0 + e, width - e);
                Raw<TYPE>  ye = xe;
                if constexpr (TWO) ye = load8<TYPE>(a.second, y0 + e, width - e);
                make_s(xe, ye, s[0]);
                if constexpr (NORM) load_gamma(e, gamma[0]);
                gather(s[0], gamma[0], fs, hu, sum, top);
            }
        }
        reduce(sum, top);
    };
    float    fs = 1.0f, hu = 1.0f, sum;
    uint32_t top;
    pass(1.0f, 1.0f, sum, top);
    const bool odd = top >= INF_BITS || top < LOW_BITS || (NORM && !(sum < 0x1p+126f && sum > 0x1p-100f)); // (the same in every lane of the row)
    if (LANES ? __any(odd && live) : odd)
    {
        // (a wavefront with several rows goes over all of them, those that need it not with factors of one)
        hu = top >= INF_BITS ? 0x1p-66f : (top < LOW_BITS ? 0x1p+72f : 1.0f);
        if (NORM) fs = !(sum < 0x1p+126f) ? 0x1p-96f : (sum > 0x1p-100f ? 1.0f : 0x1p+96f);
        pass(fs, hu, sum, top);
    }
    const bool  bad = top >= INF_BITS || (NORM && !(sum < __uint_as_float(INF_BITS)));
    const float most = __uint_as_float(top);
    // qmax / max|u| in two parts, f the quotient rounded to fp32, f_lo what that leaves out
    const float f = bad || top == 0u ? 0.0f : a.qmax / most;
    const float f_lo = bad || top == 0u ? 0.0f : __builtin_fmaf(-f, most, a.qmax) / most;

    auto put = [&](int n, uint32_t e) __attribute__((always_inline))
    {
        const int left = width - (int) e;
        if constexpr (KIND == ROWS_NORM_ADD)
            if (a.sum) store8<TYPE>(a.sum, r0 + e, left, rounded<TYPE>(s[n]));
        uint32_t c[2] = {0u, 0u};
        if (!bad)
        {
            float u[VEC];
            make_u(s[n], gamma[n], hu, u);
            if (a.code == CODE_INT8)
            {
                // added to 1.5 x 2^23 the product is rounded once, to a whole number (127 for the largest: f is off by less than
                // 2^-24), whose two's complement stands in the low byte
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    uint32_t b[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) b[i] = __float_as_uint(__builtin_fmaf(u[4 * h + i], f, 12582912.0f));
                    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000C0Cu);
                    c[h] = lo | hi;
                }
            }
            else
            {
#pragma unroll
                for (int i = 0; i < VEC; i++) u[i] = __builtin_amdgcn_fmed3f(__builtin_fmaf(u[i], f, u[i] * f_lo), -a.qmax, a.qmax);
                if (a.code == CODE_E4M3)
                {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                    {
                        int p = 0;
                        p = __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * h], u[4 * h + 1], p, false);
                        c[h] = (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * h + 2], u[4 * h + 3], p, true);
                    }
                }
                else
                {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                    {
                        int p = 0;
                        p = __builtin_amdgcn_cvt_pk_bf8_f32(u[4 * h], u[4 * h + 1], p, false);
                        c[h] = (uint32_t) __builtin_amdgcn_cvt_pk_bf8_f32(u[4 * h + 2], u[4 * h + 3], p, true);
                    }
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
            const int e = (n * lanes + lane) * VEC;
            if (e < width) put(n, e);
        }
    }
    else
    {
#pragma unroll 1
        for (uint32_t e = lane * VEC; e < (uint32_t) width; e += lanes * VEC)
        {
            const auto xe = load8<TYPE>(a.x, x0 + e, width - e);
            Raw<TYPE>  ye = xe;
            if constexpr (TWO) ye = load8<TYPE>(a.second, y0 + e, width - e);
            make_s(xe, ye, s[0]);
            if constexpr (NORM) load_gamma(e, gamma[0]);
            put(0, e);
        }
    }
    if (lane == 0 && live)
    {
        double sc = (double) most / (double) a.qmax * a.fold / ((double) hu * (double) hu);
        if (NORM)
        {
            const double ms = (double) sum / ((double) fs * (double) fs) / (double) width;
            sc = top == 0u ? 0.0 : sc / sqrt(ms + a.eps);
        }
        a.scales[row] = bad ? __uint_as_float(0x7FC00000u) : (float) sc;
    }
}

template<int KIND, int TYPE, int LANES, int NV>
hipError_t start(const RowQuantArgs& a, uint32_t threads, hipStream_t s)
{
    const uint32_t per_group = LANES ? 256 / (LANES ? LANES : 1) : 1;
    hipLaunchKernelGGL((row_quant_kernel<KIND, TYPE, LANES, NV>), dim3((a.rows - 1) / per_group + 1), dim3(threads), 0, s, a);
    return hipGetLastError();
}

template<int KIND, int TYPE>
hipError_t start_sized(const RowQuantArgs& a, hipStream_t s)
{
    constexpr bool NORM = KIND == ROWS_NORM || KIND == ROWS_NORM_ADD;
    switch (a.lanes_shared)
    {
        case 16: return start<KIND, TYPE, 16, 1>(a, 256, s);
        case 32: return start<KIND, TYPE, 32, 1>(a, 256, s);
        case 64: return start<KIND, TYPE, 64, 1>(a, 256, s);
        default: break;
    }
    if constexpr (!NORM && TYPE != REAL_FP32)
        if (a.steps == 4) return start<KIND, TYPE, 0, 4>(a, a.lanes, s);
    return a.steps == 1 ? start<KIND, TYPE, 0, 1>(a, a.lanes, s) : a.steps == 2 ? start<KIND, TYPE, 0, 2>(a, a.lanes, s) : start<KIND, TYPE, 0, 0>(a, a.lanes, s);
}

template<int KIND>
hipError_t start_typed(const RowQuantArgs& a, hipStream_t s)
{
    switch (a.type)
    {
        case REAL_BF16: return start_sized<KIND, REAL_BF16>(a, s);
        case REAL_FP16: return start_sized<KIND, REAL_FP16>(a, s);
        default: return start_sized<KIND, REAL_FP32>(a, s);
    }
}
} // namespace

// Lanes without elements cost the instructions of those that have some, so the number of lanes follows the width: as many wavefronts as
// the row needs at 8, 16 or 32 elements a lane.  us (TB/s): norm with residual, bf16 -> e4m3, 8192 x 4096 with 512 lanes x 8
// elements 43.6 (5.4), 256 x 16 46.7, 128 x 32 53.6; 16384 x 1024: 128 x 8 24.7, 64 x 16 26.9, 256 x 8 29.9; without residual, 8192 x 8192: 512 x 16
// 45.3, 1024 x 8 61.3, 256 x 32 57.9; gated, 8192 x 14336: 448 x 32 109.9 (5.3), 1024 x 16 (an eighth of them idle) 116.9.  Rows of up to 512 share a workgroup: norm with
// residual, 16384 x 64: 16 lanes each 5.5, 64 lanes each 10.8.  A workgroup that walks over rows, gamma in registers and the next row on its way,
// needs too many registers: 46.9 for the first of these.
void plan_row_quant(RowQuantArgs& a, int num_cus)
{
    auto lanes = [&](uint32_t steps) {
        a.lanes_shared = 0;
        a.steps = (int) steps;
        a.lanes = ((a.width + steps * VEC * 64 - 1) / (steps * VEC * 64)) * 64;
    };
    const bool norm = a.kind == ROWS_NORM || a.kind == ROWS_NORM_ADD;
    if (a.width <= 512)
    {
        a.lanes_shared = a.width <= 128 ? 16 : a.width <= 256 ? 32 : 64;
        a.lanes = (uint32_t) a.lanes_shared;
        a.steps = 1;
    }
    else if (a.width <= 4096)
        lanes(1);
    else if (a.width > 8192 && a.width <= 16384 && a.rows >= (uint32_t) num_cus && !norm && a.type != REAL_FP32)
        lanes(4); // (sums, gammas and wide inputs want the registers: fp32, gated, 2000 x 11008: 41.0, 38.3 with 16)
    else if (a.width <= 16384)
        lanes(2);
    else
    {
        a.lanes_shared = 0;
        a.lanes = 1024;
        a.steps = 0;
    }
}

hipError_t launch_row_quant(const RowQuantArgs& a, hipStream_t s)
{
    if (a.rows == 0 || a.width == 0) return hipSuccess;
    switch (a.kind)
    {
        case ROWS_PLAIN: return start_typed<ROWS_PLAIN>(a, s);
        case ROWS_GATED: return start_typed<ROWS_GATED>(a, s);
        case ROWS_NORM: return start_typed<ROWS_NORM>(a, s);
        default: return start_typed<ROWS_NORM_ADD>(a, s);
    }
}
} // namespace mme
