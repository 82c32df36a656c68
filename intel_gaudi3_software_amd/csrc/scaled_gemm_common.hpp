// scaled_gemm_common.hpp -- what the kernels of the scaled product share:
//   out[m][n] = (sum_k x[m][k] w[n][k]) sx[m] sw[n] + bias[n]
// over int8 codes (sums in int32, exact) or fp8 codes (sums in fp32).  The matrix-core instructions take the rows of w first, so
// that an accumulator register group runs along n: lane l holds token l % 32 (or l % 16) and four consecutive n at a time.
#pragma once
#include <type_traits>

#include "mme_numeric.hpp"
#include "scaled_kernels.hpp"

namespace mme
{
namespace
{
typedef int   s_v4i __attribute__((ext_vector_type(4)));
typedef int   s_v8i __attribute__((ext_vector_type(8)));
typedef int   s_v16i __attribute__((ext_vector_type(16)));
typedef float s_v4f __attribute__((ext_vector_type(4)));
typedef float s_v16f __attribute__((ext_vector_type(16)));

// OPS: -1 int8; 0 .. 3 fp8, bit 0: x is e5m2, bit 1: w is e5m2
template<int OPS>
struct Sums
{
    typedef s_v16f v16;
    typedef s_v4f  v4;
    typedef float  one;
};
template<>
struct Sums<-1>
{
    typedef s_v16i v16;
    typedef s_v4i  v4;
    typedef int    one;
};

// 32 rows of w x 32 rows of x over 64 k: lane l holds 32 codes of row l % 32; which k they are does not matter as long as both
// operands agree.  int8: two instructions of 32 k, the lower and the upper half of the registers.
template<int OPS>
__device__ __forceinline__ typename Sums<OPS>::v16 mma32(s_v8i w, s_v8i x, typename Sums<OPS>::v16 c)
{
    if constexpr (OPS < 0)
    {
        c = __builtin_amdgcn_mfma_i32_32x32x32_i8(s_v4i {w[0], w[1], w[2], w[3]}, s_v4i {x[0], x[1], x[2], x[3]}, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(s_v4i {w[4], w[5], w[6], w[7]}, s_v4i {x[4], x[5], x[6], x[7]}, c, 0, 0, 0);
    }
    else
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, (OPS >> 1) & 1, OPS & 1, 0, 0, 0, 0);
}
// 16 x 16 over 128 k: lane l holds 32 codes of row l % 16
template<int OPS>
__device__ __forceinline__ typename Sums<OPS>::v4 mma16(s_v8i w, s_v8i x, typename Sums<OPS>::v4 c)
{
    if constexpr (OPS < 0)
    {
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(s_v4i {w[0], w[1], w[2], w[3]}, s_v4i {x[0], x[1], x[2], x[3]}, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(s_v4i {w[4], w[5], w[6], w[7]}, s_v4i {x[4], x[5], x[6], x[7]}, c, 0, 0, 0);
    }
    else
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, (OPS >> 1) & 1, OPS & 1, 0, 0, 0, 0);
}

struct __attribute__((packed, aligned(1))) u128_any
{
    uint32_t v[4];
};

// sixteen codes moved down by n of them, zeros after them (none move for n <= 0, none stay for n >= 16)
__device__ __forceinline__ s_v4i moved_down(s_v4i v, int n)
{
    const int          bits = 8 * min(max(n, 0), 16);
    unsigned long long lo = ((unsigned long long) (uint32_t) v.y << 32) | (uint32_t) v.x, hi = ((unsigned long long) (uint32_t) v.w << 32) | (uint32_t) v.z;
    lo = bits >= 128 ? 0ull : bits >= 64 ? hi >> (bits & 63) : bits ? (lo >> bits) | (hi << (64 - bits)) : lo;
    hi = bits >= 64 ? 0ull : hi >> bits;
    return s_v4i {(int) (uint32_t) lo, (int) (uint32_t) (lo >> 32), (int) (uint32_t) hi, (int) (uint32_t) (hi >> 32)};
}
// 16 codes of a row from k on, at any alignment, zeros behind the row's end
__device__ __forceinline__ s_v4i load16(const uint8_t* row, int k, int K)
{
    if (k + 16 <= K)
    {
        const u128_any u = *(const u128_any*) (row + k);
        return s_v4i {(int) u.v[0], (int) u.v[1], (int) u.v[2], (int) u.v[3]};
    }
    if (k >= K) return s_v4i {0, 0, 0, 0};
    if (K >= 16)
    {
        // the row's last sixteen codes, moved down by those that come before k
        const u128_any u = *(const u128_any*) (row + K - 16);
        return moved_down(s_v4i {(int) u.v[0], (int) u.v[1], (int) u.v[2], (int) u.v[3]}, k + 16 - K);
    }
    uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (k + i < K) v[i / 4] |= (uint32_t) row[k + i] << (8 * (i & 3));
    return s_v4i {(int) v[0], (int) v[1], (int) v[2], (int) v[3]};
}
__device__ __forceinline__ s_v8i join(s_v4i lo, s_v4i hi) { return s_v8i {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}; }

// 16 bytes per lane from global memory to LDS at lds_off + lane * 16 (lds_off is wave-uniform), outside the compiler's memory model:
// the wavefront waits for its requests by count
__device__ __forceinline__ void dma16(const void* g, uint32_t lds_off)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds_off) : "memory");
}
// where a row of 128 bytes keeps its 16-byte chunk c: at c ^ swizzle(row).  A line of all LDS banks holds two rows, so sixteen rows with
// the same c meet every bank once.
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }
constexpr int vm_wait(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); } // at most n of the wavefront's requests outstanding

struct BatchOffsets
{
    long long x, w, out, sx, sw;
};
__device__ __forceinline__ BatchOffsets batch_offsets(const ScaledGemmArgs& a, int b)
{
    const int b0 = b % a.batch[0], r = b / a.batch[0], b1 = r % a.batch[1], b2 = r / a.batch[1];
    auto at = [&](const long long (&st)[3]) { return b0 * st[0] + b1 * st[1] + b2 * st[2]; };
    return BatchOffsets {at(a.x_bs), at(a.w_bs), at(a.out_bs), at(a.sx_bs), at(a.sw_bs)};
}

// the value that is rounded into the output: one rounding of a whole sum to fp32, two multiplications, one addition, each rounded
// once (the factors one after the other: their product may leave the fp32 range where the result does not)
template<class S>
__device__ __forceinline__ float scaled_value(S sum, float alpha, float sx, float sw, float bias, bool has_bias)
{
    float v = (float) sum;
    if constexpr (std::is_same<S, float>::value) v *= alpha;
    v *= sx;
    return has_bias ? __builtin_fmaf(v, sw, bias) : v * sw;
}
__device__ __forceinline__ uint16_t to_half(float v, int out_type)
{
    uint16_t u;
    if (out_type == SCALED_OUT_BF16)
    {
        const __bf16 h = (__bf16) v;
        __builtin_memcpy(&u, &h, 2);
    }
    else
    {
        const _Float16 h = (_Float16) v;
        __builtin_memcpy(&u, &h, 2);
    }
    return u;
}

struct __attribute__((packed, aligned(1))) u64_any
{
    uint32_t v[2];
};
struct __attribute__((packed, aligned(4))) f128_any
{
    float v[4];
};

// scales and biases of four consecutive columns n .. n + 3 (those below N)
struct Columns
{
    f128_any sw, bias;
};
__device__ __forceinline__ Columns columns_of(const ScaledGemmArgs& a, const BatchOffsets& o, int n)
{
    Columns c = {{{1.0f, 1.0f, 1.0f, 1.0f}}, {{0.0f, 0.0f, 0.0f, 0.0f}}};
    if (n + 4 <= a.N)
    {
        if (a.sw) c.sw = *(const f128_any*) (a.sw + o.sw + n);
        if (a.bias) c.bias = *(const f128_any*) (a.bias + o.sw + n);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            const int q = min(n + i, a.N - 1);
            if (a.sw) c.sw.v[i] = a.sw[o.sw + q];
            if (a.bias) c.bias.v[i] = a.bias[o.sw + q];
        }
    }
    return c;
}

// stores four consecutive outputs n .. n + 3 of row m (those below N), from their sums; sx: the row's scale
template<class S>
__device__ __forceinline__ void store_scaled4(const ScaledGemmArgs& a, const BatchOffsets& o, int m, int n, float sx, const Columns& c, const S (&sum)[4])
{
    const long long e = o.out + (long long) m * a.out_ld + n;
    const bool      whole = n + 4 <= a.N;
    float           v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = scaled_value(sum[i], a.alpha, sx, c.sw.v[i], c.bias.v[i], a.bias != nullptr);
    if constexpr (std::is_same<S, int>::value) // (fp8 operands have 16-bit outputs)
        if (a.out_type == SCALED_OUT_FP32 || a.out_type == SCALED_OUT_INT32)
        {
            uint32_t* p = (uint32_t*) a.out + e;
            uint32_t  word[4];
#pragma unroll
            for (int i = 0; i < 4; i++) word[i] = a.out_type == SCALED_OUT_INT32 ? (uint32_t) sum[i] : __float_as_uint(v[i]);
            if (whole) *(u128_any*) p = u128_any {{word[0], word[1], word[2], word[3]}};
            else
            {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (n + i < a.N) p[i] = word[i];
            }
            return;
        }
    uint16_t* p = (uint16_t*) a.out + e;
    uint32_t  half[4];
#pragma unroll
    for (int i = 0; i < 4; i++) half[i] = to_half(v[i], a.out_type);
    if (whole) *(u64_any*) p = u64_any {{half[0] | (half[1] << 16), half[2] | (half[3] << 16)}};
    else
    {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (n + i < a.N) p[i] = (uint16_t) half[i];
    }
}
__device__ __forceinline__ float scale_of_row(const ScaledGemmArgs& a, const BatchOffsets& o, int m) { return a.sx ? a.sx[o.sx + min(m, a.M - 1)] : 1.0f; }
} // namespace
} // namespace mme
