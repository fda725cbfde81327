// What the feed-forward kernels share: the activations and their slopes, rounding to 16 bits, 16-byte loads at the ends of rows, the 16x16
// matrix instruction of 16-bit floats, and the layout of 4-bit weights.
#pragma once
#include "tmi_mfma.h"
#include <type_traits>

namespace tmi
{

// act(g) in 32 bits.  Relative errors in units of 2^-24, for negative g, where the tails are (from an emulation in 32 bits; an exponent's rounding counts as
// often as it is large): SiLU and sigmoid 5 down to -16, 21 at -80; GELU 15 down to -4, 49 at -8, 126 at -13; its tanh form 22, 120 and, at -9, 193.  A
// bf16 number's rounding is 65536 such units, an fp16 one's 8192.  GELU goes by the smaller tail of the normal distribution, which keeps its digits where
// 1 + erf cancels, and its tanh form by (1 + tanh z) / 2 = 1 / (1 + exp(-2z)) for the same reason.
//
// 1 / (1 + exp(-z)) without a division and without a library's exp (which take twice as many instructions): with E = exp(-|z|) in [0, 1] it is
// 1 / (1 + E) or E / (1 + E), and the reciprocal's argument lies in [1, 2].  E is the square of 2^(-|z| log2(e) / 2), so that it may be subnormal,
// put right by what rounding the exponent took.  |z| is cut where E has long been 0, for the difference of infinities that an infinite one would make.
// Of the value p and its complement q = 1 / (1 + exp(z)) each has all its digits: 1 - p would lose those of q for positive z, all of them from 17.3 on.
__device__ __forceinline__ void logistic_both(float z, float& p, float& q)
{
    constexpr float c = -0.72134752044448170f;    // -log2(e) / 2
    const float a     = fabsf(z) > 512.0f ? 512.0f : fabsf(z);    // (NaN stays)
    const float m     = a * c, off = __builtin_fmaf(a, c, -m);
    const float root  = __builtin_amdgcn_exp2f(m);
    float e           = root * root;
    e                 = __builtin_fmaf(e, off * 1.38629436111989062f, e);    // 2 ln 2
    const float r     = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    p = z < 0.0f ? er : r, q = z < 0.0f ? r : er;
}
__device__ __forceinline__ float logistic(float z)
{
    float p, q;
    logistic_both(z, p, q);
    return p;
}
// Phi(g), the normal distribution's cdf, and its density.  The tail beyond a = |g| is exp(-a^2 / 2) t S(t) with t = 1 / (1 + 0.32 a): S is a
// polynomial of degree 9 fitted to it for the least relative error over all a (3e-8, evaluated in 32 bits 6 units of 2^-24; the exponential's argument adds
// what stands above, which grows with a^2).
__device__ __forceinline__ void normal_cdf(float g, float& cdf, float& density)
{
    const float a = fabsf(g);
    const float q = __builtin_amdgcn_exp2f(a * a * -0.36067376022224085f);    // exp(-a^2 / 4): its square may be subnormal
    const float e = q * q;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.32f, 1.0f));
    constexpr float c[10] = { 0.12766152873901945f, 0.12766094660968072f,  0.11462236066479739f, 0.0878290712309933f,   0.05865412892826976f,
                              -0.009378066554101408f, 0.06532888519285915f, -0.14670831921551367f, 0.09540772027734175f, -0.021078271849041576f };
    float s = c[9];
#pragma unroll
    for (int k = 8; k >= 0; k--)
        s = __builtin_fmaf(s, t, c[k]);
    const float tail = s * t * e;
    cdf = g > 0.0f ? 1.0f - tail : tail, density = e * 0.39894228040143268f;
}
constexpr float kGeluTwoC  = 1.5957691216057308f;    // 2 sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;
__device__ __forceinline__ float gelu_tanh_twice(float g)    // 2z
{
    return kGeluTwoC * (g + kGeluCubic * g * g * g);
}
// act(g); ACT a constant, so that a kernel chooses once and not for each element (for_act)
template <int ACT>
__device__ __forceinline__ float act_value(float g)
{
    if constexpr (ACT == TMI_ACT_SILU)
        return g * logistic(g);
    else if constexpr (ACT == TMI_ACT_GELU)
    {
        float cdf, density;
        normal_cdf(g, cdf, density);
        return g * cdf;
    }
    else if constexpr (ACT == TMI_ACT_GELU_TANH)
        return g * logistic(gelu_tanh_twice(g));
    else if constexpr (ACT == TMI_ACT_RELU)
        return g < 0.0f ? 0.0f : g;    // (NaN stays)
    else
        return logistic(g);
}
// act(g) and act'(g)
template <int ACT>
__device__ __forceinline__ void act_both(float g, float& value, float& slope)
{
    if constexpr (ACT == TMI_ACT_SILU)
    {
        float p, q;
        logistic_both(g, p, q);
        value = g * p, slope = p * (1.0f + g * q);
    }
    else if constexpr (ACT == TMI_ACT_GELU)
    {
        float cdf, density;
        normal_cdf(g, cdf, density);
        value = g * cdf, slope = cdf + g * density;
    }
    else if constexpr (ACT == TMI_ACT_GELU_TANH)
    {
        float p, q;
        logistic_both(gelu_tanh_twice(g), p, q);
        const float pq = p * q;
        // far out p is 0 or 1 and g * g may be infinite
        value = g * p, slope = pq == 0.0f ? p : p + g * pq * (kGeluTwoC * (1.0f + 3.0f * kGeluCubic * g * g));
    }
    else if constexpr (ACT == TMI_ACT_RELU)
        value = g < 0.0f ? 0.0f : g, slope = g > 0.0f ? 1.0f : 0.0f;
    else
    {
        float p, q;
        logistic_both(g, p, q);
        value = p, slope = p * q;
    }
}
template <typename F>
__device__ __forceinline__ void for_act(int act, F&& f)
{
    switch (act)
    {
        case TMI_ACT_SILU:
            return f(std::integral_constant<int, TMI_ACT_SILU>());
        case TMI_ACT_GELU:
            return f(std::integral_constant<int, TMI_ACT_GELU>());
        case TMI_ACT_GELU_TANH:
            return f(std::integral_constant<int, TMI_ACT_GELU_TANH>());
        case TMI_ACT_RELU:
            return f(std::integral_constant<int, TMI_ACT_RELU>());
        default:
            return f(std::integral_constant<int, TMI_ACT_SIGMOID>());
    }
}

// ---- 16-bit floats: T is _Float16 or bf16_t (its bits) -----------------------------------------------------------------------
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ uint16_t to_bits16(float v)    // rounded to nearest, ties to even
{
    if constexpr (sizeof(T) == 2 && !__is_same(T, bf16_t))
        return __builtin_bit_cast(uint16_t, (_Float16)v);
    else
        return __builtin_bit_cast(uint16_t, (__bf16)v);
}
template <typename T>
__device__ __forceinline__ float from_bits16(uint16_t b)
{
    if constexpr (__is_same(T, bf16_t))
        return __uint_as_float((uint32_t)b << 16);
    else
        return (float)__builtin_bit_cast(_Float16, b);
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi)
{
    return (uint32_t)to_bits16<T>(lo) | (uint32_t)to_bits16<T>(hi) << 16;
}
__device__ __forceinline__ uint16_t half_of(v4i v, int e)    // e a constant
{
    return (uint16_t)((uint32_t)v[e >> 1] >> (16 * (e & 1)));
}

// The two halves of load8 for rows of eight elements at least: what is read, and what is made of it once it is there
__device__ __forceinline__ v4i load8_raw(const uint16_t* row, int64_t k, int64_t end)
{
    return load16(reinterpret_cast<const uint8_t*>(row + (k + 8 <= end ? k : end - 8)));
}
__device__ __forceinline__ v4i settle8(v4i v, int64_t k, int64_t end, bool inside)
{
    const int beyond = k + 8 <= end ? 0 : (int)(k + 8 - end);
    if (beyond)
        v = drop_front(v, 2 * (beyond < 8 ? beyond : 7));
    return inside && beyond < 8 ? v : v4i{ 0, 0, 0, 0 };
}
// Eight elements of a row from column k on; zeros at and behind `end`, and everywhere unless `inside` (the row has to be one that can be read all
// the same).  Nothing outside the row is read, and it may begin at any element.  A piece that the row ends in is the row's last eight elements,
// moved: one load without a branch, where picking the elements one by one costs as many waits.
__device__ __forceinline__ v4i load8(const uint16_t* row, int64_t k, int64_t end, bool inside = true)
{
    if (end >= 8)
        return settle8(load8_raw(row, k, end), k, end, inside);
    v4i v = { 0, 0, 0, 0 };
#pragma unroll
    for (int e = 0; e < 7; e++)
        if (inside && k + e < end)
            v[e >> 1] |= (int)((uint32_t)row[k + e] << (16 * (e & 1)));
    return v;
}
// A row that begins at an odd element is read in words: 16 bytes from the word on that it begins in, and the one word behind them where that one
// holds more of the row; joined() then moves the halves.  Loads of 16 bytes that begin inside a word take the caches more than twice as long.
struct Halves
{
    const uint8_t* base;
    uint32_t shift;    // 0 or 16
    __device__ __forceinline__ const uint16_t* row() const { return reinterpret_cast<const uint16_t*>(base + (shift >> 3)); }
    // of the 16 bytes at `at`: the fifth word, or the fourth again
    __device__ __forceinline__ int next(int64_t at) const { return *reinterpret_cast<const int*>(base + at + 12 + (shift >> 2)); }
};
__device__ __forceinline__ Halves halves_of(const uint8_t* row)
{
    const uint32_t odd = (uint32_t)reinterpret_cast<uintptr_t>(row) & 2;
    return { row - odd, 8 * odd };
}
__device__ __forceinline__ v4i joined(v4i v, int next, uint32_t shift)
{
    return v4i{ (int)__builtin_amdgcn_alignbit(v[1], v[0], shift), (int)__builtin_amdgcn_alignbit(v[2], v[1], shift),
                (int)__builtin_amdgcn_alignbit(v[3], v[2], shift), (int)__builtin_amdgcn_alignbit(next, v[3], shift) };
}
// load8 that way
__device__ __forceinline__ v4i load8_words(const uint16_t* row, int64_t k, int64_t end, bool inside)
{
    if (end < 8)
        return load8(row, k, end, inside);
    const Halves h = halves_of(reinterpret_cast<const uint8_t*>(row + (k + 8 <= end ? k : end - 8)));
    return settle8(joined(load16(h.base), h.next(0), h.shift), k, end, inside);
}
// the same way out
__device__ __forceinline__ void store8(uint16_t* row, int64_t k, int64_t end, v4i v)
{
    if (k + 8 <= end)
    {
        __builtin_memcpy(row + k, &v, 16);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (k + e < end)
            row[k + e] = half_of(v, e);
}

// One 16x16 step over 32 columns: lane l holds columns [8 (l / 16), + 8) of row l % 16 of either operand; of the result row 4 (l / 16) + i
// of the first operand against row l % 16 of the second, i = 0..3.
template <typename T>
__device__ __forceinline__ v4f mma16(v4i a, v4i b, v4f c)
{
    if constexpr (__is_same(T, bf16_t))
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// ---- 4-bit weights: the layout that tosa_mi355.h gives --------------------------------------------------------------------------
constexpr int kInt4Rows = 16, kInt4Cols = 128, kInt4TileBytes = 1024;

__host__ __device__ inline int64_t int4_tiles(int64_t n, int64_t per)
{
    return (n + per - 1) / per;
}
// byte of the scales of tile (row tile, column tile); `tiles` = all tiles, `per` = groups of a tile
__host__ __device__ inline int64_t int4_scale_at(int64_t tiles, int64_t tile, int per)
{
    return tiles * kInt4TileBytes + tile * (kInt4Rows * 2) * per;
}

// The eight weights of a word as 16-bit floats, times kInt4Unit.  fp16: a nibble in the mantissa of 1024 gives 1024 + u, one four bits higher
// 1024 + 16 u; u - 8 is then one exact packed operation.  bf16 has seven bits of mantissa and no packed arithmetic: the conversion of a signed
// nibble to 32 bits (a sixteenth of its value), of which the upper halves are the bf16 numbers.
template <typename T>
constexpr float kInt4Unit = __is_same(T, bf16_t) ? 1.0f / 16 : 1.0f;

template <typename T>
__device__ __forceinline__ v4i int4_unpack(uint32_t w)
{
    v4i r;
    if constexpr (__is_same(T, bf16_t))
    {
        uint32_t s[2] = { w ^ 0x88888888u };    // v + 8 -> v, two's complement
        // (one operation each: the conversion itself picks the byte)
        asm("" : "+v"(s[0]));
        s[1] = s[0] >> 4;
        asm("" : "+v"(s[1]));
#pragma unroll
        for (int p = 0; p < 4; p++)
        {
            const int byte = 8 * (p >> 1);
            const float lo = __builtin_amdgcn_cvt_off_f32_i4((int)__builtin_amdgcn_ubfe(s[p & 1], byte, 8));
            const float hi = __builtin_amdgcn_cvt_off_f32_i4((int)__builtin_amdgcn_ubfe(s[p & 1], byte + 16, 8));
            r[p] = (int)__builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
        }
    }
    else
    {
        const v2h off0 = { (_Float16)-1032.0f, (_Float16)-1032.0f }, off1 = { (_Float16)-72.0f, (_Float16)-72.0f };
        const v2h sixteenth = { (_Float16)0.0625f, (_Float16)0.0625f };
        // (held in registers, so that a mask and the exponent are one operation: an instruction takes one constant)
        uint32_t low = 0x000F000Fu, high = 0x00F000F0u, exponent = 0x64006400u;
        asm("" : "+s"(low), "+s"(high), "+v"(exponent));
#pragma unroll
        for (int p = 0; p < 4; p += 2)
        {
            const uint32_t s = w >> (4 * p);
            const v2h lo = __builtin_bit_cast(v2h, (s & low) | exponent), hi = __builtin_bit_cast(v2h, (s & high) | exponent);
            r[p]     = __builtin_bit_cast(int, lo + off0);
            r[p + 1] = __builtin_bit_cast(int, __builtin_elementwise_fma(hi, sixteenth, off1));
        }
    }
    return r;
}

}    // namespace tmi
