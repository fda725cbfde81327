// What the kernels that work on rows of activations share: pieces of 16 bytes of rows that begin at any element, sums and maxima over the lanes of
// a row, and numbers into 8 bits.
#pragma once
#include "tmi_ffn.h"

namespace tmi
{

// T is _Float16, bf16_t or float; a piece holds kPiece<T> elements
template <typename T>
constexpr int kPiece = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ float piece_get(v4i v, int e)    // e a constant
{
    if constexpr (sizeof(T) == 4)
        return __int_as_float(v[e]);
    else
        return from_bits16<T>(half_of(v, e));
}
// v[0 .. kPiece) rounded to T
template <typename T>
__device__ __forceinline__ v4i piece_of(const float* v)
{
    if constexpr (sizeof(T) == 4)
        return v4i{ __float_as_int(v[0]), __float_as_int(v[1]), __float_as_int(v[2]), __float_as_int(v[3]) };
    else
        return v4i{ (int)pack16<T>(v[0], v[1]), (int)pack16<T>(v[2], v[3]), (int)pack16<T>(v[4], v[5]), (int)pack16<T>(v[6], v[7]) };
}

// Elements k, k + 1, ... of a row of `width`, zeros from its end on; k a multiple of kPiece.  Nothing outside the row is read.  WHOLE: rows are whole
// pieces and begin at whole words, so that every piece is one load; else a piece that the row ends in is made of its last elements, and what begins inside
// a word is read in words (tmi_ffn.h).
template <typename T, bool WHOLE>
__device__ __forceinline__ v4i load_piece(const T* row, int k, int width)
{
    if constexpr (WHOLE)
    {
        const v4i v = load16(reinterpret_cast<const uint8_t*>(row + (k < width ? k : 0)));
        return k < width ? v : v4i{ 0, 0, 0, 0 };
    }
    else if constexpr (sizeof(T) == 2)
        return load8_words(reinterpret_cast<const uint16_t*>(row), k, width, true);
    else
    {
        v4i v = { 0, 0, 0, 0 };
        if (width >= 4)
        {
            const int beyond = k + 4 - width;
            v                = load16(reinterpret_cast<const uint8_t*>(row + (beyond > 0 ? width - 4 : k)));
            if (beyond > 0)
                v = beyond < 4 ? drop_front(v, 4 * beyond) : v4i{ 0, 0, 0, 0 };
            return v;
        }
#pragma unroll
        for (int e = 0; e < 3; e++)
            if (k + e < width)
                v[e] = __float_as_int(row[k + e]);
        return v;
    }
}
// The same without touching another piece's elements, for passes that write the row they read
template <typename T, bool WHOLE>
__device__ __forceinline__ v4i load_piece_alone(const T* row, int k, int width)
{
    if (WHOLE || k + kPiece<T> <= width)
        return load_piece<T, WHOLE>(row, k, width);
    v4i v = { 0, 0, 0, 0 };
#pragma unroll
    for (int e = 0; e < kPiece<T> - 1; e++)
        if (k + e < width)
        {
            if constexpr (sizeof(T) == 4)
                v[e] = __float_as_int(row[k + e]);
            else
                v[e >> 1] |= (int)((uint32_t)__builtin_bit_cast(uint16_t, row[k + e]) << (16 * (e & 1)));
        }
    return v;
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void store_piece(T* row, int k, int width, v4i v)
{
    if (WHOLE ? k < width : k + kPiece<T> <= width)
        __builtin_memcpy(row + k, &v, 16);
    else if (!WHOLE)
    {
        if constexpr (sizeof(T) == 2)
            store8(reinterpret_cast<uint16_t*>(row), k, width, v);
        else
#pragma unroll
            for (int e = 0; e < 3; e++)
                if (k + e < width)
                    row[k + e] = __int_as_float(v[e]);
    }
}

// ---- over the G lanes of a row: 8 to 64 of a wave, or all of a workgroup ------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ uint32_t from_lane(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b)
{
    return a > b ? a : b;
}
// within 16 lanes (or eight): the neighbour, the other pair, the other four, the other eight
template <bool SUM, bool MOST, int G = 16>
__device__ __forceinline__ void over_16(float& sum, uint32_t& most)
{
    auto step = [&](auto CTRL) {
        if constexpr (SUM)
            sum += __uint_as_float(from_lane<decltype(CTRL)::value>(__float_as_uint(sum)));
        if constexpr (MOST)
            most = max_u32(most, from_lane<decltype(CTRL)::value>(most));
    };
    step(std::integral_constant<int, 0xB1>());
    step(std::integral_constant<int, 0x4E>());
    step(std::integral_constant<int, 0x141>());
    if constexpr (G == 16)
        step(std::integral_constant<int, 0x140>());
}
// within 32: the other 16, lane l ^ 16
template <bool SUM, bool MOST>
__device__ __forceinline__ void over_32(float& sum, uint32_t& most)
{
    over_16<SUM, MOST>(sum, most);
    auto other = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x401F); };
    if constexpr (SUM)
        sum += __uint_as_float(other(__float_as_uint(sum)));
    if constexpr (MOST)
        most = max_u32(most, other(most));
}
template <bool SUM, bool MOST>
__device__ __forceinline__ void over_64(float& sum, uint32_t& most)
{
    over_16<SUM, MOST>(sum, most);
    auto lane = [](uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    if constexpr (SUM)
    {
        const uint32_t s = __float_as_uint(sum);
        sum = (__uint_as_float(lane(s, 0)) + __uint_as_float(lane(s, 16))) + (__uint_as_float(lane(s, 32)) + __uint_as_float(lane(s, 48)));
    }
    if constexpr (MOST)
        most = max_u32(max_u32(lane(most, 0), lane(most, 16)), max_u32(lane(most, 32), lane(most, 48)));
}
// `slot`: 2 * G / 64 words of LDS that no lane reads from an earlier call once another barrier is passed
template <int G, bool SUM, bool MOST>
__device__ __forceinline__ void over_row(float& sum, uint32_t& most, uint32_t* slot)
{
    if constexpr (G <= 16)
        over_16<SUM, MOST, G>(sum, most);
    else if constexpr (G == 32)
        over_32<SUM, MOST>(sum, most);
    else
        over_64<SUM, MOST>(sum, most);
    if constexpr (G > 64)
    {
        constexpr int W = G / 64;
        const int wave  = __builtin_amdgcn_readfirstlane(threadIdx.x % G >> 6);
        if ((threadIdx.x & 63) == 0)
        {
            if constexpr (SUM)
                slot[wave] = __float_as_uint(sum);
            if constexpr (MOST)
                slot[W + wave] = most;
        }
        __syncthreads();
        if constexpr (SUM)
        {
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++)
                sum += __uint_as_float(slot[w]);
        }
        if constexpr (MOST)
        {
            most = 0;
#pragma unroll
            for (int w = 0; w < W; w++)
                most = max_u32(most, slot[W + w]);
        }
    }
}

// ---- 8 bits ---------------------------------------------------------------------------------------------------------------------
// v scale rounded to the nearest integer (ties to even) in a word's lowest byte, up to 127: 1.5 2^23 + that has no finer digits
constexpr float kByteZero = 12582912.0f;
__device__ __forceinline__ uint32_t to_byte(float v, float scale)
{
    return __float_as_uint(__builtin_fmaf(v, scale, kByteZero));
}
__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), hi = __builtin_amdgcn_perm(d, c, 0x0C0C0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
template <typename T>
constexpr bool kWholeWords = sizeof(T) == 4;
// whether rows of `width` elements, `ld` apart, are whole pieces that begin at whole words (rows of none may have no address at all: the other form reads nothing then)
template <typename T>
inline bool whole_rows(const void* p, int64_t width, int64_t ld)
{
    return width > 0 && width % kPiece<T> == 0 && (kWholeWords<T> || (((uintptr_t)p & 3) == 0 && ld % 2 == 0));
}

}    // namespace tmi
