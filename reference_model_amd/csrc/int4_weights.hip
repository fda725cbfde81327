// Weights in 4 bits with a scale for each group of columns: from 16-bit floats, from given values and scales, and back.
//
//   scale = round16(max |w| / 7) over the group, v = rint(w / scale) in -7 ... 7 (0 where the scale is 0), w' = v * scale
//
// A wave owns one tile of 16 rows x 128 columns, lane 16 q + r the columns 32 j + 8 q + (0 ... 7) of row r, j = 0 ... 3: the 32 weights whose
// 16 bytes it stores, so a tile goes out as one kilobyte in a row, and the maximum over a group of 32 is a maximum over the four lanes of a row.
// The tiles of a workgroup lie side by side, and their 16-bit side passes through LDS (piece p of row r at p ^ r), so that it is read and written
// in whole kilobytes of a row: where rows begin inside a cache line those meet one line more than they fill, where tile by tile every 64 bytes of
// a row do.  Bound by the 16-bit side: 2 bytes a weight against half of one.  16384 x 4096 takes 36.3 us into 4 bits (4.6 TB/s) and 31.6 back
// (5.3); tile by tile they were 37.5 and 42, and with rows of 4095 57.9 and 74 against 38.4 and 46.8 now.
#include "tmi_ffn.h"

namespace tmi
{
namespace
{

struct Int4Args
{
    const void* in;
    const uint16_t* scales;    // given values only: [n][groups]
    void* out;
    int64_t ld;                // elements between rows on the unpacked side
    int64_t tiles, groups;
    int64_t blocks;            // of 16 rows x 512 columns
    int32_t n, k, tiles_k, across;
};

constexpr int kWaves = 4;

typedef unsigned short v2us __attribute__((ext_vector_type(2)));

// v_cvt_i32_f32 itself: what C leaves undefined is defined there, NaN to 0 and the others to the nearest int32
__device__ __forceinline__ int to_int(float t)
{
    int v;
    asm("v_cvt_i32_f32 %0, %1" : "=v"(v) : "v"(t));
    return v;
}

// the largest bit pattern of |w| over the four lanes of a row; NaN has the largest of all and stays
__device__ __forceinline__ uint32_t row_max(uint32_t v)
{
    uint32_t o = (uint32_t)__shfl_xor((int)v, 16);
    v          = v > o ? v : o;
    o          = (uint32_t)__shfl_xor((int)v, 32);
    return v > o ? v : o;
}

// GIVEN: int8 values (kept to -8 ... 7) and scales; else 16-bit weights, of which with ODD rows begin at odd elements
template <typename T, int PER, bool GIVEN, bool ODD>
__global__ __launch_bounds__(64 * kWaves) void int4_pack_kernel(Int4Args a)
{
    __shared__ v4i lds[GIVEN ? 1 : kInt4Rows * kWaves * 16];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t b = blockIdx.x; b < a.blocks; b += gridDim.x)
    {
        const int64_t tn   = b / a.across;
        const int kt0      = (int)(b - tn * a.across) * kWaves, kt = kt0 + wave;
        const int64_t tile = tn * a.tiles_k + kt;
        const int64_t n    = tn * kInt4Rows + r;
        const bool live    = n < a.n;
        const int k0       = kt * kInt4Cols;
        if constexpr (!GIVEN)
        {
            v4i in[kInt4Rows / kWaves];
#pragma unroll
            for (int i = 0; i < kInt4Rows / kWaves; i++)
            {
                const int64_t m     = tn * kInt4Rows + wave * (kInt4Rows / kWaves) + i;
                const uint16_t* row = static_cast<const uint16_t*>(a.in) + (m < a.n ? m : 0) * a.ld;
                const int k         = kt0 * kInt4Cols + 8 * lane;
                in[i]               = ODD ? load8_words(row, k, a.k, m < a.n) : load8(row, k, a.k, m < a.n);
            }
            if (b != blockIdx.x)
                __syncthreads();    // the last block is read
#pragma unroll
            for (int i = 0; i < kInt4Rows / kWaves; i++)
            {
                const int row                           = wave * (kInt4Rows / kWaves) + i;
                lds[row * (kWaves * 16) + (lane ^ row)] = in[i];
            }
            __syncthreads();
        }
        if (kt >= a.tiles_k)
            continue;
        v4i packed;
        uint16_t scale[PER];
        if constexpr (GIVEN)
        {
            const int8_t* row = static_cast<const int8_t*>(a.in) + (live ? n : 0) * a.ld;
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                uint32_t w = 0;
#pragma unroll
                for (int e = 0; e < 8; e++)
                {
                    const int k = k0 + 32 * j + 8 * q + e;
                    int v       = live && k < a.k ? row[k] : 0;
                    v           = v < -8 ? -8 : (v > 7 ? 7 : v);
                    w |= (uint32_t)(v + 8) << (4 * (e >> 1) + 16 * (e & 1));
                }
                packed[j] = (int)w;
            }
#pragma unroll
            for (int g = 0; g < PER; g++)
            {
                const int64_t at = (int64_t)kt * PER + g;
                scale[g]         = live && at < a.groups ? a.scales[n * a.groups + at] : 0;
            }
        }
        else
        {
            v4i w[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                w[j] = lds[r * (kWaves * 16) + ((wave * 16 + 4 * j + q) ^ r)];
            v2us m[4];    // of |w|, by halves: bit patterns order like the numbers, and NaN above all
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                m[j] = v2us{ 0, 0 };
#pragma unroll
                for (int p = 0; p < 4; p++)
                    m[j] = __builtin_elementwise_max(m[j], __builtin_bit_cast(v2us, w[j][p] & 0x7FFF7FFF));
            }
#pragma unroll
            for (int g = 0; g < PER; g++)
            {
                v2us top = { 0, 0 };
#pragma unroll
                for (int j = g * 4 / PER; j < (g + 1) * 4 / PER; j++)
                    top = __builtin_elementwise_max(top, m[j]);
                scale[g] = to_bits16<T>(from_bits16<T>((uint16_t)row_max(top.x > top.y ? top.x : top.y)) / 7.0f);
                // rint(w / scale) without 32 divisions.  A quotient of two 16-bit floats between -11 and 11 is a half or 2^-13 from one at least, and w times
                // the reciprocal is off by 2^-19 at most: rounded to a multiple of 2^-14 (768 + t has no finer ones) halves are halves again, and no other
                // quotient crosses one.  (bf16 scales may be so small that their reciprocal is none: both sides times 2^64.)
                const float s    = from_bits16<T>(scale[g]);
                const float wide = __is_same(T, bf16_t) && s < 0x1p-60f ? 0x1p64f : 1.0f;
                const float r    = s == 0.0f ? 0.0f : 1.0f / (s * wide);
#pragma unroll
                for (int j = g * 4 / PER; j < (g + 1) * 4 / PER; j++)
                {
                    uint32_t word = 0x88888888u;
#pragma unroll
                    for (int e = 0; e < 8; e++)
                    {
                        float t = from_bits16<T>(half_of(w[j], e));
                        if constexpr (__is_same(T, bf16_t))
                            t *= wide;
                        t = rintf((t * r + 768.0f) - 768.0f);
                        // (the conversion makes 0 of NaN: of inf * 0, and of what is multiplied by NaN)
                        const int v = clamp_med3(to_int(t), -7, 7);
                        word += (uint32_t)v << (4 * (e >> 1) + 16 * (e & 1));
                    }
                    packed[j] = (int)word;
                }
            }
        }
        uint8_t* out = static_cast<uint8_t*>(a.out);
        *reinterpret_cast<v4i*>(out + tile * kInt4TileBytes + lane * 16) = packed;
        if (q == 0)
        {
            uint16_t* s = reinterpret_cast<uint16_t*>(out + int4_scale_at(a.tiles, tile, PER)) + r * PER;
#pragma unroll
            for (int g = 0; g < PER; g++)
                s[g] = scale[g];
        }
    }
}

template <typename T, int PER>
__global__ __launch_bounds__(64 * kWaves) void int4_unpack_kernel(Int4Args a)
{
    __shared__ v4i lds[kInt4Rows * kWaves * 16];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t b = blockIdx.x; b < a.blocks; b += gridDim.x)
    {
        const int64_t tn = b / a.across;
        const int kt0    = (int)(b - tn * a.across) * kWaves;
        if (kt0 + wave < a.tiles_k)
        {
            const int64_t tile = tn * a.tiles_k + kt0 + wave;
            const uint8_t* in  = static_cast<const uint8_t*>(a.in);
            const v4i packed   = *reinterpret_cast<const v4i*>(in + tile * kInt4TileBytes + lane * 16);
            const uint16_t* sc = reinterpret_cast<const uint16_t*>(in + int4_scale_at(a.tiles, tile, PER)) + r * PER;
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                const float s = from_bits16<T>(sc[j * PER / 4]);
                v4i w;
#pragma unroll
                for (int p = 0; p < 4; p++)
                {
                    const uint32_t u = (uint32_t)packed[j] >> (4 * p);
                    w[p] = (int)pack16<T>((float)((int)(u & 15) - 8) * s, (float)((int)(u >> 16 & 15) - 8) * s);
                }
                lds[r * (kWaves * 16) + ((wave * 16 + 4 * j + q) ^ r)] = w;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kInt4Rows / kWaves; i++)
        {
            const int row   = wave * (kInt4Rows / kWaves) + i;
            const int64_t n = tn * kInt4Rows + row;
            if (n < a.n)
                store8(static_cast<uint16_t*>(a.out) + n * a.ld, (int64_t)kt0 * kInt4Cols + lane * 8, a.k, lds[row * (kWaves * 16) + (lane ^ row)]);
        }
        if (b + gridDim.x < a.blocks)
            __syncthreads();    // the block is read
    }
}

template <typename F>
bool per_group(int group, F&& f)
{
    switch (group)
    {
        case 32:
            return f(std::integral_constant<int, 4>()), true;
        case 64:
            return f(std::integral_constant<int, 2>()), true;
        case 128:
            return f(std::integral_constant<int, 1>()), true;
        default:
            return false;
    }
}

// Eight workgroups a CU, which go on to further blocks: 16384 x 4096 36.3 us, 43.0 with a workgroup for each.  (The way back, whose stores nothing waits
// for, takes one for each.)
int grid_of(int64_t blocks)
{
    return (int)(blocks < 2048 ? blocks : 2048);
}

Int4Args int4_args(int32_t n, int32_t k, int group, const void* in, int64_t ld, void* out)
{
    Int4Args a{};
    a.in = in, a.out = out, a.ld = ld, a.n = n, a.k = k;
    a.tiles_k = (int32_t)int4_tiles(k, kInt4Cols);
    a.tiles   = int4_tiles(n, kInt4Rows) * a.tiles_k;
    a.groups  = int4_tiles(k, group);
    a.across  = (int32_t)int4_tiles(a.tiles_k, kWaves);
    a.blocks  = int4_tiles(n, kInt4Rows) * a.across;
    return a;
}

}    // namespace

const char* launch_int4_pack(hipStream_t st, int32_t dtype, int32_t group, int32_t n, int32_t k, const void* w, int64_t ld, const void* scales,
                             void* packed)
{
    Int4Args a    = int4_args(n, k, group, w, ld, packed);
    a.scales      = static_cast<const uint16_t*>(scales);
    const int grid = grid_of(a.blocks);
    const bool odd = !scales && ((ld & 1) || (reinterpret_cast<uintptr_t>(w) & 2));
    const bool ok  = per_group(group, [&](auto per) {
        constexpr int PER = decltype(per)::value;
        auto floats       = [&](auto type, auto ODD) { int4_pack_kernel<decltype(type), PER, false, decltype(ODD)::value><<<grid, 64 * kWaves, 0, st>>>(a); };
        auto typed        = [&](auto type) { odd ? floats(type, std::true_type()) : floats(type, std::false_type()); };
        if (scales)
            int4_pack_kernel<_Float16, PER, true, false><<<grid, 64 * kWaves, 0, st>>>(a);    // (the scales pass through as bits)
        else if (dtype == TMI_BF16)
            typed(bf16_t());
        else
            typed(_Float16());
    });
    return !ok ? nullptr : scales ? "int4_pack" : "int4_quantize";
}

const char* launch_int4_unpack(hipStream_t st, int32_t dtype, int32_t group, int32_t n, int32_t k, const void* packed, void* w, int64_t ld)
{
    const Int4Args a = int4_args(n, k, group, packed, ld, w);
    const int grid   = (int)(a.blocks < 1 << 23 ? a.blocks : 1 << 23);    // (2^32 threads at most)
    const bool ok    = per_group(group, [&](auto per) {
        constexpr int PER = decltype(per)::value;
        if (dtype == TMI_BF16)
            int4_unpack_kernel<bf16_t, PER><<<grid, 64 * kWaves, 0, st>>>(a);
        else
            int4_unpack_kernel<_Float16, PER><<<grid, 64 * kWaves, 0, st>>>(a);
    });
    return ok ? "int4_dequantize" : nullptr;
}

}    // namespace tmi
