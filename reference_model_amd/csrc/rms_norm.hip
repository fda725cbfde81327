// The root-mean-square norm with the residual's addition, in 16 or 32 bits or straight into 8 bits, and rows into 8 bits and back:
//
//   s = x + residual                 sum = s, rounded
//   r = 1 / sqrt(mean(s^2) + eps)    over a row
//   y = s r (offset + w)
//   8 bits: scale = max |y| / 127, q = y / scale, rounded (or of x itself, without a norm)
//
// Bound by memory: a row is read once into registers, everything is done there, and it is written once.  In 8 bits r is in no element: max |y| is
// r max |s (offset + w)|, so the one trip over the lanes that adds the squares finds the maximum too, q is s (offset + w) times 127 over that
// maximum, and r only enters the scale.
//
// A row has 8 to 64 lanes of a wave, 256 or 1024 of a workgroup, each with P pieces of 16 bytes; longer rows are read a second time (norm_long_kernel).
// us and TB/s: 4096 x 8192 fp16 with residual and sum 48.2, 5.6 (a copy of as many bytes runs at 6.1); 131072 x 128 bf16 12 to 13, 5.3; 4096 x 4096 bf16 with residual and
// sum 25.9, 5.2, into 8 bits 24.5, 4.8; 16384 x 4096 bf16 into 8 bits 37.4, 5.4 (38 to 46 right behind the way back, whose results are on their way to memory then), and back 37.5,
// 5.4 (29 behind the way there, which leaves part of q in the last cache); one row of 4096 2.9.  Rows of 4095 elements, read in words: 32.1 for 25.9, 29.7 for 24.5, 40.1
// for 37.4.  Rows of 8-byte stores: 16 bytes joined from two lanes gave the same (36.5 for 36.4).
//
// Squares and products may leave the range of 32 bits where the results do not: bf16 and 32-bit rows whose sum or maximum overflows, or is so small that digits are
// lost, are taken again times a power of two, each in its own units.  That is decided for a row as a whole, from what the reduction found.
#include "tmi_rows.h"

namespace tmi
{
namespace
{

enum
{
    NORM,         // y
    NORM_INT8,    // y in 8 bits
    INT8          // x in 8 bits
};

struct NormArgs
{
    const void *x, *residual, *weight;
    void *sum, *out;
    float* of_row;    // 1 / rms, or the scales
    int64_t ld_x, ld_residual, ld_sum, ld_out;
    int64_t rows;
    int32_t width;
    float eps, offset;
};

constexpr float kSmall = 0x1p-80f, kUp = 0x1p100f, kDown = 0x1p-80f;

// (products this small may have a scale of 0: times 2^-64, the least 1 / rms of squares that 32 bits hold, and over 127)
constexpr float kSmallProduct = 0x1p-77f;
constexpr int kUpProducts = 200, kDownProducts = -130;    // (exponents: products under that, and up to 2^256, become numbers of the usual size)

// whether products of this size need no other units
__device__ __forceinline__ bool fine(uint32_t most)
{
    return __uint_as_float(most) >= kSmallProduct && __uint_as_float(most) < __builtin_huge_valf();
}

// (fp16: squares up to 2^34 and products up to 2^33, down to 2^-48)
template <typename T>
constexpr bool kLeavesRange = !__is_same(T, _Float16);
// Whether a row's sum or its maximum, as the lanes found them, have to be taken again
template <typename T, int MODE>
__device__ __forceinline__ bool leaves_range(float squares, uint32_t most, float eps)
{
    if constexpr (!kLeavesRange<T>)
        return false;
    else if constexpr (MODE == INT8)
        return most != 0 && __uint_as_float(most) < kSmallProduct;
    else
        return !(squares < __builtin_huge_valf()) || (squares < kSmall && eps < kSmall) || (MODE == NORM_INT8 && !fine(most));
}
// What the elements are multiplied by before their squares are added again; 1: those are fine.  (So small a sum is taken again for the products' sake too: zero
// is then a row of zeros)
template <int MODE>
__device__ __forceinline__ float squares_again(float squares)
{
    return MODE == INT8 || (squares >= kSmall && squares < __builtin_huge_valf()) ? 1.0f : squares < kSmall ? kUp : kDown;
}
// The units, 2 to the minus this, in which the products are taken again; 0: they are fine, or all zero
template <int MODE>
__device__ __forceinline__ int products_again(float squares, uint32_t most)
{
    return MODE == NORM || fine(most) || (MODE == NORM_INT8 && squares == 0.0f) ? 0 : __uint_as_float(most) < kSmallProduct ? kUpProducts : kDownProducts;
}
// s w 2^units, wherever s and w are in the range; rounded once.  (The compiler is not to keep the parts of rows and weights in registers, which halved the waves a SIMD)
__device__ __forceinline__ float product_in(float s, float w, int units)
{
    asm volatile("" : "+v"(s), "+v"(w));
    return __builtin_ldexpf(__builtin_amdgcn_frexp_mantf(s) * __builtin_amdgcn_frexp_mantf(w), __builtin_amdgcn_frexp_expf(s) + __builtin_amdgcn_frexp_expf(w) + units);
}

// What becomes of a row once its sum and maximum are known
struct OfRow
{
    float times;     // NORM: r; else 127 / max |y| over r, 0 where there is no such number
    float stored;    // 1 / rms or the scale
    float unit;      // max |y| over 127 r where quotients may be halves that `times` does not send to the even number, else 0
};

// 127 / m rounded up.  What the norm makes are products of 16-bit numbers, exact in 32 bits more often than not, and halves of a row's maximum among them: 20 to 50
// in 4096 x 4096 bf16 with a residual, half of which a rounded reciprocal sends to the odd number.  127 v / m is half an odd number k where 254 v = k m: v = m / 2, or 127
// divides m.  Rounded up, v = m / 2 becomes 63.5 or more, and so 64, the even one.
__device__ __forceinline__ float reciprocal_up(float m)
{
    const float f = 127.0f / m;
    return __builtin_fmaf(f, m, -127.0f) < 0.0f ? __uint_as_float(__float_as_uint(f) + 1) : f;
}
// Other halves are in rows whose m has m / 127 in 17 bits, which is what this gives then (1 / 127 in 32 bits is off by 2^-28 of itself), and 0 of any other: one in
// 127, 3 % where neither x nor the weights have more than eight bits.  There the quotient's error, v less a multiple of that, is exact in 32 bits, and added to it.
// us into 8 bits with both, and with 127 / m as it is: 131072 x 128 13.1 and 12.8, 4096 x 4096 with residual and sum 24.2 and 24.3, 16384 x 4096 40.3 and 40.1.  A test of each
// quotient for being near a half took 14.1, 24.5 and 43.5.
__device__ __forceinline__ float whole_127th(float m)
{
    const float u = m * (1.0f / 127.0f);
    return __builtin_fmaf(u, 127.0f, -m) == 0.0f ? u : 0.0f;
}
__device__ __forceinline__ uint32_t nearest_byte(float v, float times, float unit)
{
    const float t = v * times;
    return to_byte(__builtin_fmaf(__builtin_fmaf(-t, unit, v), times, t), 1.0f);
}
// `by`: what the row was multiplied by for the squares, `first`: their sum before that; `units`: of the maximum
template <int MODE>
__device__ __forceinline__ OfRow of_row(float squares, uint32_t most, float by, float first, int units, int width, float eps)
{
    float r = 1.0f, of_r = 1.0f;    // 1 / rms is r of_r
    if constexpr (MODE != INT8)
    {
        // (so small a sum counts for nothing beside an eps of the usual size, which times by^2 may be infinite)
        if (first < __builtin_huge_valf() && (first >= kSmall || eps >= kSmall))
            r = 1.0f / __builtin_sqrtf(first / (float)width + eps);
        else
            r = 1.0f / __builtin_sqrtf(squares / (float)width + eps * by * by), of_r = by;
    }
    if constexpr (MODE == NORM)
        return { r, r * of_r, 0.0f };
    const float m     = __uint_as_float(most);
    bool number       = m > 0x1p-119f && m < __builtin_huge_valf();    // (whose reciprocal is one too)
    float scale       = MODE == INT8 ? m / 127.0f : r * m / 127.0f;
    if (by != 1.0f || units != 0)
    {
        // (r may be large where the maximum is small, or their product no number in these units)
        const float mant = MODE == INT8 ? scale : __builtin_amdgcn_frexp_mantf(r) * __builtin_amdgcn_frexp_mantf(m) / 127.0f;
        const int exp    = MODE == INT8 ? 0 : __builtin_amdgcn_frexp_expf(r) + __builtin_amdgcn_frexp_expf(of_r) - 1 + __builtin_amdgcn_frexp_expf(m);
        scale            = __builtin_ldexpf(mant, exp - units);
        number           = number && scale != 0.0f;
    }
    if constexpr (MODE == INT8)
        return { number ? 127.0f / m : 0.0f, scale, 0.0f };
    return { number ? reciprocal_up(m) : 0.0f, scale, whole_127th(m) };
}

// Quotients of 16-bit operands are halves now and then, and go to the even number then.  t = v times the reciprocal of the maximum (over 127) lies in [2^e,
// 2^(e+1)) and is off by less than 1.5 2^(e-23); a quotient that is no half is 2^(e-20) from one at least: the maximum is b 2^j and v is a 2^i with a, b <
// 2^11 and i >= j + e - 8, so that 127 v / (b 2^j) - (k + 1/2) is a multiple of 2^(i-j-1) / b.  Rounded to a multiple of 2^(e-21) halves are halves again, and no
// other quotient crosses one.  (32-bit operands are as seldom a half as any number.)
template <typename T, int MODE>
__device__ __forceinline__ uint32_t byte_of(float v, float times)
{
    if constexpr (MODE == INT8 && sizeof(T) == 2)
        return to_byte(__uint_as_float((__float_as_uint(v * times) + 2) & ~3u), 1.0f);
    else
        return to_byte(v, times);
}

// q of one piece, eight or four bytes; at(e): its elements
template <typename T, int MODE, typename F>
__device__ __forceinline__ void store_int8(int8_t* row, int k, int pitch, const OfRow& r, F&& at)
{
    if (k >= pitch)
        return;
    uint32_t b[kPiece<T>], v[kPiece<T> / 4];
#pragma unroll
    for (int e = 0; e < kPiece<T>; e++)
        b[e] = byte_of<T, MODE>(at(e), r.times);
    if (MODE == NORM_INT8 && __builtin_expect(r.unit != 0.0f, 0))
#pragma unroll
        for (int e = 0; e < kPiece<T>; e++)
            b[e] = nearest_byte(at(e), r.times, r.unit);
#pragma unroll
    for (int i = 0; i < kPiece<T> / 4; i++)
        v[i] = r.times == 0.0f ? 0 : four_bytes(b[4 * i], b[4 * i + 1], b[4 * i + 2], b[4 * i + 3]);    // (a NaN's lowest byte may be any)
    __builtin_memcpy(row + k, v, sizeof(v));
}

// (what is taken again may cost no wave: 4096 x 8191 bf16 with residual and sum into 8 bits 61.2 us, and three waves a SIMD instead of four 71.4)
template <typename T, int MODE, int G, int P, bool WHOLE>
__global__ __launch_bounds__(G > 256 ? G : 256, G == 256 && P == 4 && kLeavesRange<T> ? 4 : 1) void norm_kernel(NormArgs a)
{
    constexpr int THREADS = G > 256 ? G : 256, ROWS = THREADS / G, V = kPiece<T>;
    constexpr bool SUM = MODE != INT8, MOST = MODE != NORM;
    __shared__ uint32_t slots[4][2 * (G > 64 ? G / 64 : 1)];
    const int lane = threadIdx.x % G, width = a.width, pitch = (int)whole16(width);

    v4i w[P];
    if constexpr (MODE != INT8)
#pragma unroll
        for (int p = 0; p < P; p++)
            w[p] = load_piece<T, WHOLE>(static_cast<const T*>(a.weight), (p * G + lane) * V, width);

    int slot = 0;
    for (int64_t m = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; m < a.rows; m += (int64_t)gridDim.x * ROWS)
    {
        float s[P][V];
        const T* row = static_cast<const T*>(a.x) + m * a.ld_x;
        v4i raw[P], more[P];
#pragma unroll
        for (int p = 0; p < P; p++)
            raw[p] = load_piece<T, WHOLE>(row, (p * G + lane) * V, width);
        if (MODE != INT8 && a.residual)
        {
            const T* from = static_cast<const T*>(a.residual) + m * a.ld_residual;
#pragma unroll
            for (int p = 0; p < P; p++)
                more[p] = load_piece<T, WHOLE>(from, (p * G + lane) * V, width);
        }
        else
#pragma unroll
            for (int p = 0; p < P; p++)
                more[p] = v4i{ 0, 0, 0, 0 };
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < V; e++)
                s[p][e] = MODE != INT8 ? piece_get<T>(raw[p], e) + piece_get<T>(more[p], e) : piece_get<T>(raw[p], e);

        float squares = 0.0f;
        uint32_t most = 0;    // (bit patterns order like the numbers, and NaN above all)
        auto weight   = [&](int p, int e) { return a.offset + piece_get<T>(w[p], e); };
        auto add      = [&](float by) {
            squares = 0.0f;
#pragma unroll
            for (int p = 0; p < P; p++)
            {
                float part = 0.0f;
#pragma unroll
                for (int e = 0; e < V; e++)
                    part = __builtin_fmaf(s[p][e] * by, s[p][e] * by, part);
                squares += part;
            }
        };
        auto product = [&](int p, int e) { return MODE == INT8 ? s[p][e] : s[p][e] * weight(p, e); };
        if constexpr (SUM)
            add(1.0f);
        if constexpr (MOST)
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int e = 0; e < V; e++)
                    most = max_u32(most, __float_as_uint(product(p, e)) & 0x7FFFFFFFu);
        over_row<G, SUM, MOST>(squares, most, slots[slot]);
        slot = 1 - slot;
        // (the sum leaves before a row is taken again)
        if (MODE != INT8 && a.sum)
#pragma unroll
            for (int p = 0; p < P; p++)
                store_piece<T, WHOLE>(static_cast<T*>(a.sum) + m * a.ld_sum, (p * G + lane) * V, width, piece_of<T>(s[p]));
        const float first = squares;
        float by          = 1.0f;
        int units         = 0;
        if (__builtin_expect(leaves_range<T, MODE>(squares, most, a.eps), 0))
        {
            by = squares_again<MODE>(squares);
            if (by != 1.0f)
            {
                uint32_t none = 0;
                add(by);
                over_row<G, true, false>(squares, none, slots[2]);
            }
            units = products_again<MODE>(squares, most);
            if (units != 0)
            {
                // (from here on the elements are the products)
                float none = 0.0f;
                most       = 0;
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int e = 0; e < V; e++)
                    {
                        s[p][e] = product_in(s[p][e], MODE == INT8 ? 1.0f : weight(p, e), units);
                        most    = max_u32(most, __float_as_uint(s[p][e]) & 0x7FFFFFFFu);
                    }
                over_row<G, false, true>(none, most, slots[3]);
            }
            if constexpr (MODE == NORM)
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int e = 0; e < V; e++)
                        s[p][e] *= by;
        }
        const OfRow r = of_row<MODE>(squares, most, by, first, units, width, a.eps);
        if (a.of_row && lane == 0)
            a.of_row[m] = r.stored;
        if constexpr (MODE == NORM)
#pragma unroll
            for (int p = 0; p < P; p++)
            {
                float y[V];
#pragma unroll
                for (int e = 0; e < V; e++)
                    y[e] = s[p][e] * r.times * weight(p, e);
                store_piece<T, WHOLE>(static_cast<T*>(a.out) + m * a.ld_out, (p * G + lane) * V, width, piece_of<T>(y));
            }
        else
        {
            int8_t* to = static_cast<int8_t*>(a.out) + m * a.ld_out;
            if (MODE == NORM_INT8 && __builtin_expect(units != 0, 0))
            {
#pragma unroll
                for (int p = 0; p < P; p++)
                    store_int8<T, MODE>(to, (p * G + lane) * V, pitch, r, [&](int e) { return s[p][e]; });
            }
            else
#pragma unroll
                for (int p = 0; p < P; p++)
                    store_int8<T, MODE>(to, (p * G + lane) * V, pitch, r, [&](int e) { return product(p, e); });
        }
    }
}

// Rows that no workgroup's registers hold: read once for the sum, again if it left the range, and once more for the results (1024 x 40000 bf16 with residual and sum 86
// us, 3.8 TB/s of the bytes that one reading would take).  Results may take the place of what
// is read, so here a piece is made of its own elements alone.
template <typename T, int MODE, bool WHOLE>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs a)
{
    constexpr int G = 1024, V = kPiece<T>;
    constexpr bool SUM = MODE != INT8, MOST = MODE != NORM;
    __shared__ uint32_t slots[4][2 * (G / 64)];
    const int width = a.width, pitch = (int)whole16(width);
    int slot = 0;
    for (int64_t m = blockIdx.x; m < a.rows; m += gridDim.x)
    {
        const T *row = static_cast<const T*>(a.x) + m * a.ld_x, *from = static_cast<const T*>(a.residual) + (a.residual ? m * a.ld_residual : 0);
        auto piece = [&](int k, float* s) {
            const v4i raw = load_piece_alone<T, WHOLE>(row, k, width);
            v4i more      = { 0, 0, 0, 0 };
            if (MODE != INT8 && a.residual)
                more = load_piece_alone<T, WHOLE>(from, k, width);
#pragma unroll
            for (int e = 0; e < V; e++)
                s[e] = MODE != INT8 ? piece_get<T>(raw, e) + piece_get<T>(more, e) : piece_get<T>(raw, e);
        };
        auto weights = [&](int k, float* w) {
            v4i v = { 0, 0, 0, 0 };
            if constexpr (MODE != INT8)
                v = load_piece<T, WHOLE>(static_cast<const T*>(a.weight), k, width);
#pragma unroll
            for (int e = 0; e < V; e++)
                w[e] = MODE != INT8 ? a.offset + piece_get<T>(v, e) : 1.0f;
        };
        float squares = 0.0f;
        uint32_t most = 0;
        // (the squares of the row times `by`, and the products in `units`; without units as they are)
        auto look = [&](auto with_sum, auto with_most, float by, int units) {
            for (int k = (int)threadIdx.x * V; k < width; k += G * V)
            {
                float s[V], w[V];
                piece(k, s);
                if constexpr (decltype(with_most)::value)
                    weights(k, w);
                float part = 0.0f;
#pragma unroll
                for (int e = 0; e < V; e++)
                {
                    if constexpr (decltype(with_sum)::value)
                        part = __builtin_fmaf(s[e] * by, s[e] * by, part);
                    if constexpr (decltype(with_most)::value)
                        most = max_u32(most, __float_as_uint(units == 0 ? s[e] * w[e] : product_in(s[e], w[e], units)) & 0x7FFFFFFFu);
                }
                squares += part;
            }
        };
        look(std::bool_constant<SUM>(), std::bool_constant<MOST>(), 1.0f, 0);
        over_row<G, SUM, MOST>(squares, most, slots[slot]);
        slot              = 1 - slot;
        const float first = squares;
        float by          = 1.0f;
        int units         = 0;
        if (__builtin_expect(leaves_range<T, MODE>(squares, most, a.eps), 0))
        {
            by = squares_again<MODE>(squares);
            if (by != 1.0f)
            {
                uint32_t none = 0;
                squares       = 0.0f;
                look(std::true_type(), std::false_type(), by, 0);
                over_row<G, true, false>(squares, none, slots[2]);
            }
            units = products_again<MODE>(squares, most);
            if (units != 0)
            {
                float none = 0.0f;
                most       = 0;
                look(std::false_type(), std::true_type(), 1.0f, units);
                over_row<G, false, true>(none, most, slots[3]);
            }
        }
        const OfRow r = of_row<MODE>(squares, most, by, first, units, width, a.eps);
        if (a.of_row && threadIdx.x == 0)
            a.of_row[m] = r.stored;
        for (int k = (int)threadIdx.x * V; k < (MODE == NORM ? width : pitch); k += G * V)
        {
            float s[V], w[V];
            piece(k, s);
            weights(k, w);
            if (MODE != INT8 && a.sum)
                store_piece<T, WHOLE>(static_cast<T*>(a.sum) + m * a.ld_sum, k, width, piece_of<T>(s));
            if constexpr (MODE == NORM)
            {
                float y[V];
#pragma unroll
                for (int e = 0; e < V; e++)
                    y[e] = s[e] * by * r.times * w[e];
                store_piece<T, WHOLE>(static_cast<T*>(a.out) + m * a.ld_out, k, width, piece_of<T>(y));
            }
            else
            {
                int8_t* to = static_cast<int8_t*>(a.out) + m * a.ld_out;
                if (__builtin_expect(units != 0, 0))
                    store_int8<T, MODE>(to, k, pitch, r, [&](int e) { return product_in(s[e], w[e], units); });
                else
                    store_int8<T, MODE>(to, k, pitch, r, [&](int e) { return s[e] * w[e]; });
            }
        }
    }
}

// x = scale q, rounded; bound by memory.  2^shift lanes have a row, the pieces of a lane eight or four bytes in and 16 out.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void dequantize_kernel(NormArgs a, int shift)
{
    constexpr int V = kPiece<T>;
    const int per   = 1 << shift, lane = threadIdx.x & (per - 1);
    const int64_t step = (int64_t)gridDim.x * (256 >> shift);
    for (int64_t m = (int64_t)blockIdx.x * (256 >> shift) + (threadIdx.x >> shift); m < a.rows; m += step)
    {
        const int8_t* row = static_cast<const int8_t*>(a.x) + m * a.ld_x;
        T* out            = static_cast<T*>(a.out) + m * a.ld_out;
        const float scale = a.of_row[m];
#pragma unroll 4
        for (int k = lane * V; k < a.width; k += per * V)
        {
            int8_t q[V];
            __builtin_memcpy(q, row + k, V);    // (rows hold whole 16 bytes)
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e++)
                v[e] = scale * (float)q[e];
            store_piece<T, WHOLE>(out, k, a.width, piece_of<T>(v));
        }
    }
}

template <typename F>
void for_type(int32_t dtype, F&& f)
{
    if (dtype == TMI_FP16)
        f(_Float16{});
    else if (dtype == TMI_BF16)
        f(bf16_t{});
    else
        f(float{});
}
template <int N>
constexpr std::integral_constant<int, N> number_of{};

// a workgroup of 1024 has room for 16 numbers a lane beside what it read them from
template <typename T>
constexpr int kMostPieces = 16 * 1024 / kPiece<T>;

// lanes of a row and pieces of a lane, from the pieces that a row has.  (us with lanes of a row for 16 or 64 pieces at least: 262144 x 64 bf16 21.0, with 8 lanes 13.5;
// 44157 x 168 16.2, with 32 9.3; 16384 x 1088 with residual and sum, 256 lanes of a piece 34.3, 64 of three 29.3, but one row of 1536 2.9 and 3.1)
template <typename T, int MODE, bool WHOLE>
void launch_typed(hipStream_t st, const NormArgs& a)
{
    const int64_t pieces = ((MODE == NORM ? a.width : whole16(a.width)) + kPiece<T> - 1) / kPiece<T>;
    auto go = [&](auto G_tag, auto P_tag) {
        constexpr int G = decltype(G_tag)::value, P = decltype(P_tag)::value, THREADS = G > 256 ? G : 256, ROWS = THREADS / G;
        // (short rows: as many workgroups as there are at once, which keep the weights; longer ones a workgroup each.  us 131072 x 128 12.1 and 12.8, 44157 x 168
        // 9.4 and 10.3, 16384 x 4096 into 8 bits 38.4 and 36.4, 8192 x 4096 with a residual 51.0 and 46.7)
        const int64_t groups = (a.rows + ROWS - 1) / ROWS, most = G <= 32 ? 2048 : 1 << 20;
        norm_kernel<T, MODE, G, P, WHOLE><<<(int)(groups < most ? groups : most), THREADS, 0, st>>>(a);
    };
    if (pieces <= 8)
        go(number_of<8>, number_of<1>);
    else if (pieces <= 16)
        go(number_of<16>, number_of<1>);
    else if (pieces <= 32)
        go(number_of<32>, number_of<1>);
    else if (pieces <= 64)
        go(number_of<64>, number_of<1>);
    else if (pieces <= 128)
        go(number_of<64>, number_of<2>);
    else if (pieces <= 192 && a.rows > 256)
        go(number_of<64>, number_of<3>);
    else if (pieces <= 256)
        go(number_of<256>, number_of<1>);
    else if (pieces <= 512)
        go(number_of<256>, number_of<2>);
    else if (pieces <= 1024)
        go(number_of<256>, number_of<4>);
    else if (pieces <= kMostPieces<T>)
        go(number_of<1024>, number_of<kMostPieces<T> / 1024>);
    else
        norm_long_kernel<T, MODE, WHOLE><<<(int)(a.rows < (1 << 20) ? a.rows : 1 << 20), 1024, 0, st>>>(a);
}

}    // namespace

const char* launch_rms_norm(hipStream_t st, const tmi_rms_norm_desc_t& d, const void* x, const void* residual, const void* weight, void* sum, void* y,
                            float* of_row, bool int8, int64_t ld_y)
{
    const NormArgs a{ x, residual, weight, sum, y, of_row, d.ld_x, d.ld_residual, d.ld_sum, ld_y, d.rows, d.width, d.eps, d.weight_offset };
    for_type(d.dtype, [&](auto type) {
        using T          = decltype(type);
        const bool whole = whole_rows<T>(x, d.width, d.ld_x) && whole_rows<T>(weight, d.width, d.width) &&
                           (!residual || whole_rows<T>(residual, d.width, d.ld_residual)) && (!sum || whole_rows<T>(sum, d.width, d.ld_sum)) &&
                           (int8 || whole_rows<T>(y, d.width, ld_y));
        if (int8)
            whole ? launch_typed<T, NORM_INT8, true>(st, a) : launch_typed<T, NORM_INT8, false>(st, a);
        else
            whole ? launch_typed<T, NORM, true>(st, a) : launch_typed<T, NORM, false>(st, a);
    });
    return int8 ? "rms_norm_int8" : "rms_norm";
}

const char* launch_quantize_int8(hipStream_t st, int32_t dtype, int32_t rows, int32_t width, const void* x, int64_t ld_x, void* q, int64_t ld_q,
                                 float* scales)
{
    const NormArgs a{ x, nullptr, nullptr, nullptr, q, scales, ld_x, 0, 0, ld_q, rows, width, 0.0f, 0.0f };
    for_type(dtype, [&](auto type) {
        using T = decltype(type);
        whole_rows<T>(x, width, ld_x) ? launch_typed<T, INT8, true>(st, a) : launch_typed<T, INT8, false>(st, a);
    });
    return "quantize_int8";
}

const char* launch_dequantize_int8(hipStream_t st, int32_t dtype, int32_t rows, int32_t width, const void* q, int64_t ld_q, const float* scales, void* x,
                                   int64_t ld_x)
{
    const NormArgs a{ q, nullptr, nullptr, nullptr, x, const_cast<float*>(scales), ld_q, 0, 0, ld_x, rows, width, 0.0f, 0.0f };
    for_type(dtype, [&](auto type) {
        using T   = decltype(type);
        int shift = 4;
        while (shift < 8 && (kPiece<T> << shift) < width)
            shift++;
        const int64_t groups = ((int64_t)rows + (256 >> shift) - 1) / (256 >> shift);
        const int grid       = (int)(groups < (1 << 20) ? groups : 1 << 20);    // (16384 x 4096: 35.9 us, with 2048 of them 37.4)
        if (whole_rows<T>(x, width, ld_x))
            dequantize_kernel<T, true><<<grid, 256, 0, st>>>(a, shift);
        else
            dequantize_kernel<T, false><<<grid, 256, 0, st>>>(a, shift);
    });
    return "dequantize_int8";
}

}    // namespace tmi
