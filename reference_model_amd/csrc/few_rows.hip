// Products of a few rows with large weights, and the gated block on them:
//
//   y[m][n] = sum_k x[m][k] w[n][k]                h[m][f] = act(sum_k x[m][k] gate[f][k]) * (sum_k x[m][k] up[f][k])
//
// w in 4 bits with a scale for each group of columns (y and h), or gate and up in 16 bits (h).  With up to 64 rows the weights' bytes are all
// that counts: each is read once, by one wave, straight into the registers from which the matrix instruction takes it.
//
// 16x16x32 instructions take the rows of x as first operand and the weights as second: a single row wastes 15/16 of the matrix cores, which at 512
// weights an instruction still run four times as many weights as HBM delivers, and any other number of rows up to 16 costs the same.  4-bit
// weights become 16-bit integers (exact; 8 or 13 instructions for eight), their products are summed in 32 bits, and the sum over a group is
// multiplied by its scale: no weight is rounded, and an infinite or NaN x does to a row what it does in the formula.  (The sum of a group comes before
// its scale: bf16 x from 5e36 on may overflow in it where x times the scaled weights would not, and given scales that are infinite meet the sum.)
//
// Two kernels share this.  In both, what the waves of a workgroup have summed meets in LDS in the order of the waves, so equal calls give equal bits.
//
// few_rows_kernel: a workgroup of up to eight waves has one tile of 16 weight rows (of both matrices, if gated), a wave every eighth tile of 128
// columns of it; weights and x go straight to registers, the loads of U column tiles at once, with nothing to wait for in between.  Its
// calls are short: 2.4 us for 512 x 512 in 4 bits, 3.8 for 4096 x 4096.
//
// int4_stream_kernel: for large matrices and more rows.  A workgroup goes through blocks of WN tiles of 16 weight rows; WK of its waves share
// a tile, each with every WK-th tile of 128 columns.  A wave's weights go round in U sets of registers, the loads of the next U column tiles in
// flight, from one block of rows into the next and past the barriers (the other kernel's waves load, wait and compute in turn: 2 x 32768 x 8192 in
// bf16 69 us there, 55 here, one row: 5.0 TB/s).  x lies in LDS, all of its columns or a part of them at a time: read by each wave from L2 its rows are up to
// eight times the weights' bytes (16 rows, 16384 x 4096: 18.9 us there, 11.8 here).  Where x takes less than half of the LDS two workgroups of eight
// waves share a CU, otherwise one of sixteen has it.
#include "tmi_ffn.h"

namespace tmi
{
namespace
{

struct RowsArgs
{
    const uint16_t* x;
    const uint8_t* w[2];
    uint16_t *out, *pre_gate, *pre_up;
    int64_t ldx, ldw, ldo;    // elements
    int64_t tiles;            // 4 bits: tiles of a matrix
    int32_t rows, n, k;
    int32_t tiles_n, tiles_k;
    int32_t act;
    // few_rows_kernel: where a row's column tiles are shared by workgroups, `splits` of them, their sums as store_rows takes them from one workgroup's waves
    int32_t splits;
    int32_t per_split;        // column tiles
    float* sums;              // [row tile of x][weight row tile][split]
    // int4_stream_kernel
    int32_t n_blocks;
    int32_t wk;               // waves of a tile
    int32_t turns;            // of U steps of wk column tiles, for all of K
    int32_t part;             // turns whose columns of x are in LDS at a time
    int32_t stride;           // rows of x that a 16-byte piece of LDS columns has room for: 1, 2, 4, 8 or 16 MT
    int32_t red_at;           // byte of LDS where the waves' sums meet; 0: where x lies, which is then read again for every block
};

template <int PER>
using scales_t = std::conditional_t<PER == 4, uint64_t, std::conditional_t<PER == 2, uint32_t, uint16_t>>;

// The sums of `parts` waves at red[part][stream][row tile][4][lane], from the first of them on, added, and what is made of them stored: result o of
// MT * 256 of the weight rows from n0 and the rows of x from row0.
template <typename T, bool DENSE, int MT, bool GATED>
__device__ __forceinline__ void store_rows(const RowsArgs& a, const float* red, int parts, int o, int64_t n0, int64_t row0)
{
    constexpr int S = GATED ? 2 : 1;
    const int mt = o >> 8, ln = o & 63;
    const int64_t n = n0 + (ln & 15), m = row0 + 16 * mt + (ln >> 4) * 4 + (o >> 6 & 3);
    if (n >= a.n || m >= a.rows)
        return;
    constexpr float unit = DENSE ? 1.0f : 1.0f / kInt4Unit<T>;
    float v[S];
#pragma unroll
    for (int s = 0; s < S; s++)
    {
        v[s] = 0.0f;
        for (int p = 0; p < parts; p++)
            v[s] += red[((p * S + s) * MT + mt) * 256 + (o & 255)];
        v[s] *= unit;
    }
    const int64_t at = m * a.ldo + n;
    if constexpr (GATED)
        for_act(a.act, [&](auto ACT) { a.out[at] = to_bits16<T>(act_value<decltype(ACT)::value>(v[0]) * v[S - 1]); });
    else
        a.out[at] = to_bits16<T>(v[0]);
    if constexpr (GATED && DENSE)
        if (a.pre_gate)
            a.pre_gate[at] = to_bits16<T>(v[0]), a.pre_up[at] = to_bits16<T>(v[S - 1]);
}

constexpr int kShortWaves = 8;

// PER: groups of a 4-bit tile, 0 = 16-bit weights; MT: tiles of 16 rows of x; U: column tiles whose loads a wave has in flight together;
// ODD: rows of x or of 16-bit weights begin at odd elements; SHARED: workgroups may share a row's columns (16 bits: 0.2 us a call where they do not)
template <typename T, int PER, int MT, bool GATED, int U, bool ODD, bool SHARED>
__global__ __launch_bounds__(64 * kShortWaves, PER || SHARED ? 1 : 4) void few_rows_kernel(RowsArgs a)
{
    constexpr bool DENSE = PER == 0;
    constexpr int S      = GATED ? 2 : 1;    // streams of weights: gate and up
    constexpr int WV     = DENSE ? 4 : 1;    // 16-byte loads of a lane, stream and column tile
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    float* red = reinterpret_cast<float*>(lds);

    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int tn       = blockIdx.x;
    const int64_t row0 = (int64_t)blockIdx.y * (16 * MT);
    const int full     = a.k / kInt4Cols;    // whole column tiles

    const uint16_t* xrow[MT];
    bool live[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
    {
        const int64_t m = row0 + 16 * mt + r;
        live[mt]        = m < a.rows;
        xrow[mt]        = a.x + (live[mt] ? m : 0) * a.ldx;
    }
    const uint8_t *wbase[S], *sbase[S];    // 4 bits: the row tile's first column tile and its scales; 16 bits: the lane's row
#pragma unroll
    for (int s = 0; s < S; s++)
    {
        if constexpr (DENSE)
        {
            int64_t n = (int64_t)tn * 16 + r;
            n         = n < a.n ? n : a.n - 1;
            wbase[s]  = a.w[s] + n * a.ldw * 2;
        }
        else
        {
            const int64_t t = (int64_t)tn * a.tiles_k;
            wbase[s]        = a.w[s] + t * kInt4TileBytes;
            sbase[s]        = a.w[s] + int4_scale_at(a.tiles, t, PER);
        }
    }
    v4f acc[S][MT];
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
            acc[s][mt] = v4f{ 0.0f, 0.0f, 0.0f, 0.0f };

    struct Tile
    {
        v4i x[MT][4];
        v4i w[S][WV];
        scales_t<PER> scale[S];
        int x_next[MT][ODD ? 4 : 1], w_next[S][ODD && DENSE ? WV : 1];
    };
    Halves xhalf[MT], whalf[S];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
        xhalf[mt] = halves_of(reinterpret_cast<const uint8_t*>(xrow[mt]));
#pragma unroll
    for (int s = 0; s < S; s++)
        whalf[s] = halves_of(wbase[s]);
    // Rows of 16-bit weights may lie a power of two apart: workgroups that begin at different columns meet on different channels of the
    // memory.  us of one row with 2 x 32768 x 8192: 230 all from the first column, 178 so.  (In 4 bits a tile of rows lies in one piece.)
    const int turn = DENSE && full && !SHARED ? (int)((blockIdx.x * 5u) % (uint32_t)full) : 0;
    auto turned    = [&](int kt) { return DENSE ? (kt + turn < full ? kt + turn : kt + turn - full) : kt; };
    // TAIL: the column tile that K ends in
    auto fetch_w = [&](Tile& t, int kt, auto TAIL) {
#pragma unroll
        for (int s = 0; s < S; s++)
        {
            if constexpr (DENSE)
            {
                const uint16_t* row = ODD ? whalf[s].row() : reinterpret_cast<const uint16_t*>(wbase[s]);
#pragma unroll
                for (int j = 0; j < 4; j++)
                {
                    const int64_t k = (int64_t)kt * 128 + 32 * j + 8 * q;
                    if constexpr (decltype(TAIL)::value)
                        t.w[s][j] = settle8(load8_raw(row, k, a.k), k, a.k, true);
                    else if constexpr (ODD)
                    {
                        t.w[s][j]      = load16(whalf[s].base + 2 * k);
                        t.w_next[s][j] = whalf[s].next(2 * k);
                    }
                    else
                        t.w[s][j] = load16(reinterpret_cast<const uint8_t*>(row + k));
                }
            }
            else
            {
                t.w[s][0]  = reinterpret_cast<const v4i*>(wbase[s] + (int64_t)kt * kInt4TileBytes)[lane];
                t.scale[s] = reinterpret_cast<const scales_t<PER>*>(sbase[s] + (int64_t)kt * (kInt4Rows * 2 * PER))[r];
            }
        }
    };
    auto fetch_x = [&](Tile& t, int kt, auto TAIL) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                const int64_t k = (int64_t)kt * 128 + 32 * j + 8 * q;
                t.x[mt][j]      = v4i{ 0, 0, 0, 0 };
                if constexpr (decltype(TAIL)::value)
                    t.x[mt][j] = settle8(load8_raw(ODD ? xhalf[mt].row() : xrow[mt], k, a.k), k, a.k, live[mt]);
                else if constexpr (ODD)
                {
                    t.x_next[mt][j] = 0;
                    if (live[mt])
                    {
                        t.x[mt][j]      = load16(xhalf[mt].base + 2 * k);
                        t.x_next[mt][j] = xhalf[mt].next(2 * k);
                    }
                }
                else if (live[mt])
                    t.x[mt][j] = load16(reinterpret_cast<const uint8_t*>(xrow[mt] + k));
            }
    };
    auto join = [&](Tile& t) {
        if constexpr (ODD)
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
                    t.x[mt][j] = joined(t.x[mt][j], t.x_next[mt][j], xhalf[mt].shift);
                if constexpr (DENSE)
#pragma unroll
                    for (int s = 0; s < S; s++)
                        t.w[s][j] = joined(t.w[s][j], t.w_next[s][j], whalf[s].shift);
            }
    };
    auto multiply = [&](const Tile& t) {
#pragma unroll
        for (int s = 0; s < S; s++)
            if constexpr (DENSE)
            {
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
                        acc[s][mt] = mma16<T>(t.x[mt][j], t.w[s][j], acc[s][mt]);
            }
            else
            {
#pragma unroll
                for (int g = 0; g < PER; g++)
                {
                    v4f d[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
                        d[mt] = v4f{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
                    for (int j = g * 4 / PER; j < (g + 1) * 4 / PER; j++)
                    {
                        const v4i w = int4_unpack<T>((uint32_t)t.w[s][0][j]);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
                            d[mt] = mma16<T>(t.x[mt][j], w, d[mt]);
                    }
                    const float scale = from_bits16<T>((uint16_t)(t.scale[s] >> (16 * g)));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            acc[s][mt][i] = __builtin_fmaf(scale, d[mt][i], acc[s][mt][i]);
                }
            }
    };

    const int first = SHARED ? blockIdx.z * a.per_split : 0, behind = SHARED && first + a.per_split < a.tiles_k ? first + a.per_split : a.tiles_k;
    const int whole = behind < full ? behind : full;
    for (int k0 = first + wave; k0 < whole; k0 += U * waves)
    {
        Tile t[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k0 + u * waves < whole)
                fetch_w(t[u], turned(k0 + u * waves), std::false_type());
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k0 + u * waves < whole)
                fetch_x(t[u], turned(k0 + u * waves), std::false_type());
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k0 + u * waves < whole)
            {
                join(t[u]);
                multiply(t[u]);
            }
    }
    if (whole < behind && (whole - first) % waves == wave)
    {
        Tile t;
        fetch_w(t, full, std::true_type());
        fetch_x(t, full, std::true_type());
        multiply(t);
    }

#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                red[((wave * S + s) * MT + mt) * 256 + i * 64 + lane] = acc[s][mt][i];
    __syncthreads();
    if (!SHARED || a.splits == 1)
    {
        for (int o = threadIdx.x; o < MT * 256; o += blockDim.x)
            store_rows<T, DENSE, MT, GATED>(a, red, waves, o, (int64_t)tn * 16, row0);
        return;
    }
    float* part = a.sums + (((int64_t)blockIdx.y * a.tiles_n + tn) * a.splits + blockIdx.z) * (S * MT * 256);
    for (int o = threadIdx.x; o < S * MT * 256; o += blockDim.x)
    {
        float v = 0.0f;
        for (int p = 0; p < waves; p++)
            v += red[p * (S * MT * 256) + o];
        part[o] = v;
    }
}

// results of column tiles that workgroups shared
template <typename T, bool DENSE, int MT, bool GATED>
__global__ __launch_bounds__(256) void few_rows_join_kernel(RowsArgs a)
{
    const float* part = a.sums + ((int64_t)blockIdx.y * a.tiles_n + blockIdx.x) * a.splits * ((GATED ? 2 : 1) * MT * 256);
    for (int o = threadIdx.x; o < MT * 256; o += 256)
        store_rows<T, DENSE, MT, GATED>(a, part, a.splits, o, (int64_t)blockIdx.x * 16, (int64_t)blockIdx.y * (16 * MT));
}

constexpr int kAhead = 4;                              // pieces of x that a lane asks for at once
constexpr int kLds = 156 * 1024, kLdsHalf = 78 * 1024;    // for one workgroup of a CU, and for two

// MT: tiles of 16 rows of x; PER: groups of a tile; U: column tiles in flight
template <typename T, int PER, int MT, bool GATED, int U>
__global__ __launch_bounds__(1024) void int4_stream_kernel(RowsArgs a)
{
    constexpr int S = GATED ? 2 : 1;    // streams of weights: gate and up
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];

    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
    const int wk = wave & (a.wk - 1), wn = wave / a.wk, WN = waves / a.wk;
    const int64_t row0 = (int64_t)blockIdx.y * (16 * MT);
    const int here     = a.rows - row0 < 16 * MT ? (int)(a.rows - row0) : 16 * MT;    // rows of x

    // ---- weights ----------------------------------------------------------------------------------------------------------------
    v4i w[U][S];
    scales_t<PER> scale[U][S];
    // Step `step` (of U * turns) of block nb into set u.  Past the last tile nothing is multiplied or stored: all lanes then take the same 16 bytes, so that
    // as many loads are on their way as always and none of them costs anything.
    auto fetch_w = [&](int u, int nb, int step) {
        const int tn = nb * WN + wn, kt = step * a.wk + wk;
        const bool live = tn < a.tiles_n && kt < a.tiles_k;
        const int64_t t = live ? (int64_t)tn * a.tiles_k + kt : 0;
        const int l     = live ? lane : 0;
#pragma unroll
        for (int s = 0; s < S; s++)
        {
            w[u][s]     = reinterpret_cast<const v4i*>(a.w[s] + t * kInt4TileBytes)[l];
            scale[u][s] = reinterpret_cast<const scales_t<PER>*>(a.w[s] + int4_scale_at(a.tiles, t, PER))[l & 15];
        }
    };

    // ---- x: piece c of 8 columns and row m lie at unit c * stride + m; from 16 rows on with the low four bits of m exchanged by c ------------
    auto unit_of = [&](int c, int m) { return c * a.stride + (a.stride < 16 ? m : m ^ (c & 15)); };
    const int tiles_x = a.part * U * a.wk;    // column tiles in LDS at a time
    auto load_x       = [&](int from) {            // from `from` on
        const int pieces = (tiles_x < a.tiles_k - from ? tiles_x : a.tiles_k - from) * 16;
        const int apart  = a.stride < waves ? a.stride : waves, lanes = 64 * (waves / apart);    // waves on rows of their own, the others beside them
#pragma unroll 1
        for (int m = wave & (apart - 1); m < here; m += apart)
        {
            const uint16_t* row = a.x + (row0 + m) * a.ldx + (int64_t)from * 128;
            const int end       = a.k - from * 128;
#pragma unroll 1
            for (int c0 = wave / apart * 64 + lane; c0 < pieces; c0 += kAhead * lanes)
            {
                v4i v[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; i++)
                    v[i] = load8_raw(row, 8 * (c0 + i * lanes), end);
#pragma unroll
                for (int i = 0; i < kAhead; i++)
                    if (c0 + i * lanes < pieces)
                        *reinterpret_cast<v4i*>(lds + unit_of(c0 + i * lanes, m) * 16) = settle8(v[i], 8 * (c0 + i * lanes), end, true);
            }
        }
    };

    v4f acc[S][MT];
    auto clear = [&]() {
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
                acc[s][mt] = v4f{ 0.0f, 0.0f, 0.0f, 0.0f };
    };
    // the column tile that lies in LDS as tile `at` by the weights of set u; with four row tiles one stream after the other, as the registers
    // hold no sums of a group for both
    auto multiply = [&](int u, int at) {
        // (rows past the last one repeat it, or are whatever lies there: they are not stored)
        const int m      = a.stride < 16 ? (r < a.stride ? r : a.stride - 1) : r;
        constexpr int ST = MT == 4 ? 1 : S;
#pragma unroll
        for (int s0 = 0; s0 < S; s0 += ST)
#pragma unroll
            for (int g = 0; g < PER; g++)
            {
                v4f d[ST][MT];
#pragma unroll
                for (int s = 0; s < ST; s++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
                        d[s][mt] = v4f{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
                for (int j = g * 4 / PER; j < (g + 1) * 4 / PER; j++)
                {
                    v4i x[MT];
                    const int unit = unit_of(at * 16 + 4 * j + q, m);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
                        x[mt] = *reinterpret_cast<const v4i*>(lds + (unit + 16 * mt) * 16);
#pragma unroll
                    for (int s = 0; s < ST; s++)
                    {
                        const v4i ws = int4_unpack<T>((uint32_t)w[u][s0 + s][j]);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
                            d[s][mt] = mma16<T>(x[mt], ws, d[s][mt]);
                    }
                }
#pragma unroll
                for (int s = 0; s < ST; s++)
                {
                    const float sc = from_bits16<T>((uint16_t)(scale[u][s0 + s] >> (16 * g)));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            acc[s0 + s][mt][i] = __builtin_fmaf(sc, d[s][mt][i], acc[s0 + s][mt][i]);
                }
                if (MT == 4)
                    __builtin_amdgcn_sched_barrier(0);
            }
    };
    // The waves' sums meet in LDS, [wave][stream][row tile][4][lane]
    auto finish = [&](int nb) {
        float* red = reinterpret_cast<float*>(lds + a.red_at);
        if (!a.red_at)
            __syncthreads();    // x is read
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    red[((wave * S + s) * MT + mt) * 256 + i * 64 + lane] = acc[s][mt][i];
        __syncthreads();
#pragma unroll 1
        for (int o = tid; o < WN * MT * 256; o += blockDim.x)
        {
            const int t = o / (MT * 256);
            store_rows<T, false, MT, GATED>(a, red + (size_t)t * a.wk * S * MT * 256, a.wk, o - t * MT * 256, ((int64_t)nb * WN + t) * 16, row0);
        }
        if (nb + (int)gridDim.x < a.n_blocks)
            __syncthreads();    // the sums are read
    };

    // (no turns: sums of nothing)
    if (a.turns > 0)
#pragma unroll
        for (int u = 0; u < U; u++)
            fetch_w(u, blockIdx.x, u);
#pragma unroll 1
    for (int nb = blockIdx.x; nb < a.n_blocks; nb += gridDim.x)
    {
        clear();
#pragma unroll 1
        for (int t0 = 0; t0 < a.turns; t0 += a.part)
        {
            if (!a.red_at || nb == (int)blockIdx.x)
            {
                if (t0)
                    __syncthreads();    // x is read
                load_x(t0 * U * a.wk);
                __syncthreads();
            }
            const int t1 = t0 + a.part < a.turns ? t0 + a.part : a.turns;
#pragma unroll 1
            for (int t = t0; t < t1; t++)
            {
                const bool last = t + 1 == a.turns;
#pragma unroll
                for (int u = 0; u < U; u++)
                {
                    const int kt = (t * U + u) * a.wk + wk;
                    if (kt < a.tiles_k)
                        multiply(u, kt - t0 * U * a.wk);
                    __builtin_amdgcn_sched_barrier(0);
                    fetch_w(u, last ? nb + gridDim.x : nb, last ? u : (t + 1) * U + u);
                }
            }
        }
        finish(nb);
    }
}

template <int PER, int MT, bool GATED>
constexpr int kInFlight = GATED && MT > 1 ? 2 : 4;

// What a call costs by its parts' rates, in us: the bytes of weights and x that the busiest CU takes in at 64 a clock, those that L2 gives out at 10 TB/s
// and HBM at 6, and the vector instructions of its four SIMDs: a weight tile takes 320 clocks to unpack in bf16 and 250 in fp16, 24 for each group's
// scale and 40 of products for each row tile, and a turn's empty places a fifth of that; 8 % of what does not bound, 1.5 us for every reading of x and 1
// for every block.  Over 13 sizes and all their plans (8 and 16 waves, every split, 1, 2 and 4 row tiles) its choice is within 1 % of the best on average, 3.4 % at most.
template <typename T, int PER, int MT, bool GATED>
double plan(RowsArgs& a, int& waves)
{
    constexpr int S = GATED ? 2 : 1, U = kInFlight<PER, MT, GATED>;
    const double chunks = (a.rows + 16 * MT - 1) / (16 * MT);
    const int m         = a.rows < 16 * MT ? a.rows : 16 * MT;
    double least        = -1;
    RowsArgs best       = a;
    for (int many = 8; many <= 16; many += 8)
        for (int wk = many; wk >= 1; wk /= 2)
        {
            if (wk > 1 && wk > a.tiles_k)
                continue;
            RowsArgs t = a;
            t.wk = wk, t.turns = (a.tiles_k + wk * U - 1) / (wk * U);
            t.stride               = m > 8 ? 16 * MT : m > 4 ? 8 : m > 2 ? 4 : m;
            const int64_t turn     = (int64_t)t.stride * 256 * wk * U, red = (int64_t)many * S * MT * 1024, most = many == 8 ? kLdsHalf : kLds;
            const int64_t x_size   = (int64_t)t.stride * 256 * a.tiles_k;
            const bool resident    = x_size + red <= most;
            t.part                 = (int32_t)(resident ? t.turns : most / turn < t.turns ? most / turn : t.turns);
            t.red_at               = resident ? (int32_t)(x_size > 0 ? x_size : 16) : 0;
            if (t.turns > 0 && t.part == 0)
                continue;
            const int wn = many / wk, slots = many == 8 ? 512 : 256;
            t.n_blocks   = (a.tiles_n + wn - 1) / wn;
            const double wgs = t.n_blocks * chunks, rounds = wgs > slots ? (double)(int64_t)((wgs + slots - 1) / slots) : 1;
            const double busiest = (double)(int64_t)((wgs + 255) / 256);    // blocks of the CU that has most
            const double shared  = wgs > 256 && many == 8 ? 2 : 1;          // workgroups of a CU
            const double w_bytes = (double)wn * S * a.tiles_k * (1024 + 32 * PER), x_bytes = (double)m * a.k * 2;
            const double reads   = resident ? 1 : rounds * ((t.turns + t.part - 1) / (t.part ? t.part : 1));
            const double cu      = (busiest * w_bytes + (resident ? shared : busiest) * x_bytes) / 147e3;
            const double l2      = (wgs * w_bytes + (resident && wgs > slots ? slots : wgs) * x_bytes) / 10e6;
            const double hbm     = (double)t.n_blocks * w_bytes / 6e6;
            const double clocks  = (__is_same(T, bf16_t) ? 320 : 250) + (24 * PER + 40) * MT;
            const double vector  = busiest * wn * S * (0.8 * a.tiles_k + 0.2 * t.turns * U * wk) / 4 * clocks / 2100;
            double us            = cu > l2 ? cu : l2;
            us                   = us > hbm ? us : hbm;
            us                   = us > vector ? us : vector;
            us += 0.08 * (cu + l2 + hbm + vector - us) + 1.5 * reads / shared + rounds;
            if (least < 0 || us < least)
                least = us, best = t, waves = many;
        }
    a = best;
    return least;
}

template <typename T, int PER, int MT, bool GATED>
bool launch_stream(hipStream_t st, const RowsArgs& a, int waves)
{
    constexpr int S = GATED ? 2 : 1, U = kInFlight<PER, MT, GATED>;
    const size_t red = (size_t)waves * S * MT * 1024, x_bytes = (size_t)a.stride * 256 * a.wk * U * a.part;
    const size_t lds = a.red_at ? a.red_at + red : x_bytes > red ? x_bytes : red;
    if (!ensure_dynamic_lds<int4_stream_kernel<T, PER, MT, GATED, U>>(lds))
        return false;
    // a launch of at most 2^14 chunks of rows: a grid has 2^16 of them, and 2^32 threads
    const int64_t chunks = ((int64_t)a.rows + 16 * MT - 1) / (16 * MT), slots = waves == 8 ? 512 : 256;
    for (int64_t c = 0; c < chunks; c += 1 << 14)
    {
        RowsArgs part     = a;
        const int64_t m   = c * 16 * MT, end = (c + (1 << 14)) * 16 * MT;
        part.rows         = (int32_t)((end < a.rows ? end : a.rows) - m);
        part.x += m * a.ldx, part.out += m * a.ldo;
        const int64_t here = chunks - c < (1 << 14) ? chunks - c : 1 << 14;
        const int64_t side = slots / here > 1 ? slots / here : 1;
        int4_stream_kernel<T, PER, MT, GATED, U><<<dim3((int)(a.n_blocks < side ? a.n_blocks : side), (int)here), 64 * waves, lds, st>>>(part);
    }
    return true;
}

template <typename T, int PER, int MT, bool GATED, bool ODD, bool SHARED>
bool launch_short(hipStream_t st, const RowsArgs& a)
{
    constexpr int U = PER ? 4 : MT == 1 && !ODD ? 2 : 1, S = GATED ? 2 : 1;
    const int waves  = a.per_split < 1 ? 1 : a.per_split < kShortWaves ? a.per_split : kShortWaves;
    const size_t lds = (size_t)waves * S * MT * 1024;
    if (!ensure_dynamic_lds<few_rows_kernel<T, PER, MT, GATED, U, ODD, SHARED>>(lds))
        return false;
    // a grid has 2^16 chunks of rows, and 2^32 threads
    const int64_t chunks = ((int64_t)a.rows + 16 * MT - 1) / (16 * MT), most = (int64_t(1) << 22) / a.tiles_n < 1 << 14 ? (int64_t(1) << 22) / a.tiles_n : 1 << 14;
    const int64_t step   = most < 1 ? 1 : most;
    for (int64_t c = 0; c < chunks; c += step)
    {
        RowsArgs part   = a;
        const int64_t m = c * 16 * MT, end = (c + step) * 16 * MT;
        part.rows       = (int32_t)((end < a.rows ? end : a.rows) - m);
        part.x += m * a.ldx, part.out += m * a.ldo;
        if (a.pre_gate)
            part.pre_gate += m * a.ldo, part.pre_up += m * a.ldo;
        few_rows_kernel<T, PER, MT, GATED, U, ODD, SHARED><<<dim3(a.tiles_n, (int)(chunks - c < step ? chunks - c : step), a.splits), 64 * waves, lds, st>>>(part);
    }
    // (sums are split only where one launch has all rows)
    if (a.splits > 1)
        few_rows_join_kernel<T, PER == 0, MT, GATED><<<dim3(a.tiles_n, (int)chunks), 256, 0, st>>>(a);
    return true;
}

// Rows that begin at odd elements, us with one load for 16 bytes / in words: 1, 16 and 32 rows with 2 x 8192 x 2047 in bf16 28.2, 38.9, 51.4 / 15.1, 18.8, 24.4,
// 16 rows with 2 x 2000 x 2048 in 4 bits 7.4 / 5.6.
template <typename T, int PER, int MT, bool GATED>
bool launch_short(hipStream_t st, const RowsArgs& a)
{
    bool odd = ((a.ldx & 1) && a.rows > 1) || (reinterpret_cast<uintptr_t>(a.x) & 2);
    if (PER == 0)
        odd |= (a.ldw & 1) || ((reinterpret_cast<uintptr_t>(a.w[0]) | reinterpret_cast<uintptr_t>(a.w[1])) & 2);
    if (PER || a.splits > 1)
        return odd ? launch_short<T, PER, MT, GATED, true, true>(st, a) : launch_short<T, PER, MT, GATED, false, true>(st, a);
    return odd ? launch_short<T, PER, MT, GATED, true, PER != 0>(st, a) : launch_short<T, PER, MT, GATED, false, PER != 0>(st, a);
}

// The short kernel up to four rows and 32 MB of weights, and up to 16 rows and 8 MB (x goes to it once for every 16 weight rows).  us short /
// stream: one row 512 x 512 2.4 / 4.0, 4096 x 4096 4.1 / 5.4, 12000 x 4096 8.5 / 9.2, 16384 x 4096 10.1 / 10.4, 65536 x 8192 68 / 60, 2 x 11000 x 4096
// 16.0 / 14.7; 4 rows 8192 x 4096 7.1 / 8.4; 16 rows 4096 x 4096 6.7 / 8.6, 12000 x 4096 13.0 / 11.2, 2 x 5500 x 2048 9.4 / 8.1.
template <typename T, int PER, bool GATED>
bool choose(hipStream_t st, const RowsArgs& a)
{
    if (a.splits > 1)
        return launch_short<T, PER, 1, GATED>(st, a);
    const int64_t kb = a.tiles * (GATED ? 2 : 1);
    if (a.rows <= 16 && kb <= (a.rows <= 4 ? 32768 : 8192))
        return launch_short<T, PER, 1, GATED>(st, a);
    RowsArgs one = a, two = a, four = a;
    int w1 = 8, w2 = 8, w4 = 8;
    const double us1 = plan<T, PER, 1, GATED>(one, w1);
    if (a.rows <= 16)
        return launch_stream<T, PER, 1, GATED>(st, one, w1);
    // more row tiles a workgroup against fewer workgroups
    const double us2 = plan<T, PER, 2, GATED>(two, w2), us4 = plan<T, PER, 4, GATED>(four, w4);
    if (us1 <= us2 && us1 <= us4)
        return launch_stream<T, PER, 1, GATED>(st, one, w1);
    return a.rows <= 32 || us2 <= us4 ? launch_stream<T, PER, 2, GATED>(st, two, w2) : launch_stream<T, PER, 4, GATED>(st, four, w4);
}

template <int PER>
bool choose(hipStream_t st, int32_t dtype, bool gated, const RowsArgs& a)
{
    if (dtype == TMI_BF16)
        return gated ? choose<bf16_t, PER, true>(st, a) : choose<bf16_t, PER, false>(st, a);
    return gated ? choose<_Float16, PER, true>(st, a) : choose<_Float16, PER, false>(st, a);
}

RowsArgs rows_args(int32_t rows, int32_t n, int32_t k, const void* x, int64_t ldx, const void* w0, const void* w1, void* out, int64_t ldo)
{
    RowsArgs a{};
    a.x = static_cast<const uint16_t*>(x), a.out = static_cast<uint16_t*>(out);
    a.w[0] = static_cast<const uint8_t*>(w0), a.w[1] = static_cast<const uint8_t*>(w1);
    a.ldx = ldx, a.ldo = ldo, a.rows = rows, a.n = n, a.k = k;
    a.tiles_n = (int32_t)int4_tiles(n, kInt4Rows), a.tiles_k = (int32_t)int4_tiles(k, kInt4Cols);
    a.tiles   = (int64_t)a.tiles_n * a.tiles_k;
    a.splits  = 1, a.per_split = a.tiles_k;
    return a;
}

// How many workgroups share the columns of a weight row tile.  Few tiles with long rows leave most of the chip idle while each of eight waves goes through
// its columns in turns of U tiles, 2 to 4 us each; joining the parts is a launch more, which two turns do not pay.  More than 16 rows of x in 4 bits would
// otherwise go to the stream, whose workgroups have more rows.  us with all columns in one workgroup / shared, in 4 bits: 14 rows 256 x 24008 18.4 / 7.5,
// one row 512 x 16384 (four turns) 9.1 / 6.1, 1024 x 8192 (two) 5.4 / 6.0, 19 rows 2 x 104 x 4636 13.4 / 7.6; in 16 bits: one row 2 x 1000 x 8192 (four) 18.5
// / 11.7, 2 x 2000 x 4096 (two) 10.7 / 11.4.
int few_rows_splits(bool dense, int32_t rows, int32_t n, int32_t k)
{
    const int at_once      = kShortWaves * (dense ? (rows <= 16 ? 2 : 1) : 4), of_x = dense && rows > 16 ? 32 : 16;
    const int64_t tiles_k  = int4_tiles(k, kInt4Cols), tiles = int4_tiles(n, kInt4Rows) * int4_tiles(rows, of_x);
    const int64_t turns    = int4_tiles(tiles_k, at_once), places = 512 / (tiles > 0 ? tiles : 1);
    if (tiles > 128 || tiles_k <= (!dense && rows > 16 ? 1 : 2) * at_once)
        return 1;
    return (int)(turns < places ? turns : places);
}

void share_columns(RowsArgs& a, int splits, float* sums)
{
    a.per_split = (int32_t)int4_tiles(a.tiles_k, splits);
    a.splits    = (int32_t)int4_tiles(a.tiles_k, a.per_split);
    a.sums      = sums;
}

}    // namespace

size_t few_rows_scratch_bytes(bool dense, bool gated, int32_t rows, int32_t n, int32_t k)
{
    const int splits = few_rows_splits(dense, rows, n, k), of_x = dense && rows > 16 ? 32 : 16;
    return splits == 1 ? 0 : (size_t)int4_tiles(n, kInt4Rows) * int4_tiles(rows, of_x) * splits * (gated ? 2 : 1) * of_x * 64;
}

const char* launch_int4_rows(hipStream_t st, int32_t dtype, int32_t group, bool gated, int32_t act, int32_t rows, int32_t n, int32_t k, const void* x,
                             int64_t ldx, const void* w, const void* up, void* out, int64_t ldo, void* scratch)
{
    RowsArgs a = rows_args(rows, n, k, x, ldx, w, up, out, ldo);
    a.act      = act;
    if (scratch)
        share_columns(a, few_rows_splits(false, rows, n, k), static_cast<float*>(scratch));
    const bool ok = group == 32 ? choose<4>(st, dtype, gated, a) : group == 64 ? choose<2>(st, dtype, gated, a) : choose<1>(st, dtype, gated, a);
    return !ok ? nullptr : gated ? "int4_rows_gated" : "int4_rows";
}

const char* launch_ffn_rows(hipStream_t st, int32_t dtype, int32_t act, int32_t rows, int32_t d, int32_t f, const void* x, int64_t ldx,
                            const void* gate, const void* up, int64_t ldw, void* out, void* pre_gate, void* pre_up, int64_t ldo, void* scratch)
{
    RowsArgs a = rows_args(rows, f, d, x, ldx, gate, up, out, ldo);
    a.act = act, a.ldw = ldw;
    if (scratch)
        share_columns(a, few_rows_splits(true, rows, f, d), static_cast<float*>(scratch));
    a.pre_gate = static_cast<uint16_t*>(pre_gate), a.pre_up = static_cast<uint16_t*>(pre_up);
    bool ok;
    if (rows <= 16)
        ok = dtype == TMI_BF16 ? launch_short<bf16_t, 0, 1, true>(st, a) : launch_short<_Float16, 0, 1, true>(st, a);
    else
        ok = dtype == TMI_BF16 ? launch_short<bf16_t, 0, 2, true>(st, a) : launch_short<_Float16, 0, 2, true>(st, a);
    return ok ? "ffn_rows" : nullptr;
}

}    // namespace tmi
