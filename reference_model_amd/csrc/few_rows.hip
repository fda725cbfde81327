// Products of a few rows with large weights, and the gated block on them:
//
//   y[m][n] = sum_k x[m][k] w[n][k]                h[m][f] = act(sum_k x[m][k] gate[f][k]) * (sum_k x[m][k] up[f][k])
//
// w in 4 bits with a scale for each group of columns (y and h), or gate and up in 16 bits (h).  With up to 64 rows the weights' bytes are all
// that counts: each is read once, by one wave, straight into the registers from which the matrix instruction takes it.
//
// A workgroup owns NT tiles of 16 weight rows (of both matrices, if gated) and all of K, dealt to its waves in tiles of 128 columns; what the
// waves have summed meets in LDS in the order of the waves, so equal calls give equal bits.  16x16x32 instructions take the rows of x as first
// operand and the weights as second: a single row wastes 15/16 of the matrix cores, which at 512 weights an instruction still run four times
// as many weights as HBM delivers, and any other number of rows up to 16 costs the same.  4-bit weights become 16-bit integers (exact; 9 to 20
// instructions for eight), their products are summed in 32 bits, and the sum over a group is multiplied by its scale: no weight is
// rounded, and an infinite or NaN x does to a row what it does in the formula.
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
    int32_t tiles_n, tiles_k, full_k;    // row tiles, column tiles and those of them that are whole
    int32_t n_blocks, act;
};

constexpr int kMostWaves = 8;

// PER: groups of a 4-bit tile, 0 = 16-bit weights; U: column tiles whose loads a wave has in flight together
template <typename T, int PER, int MT, int NT, bool GATED, int U>
__global__ __launch_bounds__(64 * kMostWaves) void few_rows_kernel(RowsArgs a)
{
    constexpr bool DENSE = PER == 0;
    constexpr int S      = GATED ? 2 * NT : NT;    // streams of weights: gate and up of a row tile are neighbours
    constexpr int WV     = DENSE ? 4 : 1;          // 16-byte loads of a lane, stream and column tile
    extern __shared__ __attribute__((aligned(16))) float red[];    // [wave][stream][row tile][4][lane]

    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int chunk = blockIdx.x / a.n_blocks, nb = blockIdx.x - chunk * a.n_blocks;
    const int64_t row0 = (int64_t)chunk * (16 * MT);

    const uint16_t* xrow[MT];
    bool live[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
    {
        const int64_t m = row0 + 16 * mt + r;
        live[mt]        = m < a.rows;
        xrow[mt]        = a.x + (live[mt] ? m : 0) * a.ldx;
    }
    const uint8_t* wbase[S];      // 4 bits: the lane's bytes of the row tile's first column tile; 16 bits: the lane's row
    const uint8_t* sbase[S];
#pragma unroll
    for (int s = 0; s < S; s++)
    {
        int tn = nb * NT + (GATED ? s >> 1 : s);
        tn     = tn < a.tiles_n ? tn : a.tiles_n - 1;    // tiles past the end repeat the last one and are not stored
        const uint8_t* w = a.w[GATED ? s & 1 : 0];
        if constexpr (DENSE)
        {
            int64_t n = (int64_t)tn * 16 + r;
            n         = n < a.n ? n : a.n - 1;
            wbase[s]  = w + n * a.ldw * 2;
        }
        else
        {
            const int64_t t = (int64_t)tn * a.tiles_k;
            wbase[s]        = w + t * kInt4TileBytes + lane * 16;
            sbase[s]        = w + int4_scale_at(a.tiles, t, PER) + r * (2 * PER);
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
        uint16_t scale[S][DENSE ? 1 : PER];
    };
    auto fetch_w = [&](Tile& t, int kt, auto tail) {
#pragma unroll
        for (int s = 0; s < S; s++)
        {
            if constexpr (DENSE)
            {
                const uint16_t* row = reinterpret_cast<const uint16_t*>(wbase[s]);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    t.w[s][j] = decltype(tail)::value ? load8(row, (int64_t)kt * 128 + 32 * j + 8 * q, a.k)
                                                      : load16(reinterpret_cast<const uint8_t*>(row + (int64_t)kt * 128 + 32 * j + 8 * q));
            }
            else
            {
                t.w[s][0] = *reinterpret_cast<const v4i*>(wbase[s] + (int64_t)kt * kInt4TileBytes);
                __builtin_memcpy(t.scale[s], sbase[s] + (int64_t)kt * (kInt4Rows * 2 * PER), 2 * PER);
            }
        }
    };
    auto fetch_x = [&](Tile& t, int kt, auto tail) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                t.x[mt][j]      = v4i{ 0, 0, 0, 0 };
                const int64_t k = (int64_t)kt * 128 + 32 * j + 8 * q;
                if constexpr (decltype(tail)::value)
                    t.x[mt][j] = load8(xrow[mt], k, a.k, live[mt]);
                else if (live[mt])
                    t.x[mt][j] = load16(reinterpret_cast<const uint8_t*>(xrow[mt] + k));
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
                    const float scale = from_bits16<T>(t.scale[s][g]);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            acc[s][mt][i] = __builtin_fmaf(scale, d[mt][i], acc[s][mt][i]);
                }
            }
    };

    for (int k0 = wave; k0 < a.full_k; k0 += U * waves)
    {
        Tile t[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k0 + u * waves < a.full_k)
                fetch_w(t[u], k0 + u * waves, std::false_type());
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k0 + u * waves < a.full_k)
                fetch_x(t[u], k0 + u * waves, std::false_type());
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k0 + u * waves < a.full_k)
                multiply(t[u]);
    }
    if (a.full_k < a.tiles_k && a.full_k % waves == wave)
    {
        Tile t;
        fetch_w(t, a.full_k, std::true_type());
        fetch_x(t, a.full_k, std::true_type());
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
    auto results = [&](auto ACT) {
        for (int o = threadIdx.x; o < NT * MT * 256; o += blockDim.x)
        {
            const int t = o / (MT * 256), mt = o / 256 % MT, ln = o & 63;
            const int64_t n = ((int64_t)nb * NT + t) * 16 + (ln & 15);
            const int64_t m = row0 + 16 * mt + (ln >> 4) * 4 + (o >> 6 & 3);
            if (n >= a.n || m >= a.rows)
                continue;
            constexpr float unit = DENSE ? 1.0f : 1.0f / kInt4Unit<T>;
            float v[2] = { 0.0f, 0.0f };
#pragma unroll
            for (int half = 0; half < (GATED ? 2 : 1); half++)
            {
                const int s = GATED ? 2 * t + half : t;
                for (int w = 0; w < waves; w++)
                    v[half] += red[((w * S + s) * MT + mt) * 256 + (o & 255)];
                v[half] *= unit;
            }
            const int64_t at = m * a.ldo + n;
            if constexpr (GATED)
                a.out[at] = to_bits16<T>(act_value<decltype(ACT)::value>(v[0]) * v[1]);
            else
                a.out[at] = to_bits16<T>(v[0]);
            if constexpr (GATED && DENSE)
                if (a.pre_gate)
                    a.pre_gate[at] = to_bits16<T>(v[0]), a.pre_up[at] = to_bits16<T>(v[1]);
        }
    };
    if constexpr (GATED)
        for_act(a.act, results);
    else
        results(0);
}

template <typename T, int PER, int MT, int NT, bool GATED>
bool launch(hipStream_t st, RowsArgs a)
{
    constexpr int U = MT == 1 ? (PER ? 4 : 2) : (MT == 2 && PER ? 2 : 1);
    constexpr int S = GATED ? 2 * NT : NT;
    auto kernel     = few_rows_kernel<T, PER, MT, NT, GATED, U>;
    const int waves = a.tiles_k < 1 ? 1 : (a.tiles_k < kMostWaves ? a.tiles_k : kMostWaves);
    const size_t lds = (size_t)waves * S * MT * 1024;
    a.n_blocks       = (a.tiles_n + NT - 1) / NT;
    if (!ensure_dynamic_lds<few_rows_kernel<T, PER, MT, NT, GATED, U>>(lds))
        return false;
    // a launch of at most 2^22 workgroups (or one row chunk of them), as a grid may not have 2^32 threads
    const int64_t chunks = ((int64_t)a.rows + 16 * MT - 1) / (16 * MT), most = (int64_t(1) << 22) / a.n_blocks;
    const int64_t step   = most < 1 ? 1 : most;
    for (int64_t c = 0; c < chunks; c += step)
    {
        RowsArgs part     = a;
        const int64_t m   = c * 16 * MT;
        const int64_t end = (c + step) * 16 * MT;
        part.rows = (int32_t)((end < a.rows ? end : a.rows) - m);
        part.x += m * a.ldx, part.out += m * a.ldo;
        if (a.pre_gate)
            part.pre_gate += m * a.ldo, part.pre_up += m * a.ldo;
        kernel<<<(int)(a.n_blocks * (step < chunks - c ? step : chunks - c)), 64 * waves, lds, st>>>(part);
    }
    return true;
}

template <typename T, int PER, bool GATED>
bool choose(hipStream_t st, const RowsArgs& a)
{
    const bool wide = (int64_t)a.tiles_n >= (GATED ? 1024 : 2048);
    if (a.rows <= 16)
        return wide ? launch<T, PER, 1, 2, GATED>(st, a) : launch<T, PER, 1, 1, GATED>(st, a);
    if (a.rows <= 32)
        return wide ? launch<T, PER, 2, 2, GATED>(st, a) : launch<T, PER, 2, 1, GATED>(st, a);
    return launch<T, PER, 4, 1, GATED>(st, a);
}

template <int PER, bool GATED>
bool choose(hipStream_t st, int32_t dtype, const RowsArgs& a)
{
    return dtype == TMI_BF16 ? choose<bf16_t, PER, GATED>(st, a) : choose<_Float16, PER, GATED>(st, a);
}

RowsArgs rows_args(int32_t rows, int32_t n, int32_t k, const void* x, int64_t ldx, const void* w0, const void* w1, void* out, int64_t ldo)
{
    RowsArgs a{};
    a.x = static_cast<const uint16_t*>(x), a.out = static_cast<uint16_t*>(out);
    a.w[0] = static_cast<const uint8_t*>(w0), a.w[1] = static_cast<const uint8_t*>(w1);
    a.ldx = ldx, a.ldo = ldo, a.rows = rows, a.n = n, a.k = k;
    a.tiles_n = (int32_t)int4_tiles(n, kInt4Rows), a.tiles_k = (int32_t)int4_tiles(k, kInt4Cols), a.full_k = k / kInt4Cols;
    a.tiles   = (int64_t)a.tiles_n * a.tiles_k;
    return a;
}

}    // namespace

const char* launch_int4_rows(hipStream_t st, int32_t dtype, int32_t group, bool gated, int32_t act, int32_t rows, int32_t n, int32_t k, const void* x,
                             int64_t ldx, const void* w, const void* up, void* out, int64_t ldo)
{
    RowsArgs a = rows_args(rows, n, k, x, ldx, w, up, out, ldo);
    a.act      = act;
    bool ok    = false;
    if (group == 32)
        ok = gated ? choose<4, true>(st, dtype, a) : choose<4, false>(st, dtype, a);
    else if (group == 64)
        ok = gated ? choose<2, true>(st, dtype, a) : choose<2, false>(st, dtype, a);
    else if (group == 128)
        ok = gated ? choose<1, true>(st, dtype, a) : choose<1, false>(st, dtype, a);
    return !ok ? nullptr : gated ? "int4_rows_gated" : "int4_rows";
}

const char* launch_ffn_rows(hipStream_t st, int32_t dtype, int32_t act, int32_t rows, int32_t d, int32_t f, const void* x, int64_t ldx,
                            const void* gate, const void* up, int64_t ldw, void* out, void* pre_gate, void* pre_up, int64_t ldo)
{
    RowsArgs a = rows_args(rows, f, d, x, ldx, gate, up, out, ldo);
    a.act = act, a.ldw = ldw;
    a.pre_gate = static_cast<uint16_t*>(pre_gate), a.pre_up = static_cast<uint16_t*>(pre_up);
    return choose<0, true>(st, dtype, a) ? "ffn_rows" : nullptr;
}

}    // namespace tmi
