// The gated feed-forward block on many rows, and its gradients, on the matrix cores:
//
//   forward    h[m][f]  = act(sum_d x[m][d] gate[f][d]) * (sum_d x[m][d] up[f][d])
//   slopes     dp[m]    = [ dh u act'(g) | dh act(g) ], rows of 2 FP elements, FP = F up to whole blocks of 64, zeros behind F
//   d_x        dx[m][d] = sum_f dp[m][f] gate[f][d] + dp[m][FP + f] up[f][d]
//   d_w        dw[f][d] = sum_m dp[m][f] x[m][d], f over gate and up
//
// One kernel makes all three products.  The operand whose index runs along an output row ("columns": weights, weights, x) is the first of the
// 32x32x16 matrix instruction, so that a lane owns 16 neighbouring results of one row; the other ("rows": x, dp, dp) is the second.  An operand
// lies in memory with the summed index innermost (forward: both; d_x: dp) or outermost (d_x: the weights; d_w: both).  Either way 16-byte pieces
// go to LDS as they lie; an outermost one comes out through the transposing reads ds_read_b64_tr_b16.  So nothing is transposed in memory.
//
// The forward pass deals gate and up rows of the same 32 features to one wave as its two column tiles: activation and product are done on the
// accumulators, and the pre-activations leave the chip only if they are asked for.
//
// LDS: a stage holds 64 of the summed index.  Innermost: rows of 128 bytes, 16-byte piece c of row r at c ^ (r / 2 % 8).  Outermost: 64 rows
// of the tile's width, their 64-byte segments moved by the row's number mod 4.  Both keep the 16 (32) lanes that the LDS serves at once on
// banks of their own.
#include "tmi_ffn.h"
#include <type_traits>

namespace tmi
{
namespace
{

enum
{
    OP_FORWARD,
    OP_DX,
    OP_DW
};

struct GemmFfnArgs
{
    const uint16_t* col[2];    // gate and up, or x twice
    const uint16_t* row;       // x or dp
    uint16_t* out[2];          // h; dx; d_gate and d_up
    uint16_t *pre_gate, *pre_up;
    float* part;               // partial sums [split][(gate, up)][M][N], where the sum is split
    const uint8_t* zeros;      // 64 bytes
    int64_t ldc, ldr, ldo;     // elements
    int32_t M, N;              // results: rows and columns (features of h; d; d)
    int32_t K;                 // summed index (of one half, for d_x)
    int32_t half;              // FP, the columns of each half of dp
    int32_t features;          // F
    int32_t blocks;            // of 64 of the summed index
    int32_t tiles_m, tiles_n, tiles, per_xcd;
    int32_t splits, per_split; // blocks of a split
    int32_t act;
};

__device__ __forceinline__ int swizzle_in(int r)
{
    return (r >> 1) & 7;
}

constexpr int kGroup = 8;    // row tiles that neighbouring workgroups share column tiles over

template <typename T, int OP, int WC, int WR, int RT, bool FAST>
__global__ __launch_bounds__(64 * WC * WR, 2) void gated_gemm_kernel(GemmFfnArgs a)
{
    constexpr int THREADS  = 64 * WC * WR;
    constexpr int BN       = 64 * WC, BM = 32 * RT * WR;
    constexpr bool CIN     = OP == OP_FORWARD;    // summed index innermost: columns operand
    constexpr bool RIN     = OP != OP_DW;         // rows operand
    constexpr int CB       = BN * 128, STAGE = (BN + BM) * 128;
    constexpr int CL       = BN * 8 / THREADS, RL = BM * 8 / THREADS;    // 16-byte loads of a thread and block
    constexpr int TN       = CIN ? BN / 2 : BN;    // results a tile's columns make
    static_assert(CL * THREADS == BN * 8 && RL * THREADS == BM * 8, "a block must split evenly over the threads");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wc = wave % WC, wr = wave / WC;
    const int rho = lane & 31, h = lane >> 5;

    // workgroups go round-robin to the 8 XCDs; each takes a contiguous range of the tile list, along rows in groups of kGroup
    const int t = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
    if (t >= a.tiles * a.splits)
        return;
    const int split = t / a.tiles, tile = t - split * a.tiles;
    const int in_group = kGroup * a.tiles_n, group = tile / in_group, rest = tile - group * in_group;
    const int rows_here = a.tiles_m - group * kGroup < kGroup ? a.tiles_m - group * kGroup : kGroup;
    const int tn = rest / rows_here, tm = group * kGroup + rest - tn * rows_here;
    const int64_t n0 = (int64_t)tn * TN, m0 = (int64_t)tm * BM;
    const int block0 = split * a.per_split;
    const int block1 = block0 + a.per_split < a.blocks ? block0 + a.per_split : a.blocks;

    // ---- what a thread loads: 16-byte unit u = j * THREADS + tid of either operand's part of a stage -------------------------
    struct Unit
    {
        int64_t row;    // innermost: row of the operand, past the end the last one; outermost: row of the block
        int col;        // first element of the piece: of the block, or of the tile
    };
    auto col_unit = [&](int j) {
        const int u = j * THREADS + tid;
        if constexpr (CIN)
        {
            const int r     = u >> 3;
            const int64_t f = n0 + (r >> 6) * 32 + (r & 31);    // rows 0..31 of 64 are gate's, the others up's
            return Unit{ f < a.N ? f : a.N - 1, ((u & 7) ^ swizzle_in(r)) * 8 };
        }
        else
        {
            const int k = u / (BN / 8);
            return Unit{ k, ((u % (BN / 8)) ^ ((k & 3) << 2)) * 8 };
        }
    };
    auto row_unit = [&](int j) {
        const int u = j * THREADS + tid;
        if constexpr (RIN)
        {
            const int r     = u >> 3;
            const int64_t m = m0 + r;
            return Unit{ m < a.M ? m : a.M - 1, ((u & 7) ^ swizzle_in(r)) * 8 };
        }
        else
        {
            const int k = u / (BM / 8);
            return Unit{ k, ((u % (BM / 8)) ^ ((k & 3) << 2)) * 8 };
        }
    };
    // which of the two column operands load j of this wave (forward), or block n (d_x), comes from
    auto col_base = [&](int j, int n) {
        if constexpr (CIN)
            return a.col[((j * THREADS + wave * 64) >> 3 >> 5) & 1];
        else
            return a.col[OP == OP_DX && n * 64 >= a.half ? 1 : 0];
    };
    // first of the summed index of block n, within its half, and where it ends
    auto block_k = [&](int n) { return OP == OP_DX && n * 64 >= a.half ? n * 64 - a.half : n * 64; };

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    uint32_t cvoff[FAST ? CL : 1], rvoff[FAST ? RL : 1];
    if constexpr (FAST)
    {
#pragma unroll
        for (int j = 0; j < CL; j++)
        {
            const Unit u = col_unit(j);
            if constexpr (CIN)
                cvoff[j] = (uint32_t)((u.row - n0) * a.ldc + u.col) * 2;
            else    // pieces past the row's end repeat the last one; never stored
                cvoff[j] = (uint32_t)(u.row * a.ldc + (u.col < a.N - 8 - n0 ? u.col : a.N - 8 - n0)) * 2;
        }
#pragma unroll
        for (int j = 0; j < RL; j++)
        {
            const Unit u = row_unit(j);
            if constexpr (RIN)
                rvoff[j] = (uint32_t)((u.row - m0) * a.ldr + u.col) * 2;
            else
                rvoff[j] = (uint32_t)(u.row * a.ldr + (u.col < a.M - 8 - m0 ? u.col : a.M - 8 - m0)) * 2;
        }
    }
    auto direct = [&](const uint16_t* base, uint32_t voff, uint32_t dst) {
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(base), "s"(dst) : "memory");
    };
    auto direct_or_zero = [&](const uint16_t* base, uint32_t voff, bool inside, uint32_t dst) {
        const uint8_t* src = inside ? reinterpret_cast<const uint8_t*>(base) + voff : a.zeros;
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(dst) : "memory");
    };
    // FAST: all loads of block n into stage s, straight to LDS
    auto issue = [&](int n, int s) {
        const int k0         = block_k(n);
        const bool whole     = k0 + 64 <= a.K;
        const uint32_t stage = lds0 + s * STAGE + wave * 1024;
#pragma unroll
        for (int j = 0; j < CL; j++)
        {
            const uint16_t* base = col_base(j, n) + (CIN ? n0 * a.ldc + k0 : k0 * a.ldc + n0);
            const uint32_t dst   = stage + j * THREADS * 16;
            if (whole)
                direct(base, cvoff[j], dst);
            else
            {
                const Unit u = col_unit(j);
                direct_or_zero(base, cvoff[j], k0 + (CIN ? u.col : (int)u.row) < a.K, dst);
            }
        }
        const int rk = OP == OP_DX ? n * 64 : k0;    // dp holds both halves, filled up with zeros
#pragma unroll
        for (int j = 0; j < RL; j++)
        {
            const uint16_t* base = a.row + (RIN ? m0 * a.ldr + rk : rk * a.ldr + m0);
            const uint32_t dst   = stage + CB + j * THREADS * 16;
            if (whole || OP == OP_DX)
                direct(base, rvoff[j], dst);
            else
            {
                const Unit u = row_unit(j);
                direct_or_zero(base, rvoff[j], k0 + (RIN ? u.col : (int)u.row) < a.K, dst);
            }
        }
    };
    // otherwise through registers: rows that begin at any element, and that end inside a piece
    v4i creg[FAST ? 1 : CL], rreg[FAST ? 1 : RL];
    auto fetch = [&](int n) {
        const int k0 = block_k(n);
#pragma unroll
        for (int j = 0; j < CL; j++)
        {
            const Unit u         = col_unit(j);
            const uint16_t* base = col_base(j, n);
            if constexpr (CIN)
                creg[j] = load8(base + u.row * a.ldc, k0 + u.col, a.K);
            else
                creg[j] = load8(base + (k0 + u.row) * a.ldc, n0 + u.col, k0 + u.row < a.K ? a.N : 0);
        }
#pragma unroll
        for (int j = 0; j < RL; j++)
        {
            const Unit u = row_unit(j);
            if constexpr (OP == OP_DX)
                rreg[j] = *reinterpret_cast<const v4i*>(a.row + u.row * a.ldr + n * 64 + u.col);
            else if constexpr (RIN)
                rreg[j] = load8(a.row + u.row * a.ldr, k0 + u.col, a.K);
            else
                rreg[j] = load8(a.row + (k0 + u.row) * a.ldr, m0 + u.col, k0 + u.row < a.K ? a.M : 0);
        }
    };
    auto put = [&](int s) {
        uint8_t* stage = lds + s * STAGE;
#pragma unroll
        for (int j = 0; j < CL; j++)
            *reinterpret_cast<v4i*>(stage + (j * THREADS + tid) * 16) = creg[j];
#pragma unroll
        for (int j = 0; j < RL; j++)
            *reinterpret_cast<v4i*>(stage + CB + (j * THREADS + tid) * 16) = rreg[j];
    };

    // ---- what a lane reads --------------------------------------------------------------------------------------------------
    const int crow = channel_of_row(rho);
    const int sl = lane & 15, m4 = sl >> 2, a4 = sl & 3, brho = (lane >> 4) & 1;
    uint32_t caddr[CIN ? 4 : 2], raddr[RIN ? 4 : RT];    // by step, or by tile
    if constexpr (CIN)
#pragma unroll
        for (int s = 0; s < 4; s++)
            caddr[s] = (wc * 64 + crow) * 128 + (((2 * s + h) ^ swizzle_in(crow)) * 16);
    else
#pragma unroll
        for (int c = 0; c < 2; c++)    // source lane: row m4 of four, columns of the lanes 4 a4 ... 4 a4 + 3
            caddr[c] = (8 * h + m4) * (BN * 2) + (((wc * 2 + c) ^ m4) << 6) + 2 * (16 * (a4 & 1) + 4 * (2 * brho + (a4 >> 1)));
    if constexpr (RIN)
#pragma unroll
        for (int s = 0; s < 4; s++)
            raddr[s] = CB + (wr * 32 * RT + rho) * 128 + (((2 * s + h) ^ swizzle_in(rho)) * 16);
    else
#pragma unroll
        for (int i = 0; i < RT; i++)
            raddr[i] = CB + (8 * h + m4) * (BM * 2) + (((wr * RT + i) ^ m4) << 6) + 2 * (16 * brho + 4 * a4);
    auto transposed = [&](const uint8_t* at, int rows_apart) {
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
        const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + rows_apart)));
        return v4i{ lo.x, lo.y, hi.x, hi.y };
    };

    v16f acc[2][RT];
#pragma unroll
    for (int c = 0; c < 2; c++)
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                acc[c][i][e] = 0.0f;

    auto multiply = [&](int stage) {
        const uint8_t* sb = lds + stage * STAGE;
#pragma unroll
        for (int s = 0; s < 4; s++)
        {
            v4i fc[2], fr[RT];
#pragma unroll
            for (int c = 0; c < 2; c++)
                if constexpr (CIN)
                    fc[c] = *reinterpret_cast<const v4i*>(sb + caddr[s] + c * 4096);
                else
                    fc[c] = transposed(sb + caddr[c] + 16 * s * (BN * 2), 4 * (BN * 2));
#pragma unroll
            for (int i = 0; i < RT; i++)
                if constexpr (RIN)
                    fr[i] = *reinterpret_cast<const v4i*>(sb + raddr[s] + i * 4096);
                else
                    fr[i] = transposed(sb + raddr[i] + 16 * s * (BM * 2), 4 * (BM * 2));
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int c = 0; c < 2; c++)
                    acc[c][i] = Mma<T>::mma(fc[c], fr[i], acc[c][i]);
        }
    };

    if constexpr (FAST)
    {
        if (block0 < block1)
            issue(block0, 0);
        for (int n = block0; n < block1; n++)
        {
            // block n has landed, and every wave is past block n - 1, whose stage the next loads overwrite
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (n + 1 < block1)
                issue(n + 1, (n + 1 - block0) & 1);
            multiply((n - block0) & 1);
        }
    }
    else
    {
        if (block0 < block1)
        {
            fetch(block0);
            put(0);
        }
        __syncthreads();
        for (int n = block0; n < block1; n++)
        {
            if (n + 1 < block1)
                fetch(n + 1);
            multiply((n - block0) & 1);
            if (n + 1 < block1)
                put((n + 1 - block0) & 1);
            __syncthreads();
        }
    }

    // ---- results: a lane has 16 neighbours of a row from each accumulator tile -----------------------------------------------
    auto store16 = [&](uint16_t* row, int64_t at, int64_t end, const float* v) {
#pragma unroll
        for (int q = 0; q < 2; q++)
        {
            v4i w;
#pragma unroll
            for (int p = 0; p < 4; p++)
                w[p] = (int)pack16<T>(v[8 * q + 2 * p], v[8 * q + 2 * p + 1]);
            store8(row, at + 8 * q, end, w);
        }
    };
    auto store_part = [&](int which, int64_t m, int64_t at, const v16f& v) {
        float* row = a.part + (((int64_t)split * (CIN ? 2 : 1) + which) * a.M + m) * a.N;
#pragma unroll
        for (int q = 0; q < 4; q++)
        {
            const v4f w = { v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3] };
            if (at + 4 * q + 4 <= a.N)
                __builtin_memcpy(row + at + 4 * q, &w, 16);
            else
#pragma unroll
                for (int e = 0; e < 3; e++)
                    if (at + 4 * q + e < a.N)
                        row[at + 4 * q + e] = w[e];
        }
    };
#pragma unroll
    for (int i = 0; i < RT; i++)
    {
        const int64_t m = m0 + (wr * RT + i) * 32 + rho;
        if (m >= a.M)
            continue;
        if constexpr (OP == OP_FORWARD)
        {
            const int64_t f = n0 + wc * 32 + 16 * h;
            if (a.splits > 1)
            {
                store_part(0, m, f, acc[0][i]);
                store_part(1, m, f, acc[1][i]);
                continue;
            }
            float v[16];
            if (a.pre_gate)
            {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    v[e] = acc[0][i][e];
                store16(a.pre_gate + m * a.ldo, f, a.N, v);
#pragma unroll
                for (int e = 0; e < 16; e++)
                    v[e] = acc[1][i][e];
                store16(a.pre_up + m * a.ldo, f, a.N, v);
            }
#pragma unroll
            for (int e = 0; e < 16; e++)
                v[e] = act_value(a.act, acc[0][i][e]) * acc[1][i][e];
            store16(a.out[0] + m * a.ldo, f, a.N, v);
        }
        else
        {
            uint16_t* row = a.out[0];
            int64_t r     = m;
            if constexpr (OP == OP_DW)
            {
                // rows of dp's halves behind their F features are none of a gradient's
                const int half = m >= a.half ? 1 : 0;
                r              = m - (half ? a.half : 0);
                row            = a.out[half];
                if (r >= a.features)
                    continue;
            }
#pragma unroll
            for (int c = 0; c < 2; c++)
            {
                const int64_t d = n0 + wc * 64 + c * 32 + 16 * h;
                if (a.splits > 1)
                {
                    store_part(0, m, d, acc[c][i]);
                    continue;
                }
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; e++)
                    v[e] = acc[c][i][e];
                store16(row + r * a.ldo, d, a.N, v);
            }
        }
    }
}

// Results of a sum that was split: the parts in the order of the splits, then what the unsplit kernel does with a sum.
template <typename T, int OP>
__global__ __launch_bounds__(256) void gated_join_kernel(GemmFfnArgs a)
{
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
    if (n >= a.N)
        return;
    constexpr int W     = OP == OP_FORWARD ? 2 : 1;
    const int64_t plane = (int64_t)a.M * a.N;
    const float* part   = a.part + m * a.N + n;
    float v[W];
#pragma unroll
    for (int w = 0; w < W; w++)
        v[w] = 0.0f;
    for (int s = 0; s < a.splits; s++)
#pragma unroll
        for (int w = 0; w < W; w++)
            v[w] += part[(s * W + w) * plane];
    if constexpr (OP == OP_FORWARD)
    {
        const int64_t at = m * a.ldo + n;
        if (a.pre_gate)
            a.pre_gate[at] = to_bits16<T>(v[0]), a.pre_up[at] = to_bits16<T>(v[W - 1]);
        a.out[0][at] = to_bits16<T>(act_value(a.act, v[0]) * v[W - 1]);
    }
    else
    {
        const int half  = OP == OP_DW && m >= a.half ? 1 : 0;
        const int64_t r = m - (half ? a.half : 0);
        if (OP == OP_DX || r < a.features)
            a.out[half][r * a.ldo + n] = to_bits16<T>(v[0]);
    }
}

// dp: eight features of a row a thread, of both halves
struct SlopeArgs
{
    const uint16_t *pre_gate, *pre_up, *dh;
    uint16_t* dp;
    int64_t ld, units;    // units: rows * half / 8
    int32_t features, half, act;
};

template <typename T>
__global__ __launch_bounds__(256) void gated_slope_kernel(SlopeArgs a)
{
    const int per_row = a.half / 8;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < a.units; u += (int64_t)gridDim.x * 256)
    {
        const int64_t m = u / per_row;
        const int f     = (int)(u - m * per_row) * 8;
        const v4i g = load8(a.pre_gate + m * a.ld, f, a.features), up = load8(a.pre_up + m * a.ld, f, a.features),
                  dh = load8(a.dh + m * a.ld, f, a.features);
        v4i dg, du;
#pragma unroll
        for (int p = 0; p < 4; p++)
        {
            float x[2], y[2];
#pragma unroll
            for (int e = 0; e < 2; e++)
            {
                float value, slope;
                act_both(a.act, from_bits16<T>(half_of(g, 2 * p + e)), value, slope);
                const float d = from_bits16<T>(half_of(dh, 2 * p + e));
                x[e] = d * from_bits16<T>(half_of(up, 2 * p + e)) * slope;
                y[e] = d * value;
                if (f + 2 * p + e >= a.features)
                    x[e] = 0.0f, y[e] = 0.0f;
            }
            dg[p] = (int)pack16<T>(x[0], x[1]);
            du[p] = (int)pack16<T>(y[0], y[1]);
        }
        uint16_t* row = a.dp + m * 2 * a.half + f;
        *reinterpret_cast<v4i*>(row)          = dg;
        *reinterpret_cast<v4i*>(row + a.half) = du;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

struct Shape
{
    bool large;      // 256 x 256 (eight waves) or 128 x 128 (four waves, two workgroups a CU)
    int splits, per_split;
    int tiles_m, tiles_n;
};

// 256 x 256 where that fills two thirds of the CUs.  Smaller products go to 128 x 128, and where those are few and the sum is long it is split,
// into parts of eight blocks (512 of the summed index) at least.  Operands that are read through registers take 128 x 128: the others' accumulators
// leave no room.
Shape shape_of(int op, int64_t M, int64_t N, int blocks, bool fast)
{
    Shape s{};
    auto tiles = [&](int size) {
        s.tiles_m = (int)((M + size - 1) / size);
        const int tn = op == OP_FORWARD ? size / 2 : size;
        s.tiles_n = (int)((N + tn - 1) / tn);
        return (int64_t)s.tiles_m * s.tiles_n;
    };
    s.large = fast && tiles(256) >= 170;
    s.splits = 1, s.per_split = blocks;
    if (!s.large)
    {
        const int64_t n = tiles(128);
        int64_t want = n >= 256 || n < 1 ? 1 : (512 + n - 1) / n;    // (a product of no results is planned too)
        want         = want < blocks / 8 ? want : blocks / 8;
        if (want > 1)
        {
            s.per_split = (int)((blocks + want - 1) / want);
            s.splits    = (blocks + s.per_split - 1) / s.per_split;
        }
    }
    return s;
}

size_t part_bytes(int op, const Shape& s, int64_t M, int64_t N)
{
    return s.splits > 1 ? (size_t)s.splits * (op == OP_FORWARD ? 2 : 1) * M * N * 4 : 0;
}

template <typename T, int OP, int WC, int WR, int RT, bool FAST>
bool launch_tiles(hipStream_t st, const GemmFfnArgs& a)
{
    constexpr size_t lds = 2 * (64 * WC + 32 * RT * WR) * 128;
    if (!ensure_dynamic_lds<gated_gemm_kernel<T, OP, WC, WR, RT, FAST>>(lds))
        return false;
    gated_gemm_kernel<T, OP, WC, WR, RT, FAST><<<a.per_xcd * 8, 64 * WC * WR, lds, st>>>(a);
    return true;
}

template <int OP>
bool launch_product(hipStream_t st, int32_t dtype, GemmFfnArgs a, const Shape& s, bool fast)
{
    a.tiles_m = s.tiles_m, a.tiles_n = s.tiles_n, a.tiles = s.tiles_m * s.tiles_n;
    a.splits = s.splits, a.per_split = s.per_split;
    a.per_xcd = (a.tiles * a.splits + 7) / 8;
    auto typed = [&](auto type) {
        using T = decltype(type);
        bool ok;
        if (s.large)
            ok = launch_tiles<T, OP, 4, 2, 4, true>(st, a);
        else
            ok = fast ? launch_tiles<T, OP, 2, 2, 2, true>(st, a) : launch_tiles<T, OP, 2, 2, 2, false>(st, a);
        if (ok && s.splits > 1)
            gated_join_kernel<T, OP><<<dim3((a.N + 255) / 256, a.M), 256, 0, st>>>(a);
        return ok;
    };
    return dtype == TMI_BF16 ? typed(bf16_t{}) : typed(_Float16{});
}

// whether rows of `width` elements, `ld` apart, are whole 16-byte pieces, and near enough for 32-bit offsets over a tile
bool whole_pieces(const void* p, int64_t width, int64_t ld)
{
    return ((uintptr_t)p & 15) == 0 && width % 8 == 0 && ld % 8 == 0 && ld < (int64_t(1) << 22);
}

// What a call launches, from its sizes, strides and addresses
struct ForwardPlan
{
    int blocks;
    bool fast;
    Shape shape;
};
ForwardPlan forward_plan(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up)
{
    ForwardPlan p;
    p.blocks = (int)(((int64_t)d.in_features + 63) / 64);
    p.fast   = whole_pieces(x, d.in_features, d.ld_x) && whole_pieces(gate, d.in_features, d.ld_w) && whole_pieces(up, d.in_features, d.ld_w);
    p.shape  = shape_of(OP_FORWARD, d.rows, d.hidden_features, p.blocks, p.fast);
    return p;
}
struct BackwardPlan
{
    int64_t half;
    size_t dp_bytes;
    int dx_blocks, dw_blocks;
    bool dx_fast, dw_fast;
    Shape dx, dw;
};
BackwardPlan backward_plan(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up)
{
    BackwardPlan p;
    p.half           = ((int64_t)d.hidden_features + 63) / 64 * 64;
    p.dp_bytes       = (size_t)d.rows * 2 * p.half * 2;
    p.dx_blocks      = (int)(2 * p.half / 64);
    p.dw_blocks      = (int)(((int64_t)d.rows + 63) / 64);
    const bool near  = 2 * p.half < (int64_t(1) << 22);
    p.dx_fast        = near && whole_pieces(gate, d.in_features, d.ld_w) && whole_pieces(up, d.in_features, d.ld_w);
    p.dw_fast        = near && whole_pieces(x, d.in_features, d.ld_x);
    p.dx             = shape_of(OP_DX, d.rows, d.in_features, p.dx_blocks, p.dx_fast);
    p.dw             = shape_of(OP_DW, 2 * p.half, d.in_features, p.dw_blocks, p.dw_fast);
    return p;
}

}    // namespace

size_t gated_ffn_scratch_bytes(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up)
{
    return part_bytes(OP_FORWARD, forward_plan(d, x, gate, up).shape, d.rows, d.hidden_features);
}

const char* launch_gated_ffn(hipStream_t st, const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up, void* h, void* pre_gate,
                             void* pre_up, void* scratch, const void* zeros)
{
    ForwardPlan p = forward_plan(d, x, gate, up);
    if (!scratch)
        p.shape.splits = 1, p.shape.per_split = p.blocks;
    GemmFfnArgs a{};
    a.col[0] = static_cast<const uint16_t*>(gate), a.col[1] = static_cast<const uint16_t*>(up), a.row = static_cast<const uint16_t*>(x);
    a.out[0] = static_cast<uint16_t*>(h);
    a.pre_gate = static_cast<uint16_t*>(pre_gate), a.pre_up = static_cast<uint16_t*>(pre_up);
    a.part = static_cast<float*>(scratch), a.zeros = static_cast<const uint8_t*>(zeros);
    a.ldc = d.ld_w, a.ldr = d.ld_x, a.ldo = d.ld_h;
    a.M = d.rows, a.N = d.hidden_features, a.K = d.in_features, a.blocks = p.blocks, a.act = d.activation;
    return launch_product<OP_FORWARD>(st, d.dtype, a, p.shape, p.fast) ? "gated_ffn" : nullptr;
}

// dp, then the partial sums of one product after the other
size_t gated_ffn_backward_scratch_bytes(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up, bool dx, bool dw)
{
    const BackwardPlan p = backward_plan(d, x, gate, up);
    const size_t of_dx   = dx ? part_bytes(OP_DX, p.dx, d.rows, d.in_features) : 0;
    const size_t of_dw   = dw ? part_bytes(OP_DW, p.dw, 2 * p.half, d.in_features) : 0;
    return p.dp_bytes + (of_dx > of_dw ? of_dx : of_dw);
}

const char* launch_gated_ffn_backward(hipStream_t st, const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up,
                                      const void* pre_gate, const void* pre_up, const void* d_h, void* d_x, void* d_gate, void* d_up, void* scratch,
                                      const void* zeros)
{
    const BackwardPlan p = backward_plan(d, x, gate, up);
    SlopeArgs q{};
    q.pre_gate = static_cast<const uint16_t*>(pre_gate), q.pre_up = static_cast<const uint16_t*>(pre_up), q.dh = static_cast<const uint16_t*>(d_h);
    q.dp = static_cast<uint16_t*>(scratch), q.ld = d.ld_h, q.units = d.rows * (p.half / 8);
    q.features = d.hidden_features, q.half = (int32_t)p.half, q.act = d.activation;
    const int64_t groups = (q.units + 255) / 256;
    const int grid       = (int)(groups < 4096 ? groups : 4096);
    if (grid > 0 && d.dtype == TMI_BF16)
        gated_slope_kernel<bf16_t><<<grid, 256, 0, st>>>(q);
    else if (grid > 0)
        gated_slope_kernel<_Float16><<<grid, 256, 0, st>>>(q);

    GemmFfnArgs a{};
    a.row = q.dp, a.ldr = 2 * p.half, a.half = (int32_t)p.half, a.features = d.hidden_features;
    a.part  = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + p.dp_bytes);
    a.zeros = static_cast<const uint8_t*>(zeros);
    a.N     = d.in_features;
    bool ok = true;
    if (d_x)
    {
        a.col[0] = static_cast<const uint16_t*>(gate), a.col[1] = static_cast<const uint16_t*>(up), a.ldc = d.ld_w;
        a.out[0] = static_cast<uint16_t*>(d_x), a.out[1] = nullptr, a.ldo = d.ld_x;
        a.M = d.rows, a.K = d.hidden_features, a.blocks = p.dx_blocks;
        ok = launch_product<OP_DX>(st, d.dtype, a, p.dx, p.dx_fast);
    }
    if (ok && d_gate)
    {
        a.col[0] = a.col[1] = static_cast<const uint16_t*>(x), a.ldc = d.ld_x;
        a.out[0] = static_cast<uint16_t*>(d_gate), a.out[1] = static_cast<uint16_t*>(d_up), a.ldo = d.ld_w;
        a.M = (int32_t)(2 * p.half), a.K = d.rows, a.blocks = p.dw_blocks;
        ok = launch_product<OP_DW>(st, d.dtype, a, p.dw, p.dw_fast);
    }
    return ok ? "gated_ffn_backward" : nullptr;
}

}    // namespace tmi
