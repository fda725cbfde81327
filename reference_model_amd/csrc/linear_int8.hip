// The linear layer on 8-bit activations and weights, with a scale for each token and each output feature:
//
//   y[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n]
//
// The sum is exact: products of 8 bits in 32-bit integers, by the matrix instruction 16x16x64.  It becomes a 32-bit float (rounded to 24 bits), is
// multiplied by both scales, and rounded once.  Rows of x and w begin at multiples of 16 bytes and are filled up with zeros to the next one, so that
// every piece of 16 bytes goes as it lies into LDS or a matrix instruction.
//
// The weights are the first operand of the instruction and x the second, so that a lane owns neighbouring features of one token.
//
// linear_tile_kernel: many tokens.  Workgroups that stay go through a list of tiles.  Operands go straight from memory into LDS, 128 columns of 8 rows an
// instruction: whole cache lines (loads of 64 bytes of 16 rows bring 51 bytes a nanosecond and CU out of L2, of 128 bytes of 8 rows 136).  They are requested
// four to two matrix instruction depths ahead, across the borders of tiles: while a workgroup stores one tile's results the next one's operands are on their way.
//
// linear_rows_kernel: few tokens, bound by the weights' bytes.  A workgroup has 16 weight rows, its eight or 16 waves split the columns, operands go
// from memory into the instruction's registers, and the sums meet in LDS.
#include "tmi_rows.h"

namespace tmi
{
namespace
{

struct LinearArgs
{
    const uint8_t *w, *x;
    const float *w_scales, *x_scales;
    const void* bias;
    void* out;
    int32_t* part;           // partial sums [split][M][N], where the sum is split
    const uint8_t* zeros;    // 64 bytes
    int64_t ldw, ldx, ldo;   // bytes, bytes, elements
    int32_t M, N;
    int32_t K;               // columns, up to whole 16s
    int32_t blocks;          // of 64 columns, up to a whole pair
    int32_t tiles_m, tiles_n, tiles;
    int32_t splits, per_split;    // blocks of a split
    int32_t items, per_xcd;       // tiles times splits
};

constexpr int kGroup = 8;    // row tiles that neighbouring workgroups share column tiles over
constexpr int kBlock = 64;   // columns of a matrix instruction
constexpr int kPair  = 128;  // of a unit in LDS

__device__ __forceinline__ v4i mma_int8(v4i a, v4i b, v4i c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ float bias_at(const void* bias, int64_t n)
{
    if constexpr (sizeof(T) == 4)
        return static_cast<const float*>(bias)[n];
    else
        return from_bits16<T>(static_cast<const uint16_t*>(bias)[n]);
}
template <typename T>
__device__ __forceinline__ void store_one(void* out, int64_t at, float v)
{
    if constexpr (sizeof(T) == 4)
        static_cast<float*>(out)[at] = v;
    else
        static_cast<uint16_t*>(out)[at] = to_bits16<T>(v);
}

// Piece c (16 bytes) of row r (128 bytes) of a unit lies at c ^ swizzle(r).  The LDS serves 16-byte reads of 16 lanes at once, of each half wave the quads (4
// lanes) {0, 3, 5, 6} and then {1, 2, 4, 7}; lane l reads piece l / 16 (and 4 more for the second block) of row l % 16.  Of the 16 rows of a set eight are even
// and eight odd, which use different halves of 256 bytes; of the even ones four read one piece and four its neighbour, at r / 2 = 0, 1, 6, 7 and 2, 3, 4, 5: all
// eight places are taken once.
__device__ __forceinline__ int swizzle(int r)
{
    return (r >> 1) & 7;
}
// WC x WR waves (features x tokens) that compute, of 64 features and 16 RT tokens each, and LW that load; LDS holds R pairs of blocks.  SPLIT: partial sums
template <typename T, int WC, int WR, int RT, int LW, int R, bool SPLIT>
__global__ __launch_bounds__(64 * (WC * WR + LW), (WC * WR + LW) / 4) void linear_tile_kernel(LinearArgs a)
{
    constexpr int CT = 4, BN = 16 * CT * WC, BM = 16 * RT * WR;
    constexpr int PAIR = (BN + BM) * kPair;    // of LDS: the weights, then x
    using Out = std::conditional_t<SPLIT, float, T>;    // (a partial sum is a word, as a float is)
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Workgroups go round-robin to the 8 XCDs; each of those has a contiguous range of the list, along rows in groups of kGroup, which its workgroups go
    // through side by side.
    const int per_turn = gridDim.x >> 3, first_item = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
    const int of_xcd = ((int)(blockIdx.x & 7) + 1) * a.per_xcd, last_item = of_xcd < a.items ? of_xcd : a.items;
    if (first_item >= last_item)
        return;
    struct Item
    {
        int64_t m0, n0;
        int split, block0, block1;
    };
    auto item_of = [&](int t) {
        Item r;
        r.split        = SPLIT ? t / a.tiles : 0;
        const int tile = t - r.split * a.tiles, in_group = kGroup * a.tiles_n, group = tile / in_group, rest = tile - group * in_group;
        const int rows_here = a.tiles_m - group * kGroup < kGroup ? a.tiles_m - group * kGroup : kGroup;
        const int tn = rest / rows_here, tm = group * kGroup + rest - tn * rows_here;
        r.m0 = (int64_t)tm * BM, r.n0 = (int64_t)tn * BN;
        r.block0 = SPLIT ? r.split * a.per_split : 0;
        r.block1 = SPLIT && r.block0 + a.per_split < a.blocks ? r.block0 + a.per_split : a.blocks;
        return r;
    };
    // For results of 16 bits row 16 c + p of 32 holds feature 8 (p / 4) + 4 c + p % 4: a lane then owns eight neighbours, and four lanes 64 bytes in a row, as
    // they do of 32 bits where row and feature are the same.
    auto feature_of_row = [](int r) { return sizeof(Out) == 4 ? r : (r & ~31) + 8 * (r >> 2 & 3) + 4 * (r >> 4 & 1) + (r & 3); };

    // Barrier p (behind the first, which says that pair 0 is there) says that pair p + 1 is there and that nobody reads pair p any more.
    if (wave >= WC * WR)
    {
        // ---- waves that load: 16-byte piece u = j * 64 LW + tid of a pair, row u / 8, of the weights' rows and then of x's ------------
        constexpr int STEP = 8 * LW, WJ = BN / STEP, XJ = BM / STEP, LOADS = WJ + XJ;
        static_assert(WJ * STEP == BN && XJ * STEP == BM && STEP % 16 == 0, "all pieces of a thread have one place in their rows");
        static_assert(R >= 2 && (R - 1) * LOADS < 64, "loads in flight are counted in six bits");
        const int tid       = threadIdx.x - 64 * WC * WR, row0 = tid >> 3, piece = ((tid & 7) ^ swizzle(row0)) * 16;
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + (wave - WC * WR) * 1024;
        const uint32_t woff = (uint32_t)(feature_of_row(row0) * a.ldw), xoff = (uint32_t)(row0 * a.ldx);
        // the item, its block that is requested next, where that lies, the last rows' offsets from there, and the place it goes to
        int item, block, end, slot = 0;
        const uint8_t *wat, *xat;
        uint32_t wlast, xlast;
        auto begin = [&](int t) {
            const Item it       = item_of(t);
            const int64_t lastw = a.N - 1 - it.n0, lastx = a.M - 1 - it.m0;
            item = t, block = it.block0, end = it.block1;
            wat = a.w + it.n0 * a.ldw + it.block0 * kBlock, xat = a.x + it.m0 * a.ldx + it.block0 * kBlock;
            wlast = (uint32_t)((lastw < BN - 1 ? lastw : BN - 1) * a.ldw), xlast = (uint32_t)((lastx < BM - 1 ? lastx : BM - 1) * a.ldx);
        };
        // Past the last pair it is requested again, into places nobody reads: the loads in flight are then as many all the time.
        auto request = [&]() {
            const bool inside = block * kBlock + piece < a.K;
#pragma unroll
            for (int j = 0; j < LOADS; j++)
            {
                // (rows past the last repeat it and are not stored; j steps are other bits of a row than the thread's, so that features add up)
                const bool is_w    = j < WJ;
                const uint32_t row = is_w ? woff + (uint32_t)(feature_of_row(j * STEP) * a.ldw) : xoff + (uint32_t)((j - WJ) * STEP * a.ldx);
                const uint32_t off = (is_w ? (row < wlast ? row : wlast) : (row < xlast ? row : xlast)) + piece;
                // (zeros where the columns end in the pair)
                const uint8_t* src = inside ? (is_w ? wat : xat) + off : a.zeros;
                asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds0 + slot * PAIR + j * (STEP * kPair)) : "memory");
            }
            slot = slot + 1 < R ? slot + 1 : 0;
            block += 2, wat += kPair, xat += kPair;
            if (block >= end)
            {
                if (item + per_turn < last_item)
                    begin(item + per_turn);
                else
                    block -= 2, wat -= kPair, xat -= kPair;
            }
        };
        begin(first_item);
#pragma unroll 1
        for (int p = 0; p < R; p++)
            request();
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((R - 1) * LOADS) : "memory");
#pragma unroll 1
        for (int t = first_item; t < last_item; t += per_turn)
        {
            const Item it = item_of(t);
#pragma unroll 1
            for (int n = it.block0; n < it.block1; n += 2)
            {
                asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((R - 2) * LOADS) : "memory");
                request();
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        return;
    }

    // ---- waves that compute: a lane reads piece q4 (and q4 + 4 in the second block) of row l16 of a tile -------------------------------
    const int wc = wave % WC, wr = wave / WC, l16 = lane & 15, q4 = lane >> 4;
    const uint32_t place = ((q4 ^ swizzle(l16)) * 16), waddr = (wc * 16 * CT + l16) * kPair + place, xaddr = (BN + wr * 16 * RT + l16) * kPair + place;
    v4i acc[CT][RT];
    v4i fw[2][CT], fx[RT];
    auto read_w = [&](int set, uint32_t at, int c) { fw[set][c] = *reinterpret_cast<const v4i*>(lds + at + c * (16 * kPair)); };
    auto read_x = [&](uint32_t at, int i) { fx[i] = *reinterpret_cast<const v4i*>(lds + at + i * (16 * kPair)); };

    // A block is one matrix instruction deep.  A wave takes it row tile by row tile; when a row tile is done its fragment is read from the next
    // block, a block ahead of its use, and the column tiles' fragments into a second set.  So behind the first row tile of a pair's second block all of the pair
    // is read.  Reads stand behind matrix instructions one by one, and are kept there: their wait for a slot passes while the matrix cores work.
    uint32_t slot = 0;    // bytes
    auto one_block = [&](auto SET) {
        constexpr int P = decltype(SET)::value;    // which of the pair
        if constexpr (P == 1)
            slot = slot + PAIR < R * PAIR ? slot + PAIR : 0;
        const uint32_t wat = slot + (P == 1 ? waddr : waddr ^ 64), xat = slot + (P == 1 ? xaddr : xaddr ^ 64);
#pragma unroll
        for (int i = 0; i < RT; i++)
        {
#pragma unroll
            for (int k = 0; k < CT; k++)
            {
                const int c = i & 1 ? CT - 1 - k : k;    // (one operand changes at a time)
                acc[c][i]   = mma_int8(fw[P][c], fx[i], acc[c][i]);
                if (i > 0 && (RT >= CT ? k == 2 && i < CT : k >= 1))
                    read_w(1 - P, wat, RT >= CT ? i : k);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i == 0)
            {
                if constexpr (P == 1)
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                read_w(1 - P, wat, 0);
            }
            read_x(xat, i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    static_assert(RT == 2 || RT >= CT, "where the weights' fragments are read");

    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int c = 0; c < CT; c++)
        read_w(0, waddr, c);
#pragma unroll
    for (int i = 0; i < RT; i++)
        read_x(xaddr, i);
    __builtin_amdgcn_sched_barrier(0);

#pragma unroll 1
    for (int t = first_item; t < last_item; t += per_turn)
    {
        const Item it = item_of(t);
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int i = 0; i < RT; i++)
                acc[c][i] = v4i{ 0, 0, 0, 0 };
#pragma unroll 1
        for (int n = it.block0; n < it.block1; n += 2)
        {
            one_block(std::integral_constant<int, 0>());
            one_block(std::integral_constant<int, 1>());
        }

        // ---- results: of each of a lane's rows four or two pieces of 16 bytes, of the features of_piece(0), ... on -----------------------
        constexpr int V = kPiece<Out>, TILES = V / 4;    // (column tiles that a piece comes from)
        auto of_piece = [&](int p) { return it.n0 + wc * 16 * CT + 16 * TILES * p + V * q4; };
        float of_row[RT];
        if constexpr (!SPLIT)
#pragma unroll
            for (int i = 0; i < RT; i++)
            {
                const int64_t m = it.m0 + (wr * RT + i) * 16 + l16;
                of_row[i]       = a.x_scales[m < a.M ? m : a.M - 1];
            }
#pragma unroll
        for (int p = 0; p < CT / TILES; p++)
        {
            const int64_t n = of_piece(p);
            float scale[V], bias[V];
            if constexpr (!SPLIT)
#pragma unroll
                for (int e = 0; e < V; e++)
                {
                    const int64_t f = n + e < a.N ? n + e : a.N - 1;
                    scale[e] = a.w_scales[f], bias[e] = a.bias ? bias_at<T>(a.bias, f) : 0.0f;
                }
#pragma unroll
            for (int i = 0; i < RT; i++)
            {
                const int64_t m = it.m0 + (wr * RT + i) * 16 + l16;
                float y[V];
#pragma unroll
                for (int e = 0; e < V; e++)
                {
                    const int sum = acc[TILES * p + e / 4][i][e & 3];
                    if constexpr (SPLIT)
                        y[e] = __int_as_float(sum);
                    else
                        y[e] = __builtin_fmaf((float)sum * scale[e], of_row[i], bias[e]);
                }
                Out* row = SPLIT ? reinterpret_cast<Out*>(a.part) + ((int64_t)it.split * a.M + m) * a.N : static_cast<Out*>(a.out) + m * a.ldo;
                if (m < a.M && n < a.N)
                    store_piece<Out, false>(row + n, 0, (int)(a.N - n < V ? a.N - n : V), piece_of<Out>(y));
            }
        }
    }
}

// Results of a sum that was split, four of a row a thread: integers, so the order does not matter
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a)
{
    const int64_t n = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= a.N)
        return;
    const int live      = a.N - n < 4 ? (int)(a.N - n) : 4;
    const int64_t plane = (int64_t)a.M * a.N;
    for (int64_t m = blockIdx.y; m < a.M; m += gridDim.y)
    {
        v4i v = { 0, 0, 0, 0 };
        for (int s = 0; s < a.splits; s++)
        {
            const int32_t* at = a.part + s * plane + m * a.N + n;
            v4i t             = { 0, 0, 0, 0 };
            if (live == 4)
                __builtin_memcpy(&t, at, 16);
            else
#pragma unroll
                for (int e = 0; e < 3; e++)
                    if (e < live)
                        t[e] = at[e];
            v += t;
        }
        const float xs = a.x_scales[m];
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (e < live)
                store_one<T>(a.out, m * a.ldo + n + e, __builtin_fmaf((float)v[e] * a.w_scales[n + e], xs, a.bias ? bias_at<T>(a.bias, n + e) : 0.0f));
    }
}

// RT tiles of 16 tokens against 16 features; a wave has every pair of blocks of WAVES, U pairs on their way at once.  SPLIT: partial sums
template <typename T, int RT, int U, int WAVES, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES) void linear_rows_kernel(LinearArgs a)
{
    __shared__ v4i met[WAVES][RT * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (16 * RT);

    // (rows past the last repeat it)
    const int64_t f  = n0 + l16 < a.N ? n0 + l16 : a.N - 1;
    const uint8_t *w = a.w + f * a.ldw, *x[RT];
#pragma unroll
    for (int i = 0; i < RT; i++)
    {
        const int64_t m = m0 + i * 16 + l16;
        x[i]            = a.x + (m < a.M ? m : a.M - 1) * a.ldx;
    }
    v4i acc[RT];
#pragma unroll
    for (int i = 0; i < RT; i++)
        acc[i] = v4i{ 0, 0, 0, 0 };

    const int pairs = a.blocks / 2, first = SPLIT ? (int)blockIdx.z * (a.per_split / 2) : 0;
    const int last  = SPLIT && first + a.per_split / 2 < pairs ? first + a.per_split / 2 : pairs;
#pragma unroll 1
    for (int p = first + wave; p < last; p += WAVES * U)
    {
        v4i fw[U * 2], fx[U * 2][RT];
        bool inside[U * 2];
#pragma unroll
        for (int u = 0; u < U * 2; u++)
        {
            const int pair = p + (u >> 1) * WAVES, k = pair * kPair + (u & 1) * kBlock + q4 * 16;
            inside[u]      = pair < last && k < a.K;
            const int at   = inside[u] ? k : 0;
            fw[u]          = *reinterpret_cast<const v4i*>(w + at);
#pragma unroll
            for (int i = 0; i < RT; i++)
                fx[u][i] = *reinterpret_cast<const v4i*>(x[i] + at);
        }
#pragma unroll
        for (int u = 0; u < U * 2; u++)
        {
            const v4i live = inside[u] ? fw[u] : v4i{ 0, 0, 0, 0 };
#pragma unroll
            for (int i = 0; i < RT; i++)
                acc[i] = mma_int8(live, fx[u][i], acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < RT; i++)
        met[wave][i * 64 + lane] = acc[i];
    __syncthreads();
#pragma unroll
    for (int u = tid; u < RT * 64; u += 64 * WAVES)
    {
        v4i v = met[0][u];
#pragma unroll
        for (int k = 1; k < WAVES; k++)
            v += met[k][u];
        const int l = u & 63;
        const int64_t m = m0 + (u >> 6) * 16 + (l & 15), n = n0 + 4 * (l >> 4);
        if (m >= a.M)
            continue;
        const float of_row = SPLIT ? 1.0f : a.x_scales[m];
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < a.N)
            {
                if constexpr (SPLIT)
                    a.part[((int64_t)blockIdx.z * a.M + m) * a.N + n + e] = v[e];
                else
                    store_one<T>(a.out, m * a.ldo + n + e,
                                 __builtin_fmaf((float)v[e] * a.w_scales[n + e], of_row, a.bias ? bias_at<T>(a.bias, n + e) : 0.0f));
            }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

enum
{
    ROWS,        // linear_rows_kernel
    TILE_256,    // 256 features x 128 tokens, eight waves that compute and four that load
    TILE_128,    // 128 x 128, four and four
    TILE_64      // 64 x 64, two and two, three workgroups a CU
};
struct Plan
{
    int kind;
    int splits, per_split;
};
constexpr int kMostSplits = 16;

// of 64 columns, in whole pairs
int blocks_of(int32_t columns)
{
    return (int)((whole16(columns) + kPair - 1) / kPair) * 2;
}

int64_t tiles_of(int64_t n, int64_t per)
{
    return (n + per - 1) / per;
}

// What linear_rows_kernel takes, us
double rows_us(int64_t M, int64_t N, int blocks)
{
    const int rt       = M > 48 ? 4 : (int)tiles_of(M, 16);
    const double turns = (double)tiles_of(blocks, rt > 1 ? 16 : blocks >= 64 ? 64 : 32) * (rt > 1 ? 1.0 + 0.12 * rt : 1.1);
    const double w = (double)N * blocks * 64, x = (double)(M < 64 ? M : tiles_of(M, 64) * 64) * tiles_of(N, 16) * blocks * 64;
    const double bytes = w * tiles_of(M, 64) / 6.2e6, all = (w * tiles_of(M, 64) + x) / 8.5e6;
    return 2.0 + (turns > bytes ? (turns > all ? turns : all) : bytes > all ? bytes : all);
}
double join_us(int64_t M, int64_t N, int splits)
{
    return splits > 1 ? 2.3 + (double)M * N * 8 * splits / 7.5e6 : 0;
}

Plan plan_of(const tmi_linear_int8_desc_t& d)
{
    const int64_t M = d.rows, N = d.out_features;
    const int blocks = blocks_of(d.in_features);
    Plan p{ ROWS, 1, blocks };
    // (a lane's offset over a tile is held in 32 bits)
    const bool far = d.ld_x >= (int64_t(1) << 23) || d.ld_w >= (int64_t(1) << 23);
    if (far || blocks == 0)
        return p;
    double least = M <= 256 ? rows_us(M, N, blocks) : 1e30;
    auto take    = [&](int kind, double us, int splits, int per) {
        if (us < least)
            least = us, p = Plan{ kind, splits, per };
    };
    auto per_cu = [](int64_t items) { return (double)((items + 255) / 256); };
    const int64_t t256 = tiles_of(M, 128) * tiles_of(N, 256), t128 = tiles_of(M, 128) * tiles_of(N, 128), t64 = tiles_of(M, 64) * tiles_of(N, 64);
    take(TILE_256, 4.5 + per_cu(t256) * (blocks * (t256 >= 200 ? 0.377 : 0.29) + 2.4), 1, blocks);
    take(TILE_128, 3.6 + per_cu(t128) * (blocks * (t128 >= 200 ? 0.22 : 0.165) + 2.4), 1, blocks);
    for (int want = 1; want <= kMostSplits && want <= blocks / 2; want++)
    {
        const int per = (blocks / 2 + want - 1) / want * 2, splits = (blocks + per - 1) / per;
        const double n = per_cu(t64 * splits);
        take(TILE_64, 3.6 + per * (0.105 * n > 0.145 ? 0.105 * n : 0.145) + 0.7 * n + join_us(M, N, splits), splits, per);
        if (M <= 64 && splits > 1)
            take(ROWS, rows_us(M, N * splits, per) + join_us(M, N, splits), splits, per);
    }
    return p;
}

template <typename T, int WC, int WR, int RT, int LW, int R, bool SPLIT>
bool launch_tiles(hipStream_t st, LinearArgs a, int places)
{
    constexpr int BN = 64 * WC, BM = 16 * RT * WR;
    constexpr size_t lds  = R * (BN + BM) * kPair;
    constexpr auto kernel = linear_tile_kernel<T, WC, WR, RT, LW, R, SPLIT>;
    if (!ensure_dynamic_lds<kernel>(lds))
        return false;
    a.tiles_m = (a.M + BM - 1) / BM, a.tiles_n = (a.N + BN - 1) / BN, a.tiles = a.tiles_m * a.tiles_n;
    a.items = a.tiles * a.splits, a.per_xcd = (a.items + 7) / 8;
    const int grid = a.per_xcd * 8 < places ? a.per_xcd * 8 : places;
    kernel<<<grid, 64 * (WC * WR + LW), lds, st>>>(a);
    return true;
}

template <int N>
constexpr std::integral_constant<int, N> number_of{};

template <typename T>
void launch_join(hipStream_t st, const LinearArgs& a)
{
    if (a.splits > 1)
        linear_join_kernel<T><<<dim3((a.N + 1023) / 1024, a.M < 32768 ? a.M : 32768), 256, 0, st>>>(a);
}

template <typename T>
bool launch_typed(hipStream_t st, const LinearArgs& a, const Plan& p)
{
    if (p.kind == ROWS)
    {
        auto go = [&](auto SPLIT, auto RT, auto U, auto WAVES) {
            constexpr int rt = decltype(RT)::value, waves = decltype(WAVES)::value;
            linear_rows_kernel<T, rt, decltype(U)::value, waves, decltype(SPLIT)::value>
                <<<dim3((a.N + 15) / 16, (a.M + 16 * rt - 1) / (16 * rt), a.splits), 64 * waves, 0, st>>>(a);
        };
        auto rows = [&](auto SPLIT) {
            // Few waves and loads on their way for short columns, more for long ones.  us 1 x 1024 x 4096 with two pairs and eight waves 3.5, with two and 16 3.6,
            // with four and eight 4.6; 1 x 8192 x 8192 14.4, 12.8 and 13.2.
            if (a.M <= 16 && a.per_split >= 64)
                go(SPLIT, number_of<1>, number_of<2>, number_of<16>);
            else if (a.M <= 16)
                go(SPLIT, number_of<1>, number_of<2>, number_of<8>);
            else if (a.M <= 32)
                go(SPLIT, number_of<2>, number_of<1>, number_of<8>);
            else if (a.M <= 48)
                go(SPLIT, number_of<3>, number_of<1>, number_of<8>);
            else
                go(SPLIT, number_of<4>, number_of<1>, number_of<8>);
        };
        if (a.splits > 1)
            rows(std::true_type());
        else
            rows(std::false_type());
        launch_join<T>(st, a);
        return true;
    }
    bool ok;
    if (p.kind == TILE_256)
        ok = launch_tiles<T, 4, 2, 4, 4, 3, false>(st, a, 256);
    else if (p.kind == TILE_128)
        ok = launch_tiles<T, 2, 2, 4, 4, 5, false>(st, a, 256);
    else
        ok = p.splits > 1 ? launch_tiles<float, 1, 2, 2, 2, 3, true>(st, a, 768) : launch_tiles<T, 1, 2, 2, 2, 3, false>(st, a, 768);
    if (ok)
        launch_join<T>(st, a);
    return ok;
}

}    // namespace

size_t linear_int8_scratch_bytes(const tmi_linear_int8_desc_t& d)
{
    const Plan p = plan_of(d);
    return p.splits > 1 ? (size_t)p.splits * d.rows * d.out_features * 4 : 0;
}

const char* launch_linear_int8(hipStream_t st, const tmi_linear_int8_desc_t& d, const void* x, const float* x_scales, const void* w, const float* w_scales,
                               const void* bias, void* y, void* scratch, const void* zeros)
{
    Plan p           = plan_of(d);
    const int blocks = blocks_of(d.in_features);
    if (!scratch)
        p.splits = 1, p.per_split = blocks;
    LinearArgs a{};
    a.w = static_cast<const uint8_t*>(w), a.x = static_cast<const uint8_t*>(x), a.w_scales = w_scales, a.x_scales = x_scales;
    a.bias = bias, a.out = y, a.part = static_cast<int32_t*>(scratch), a.zeros = static_cast<const uint8_t*>(zeros);
    a.ldw = d.ld_w, a.ldx = d.ld_x, a.ldo = d.ld_y;
    a.M = d.rows, a.N = d.out_features, a.K = (int32_t)whole16(d.in_features), a.blocks = blocks;
    a.splits = p.splits, a.per_split = p.per_split;
    const bool ok = d.dtype == TMI_FP16 ? launch_typed<_Float16>(st, a, p) : d.dtype == TMI_BF16 ? launch_typed<bf16_t>(st, a, p) : launch_typed<float>(st, a, p);
    return ok ? "linear_int8" : nullptr;
}

}    // namespace tmi
