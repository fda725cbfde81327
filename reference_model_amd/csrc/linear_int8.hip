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
// linear_tile_kernel: many tokens.  Workgroups that stay go through a list of tiles.  LDS is a ring of stages of 64 columns, filled straight from memory
// four stages ahead, across the borders of tiles: while a workgroup stores one tile's results the next one's operands are on their way.
//
// linear_rows_kernel: few tokens, bound by the weights' bytes.  A workgroup has 16 or 32 weight rows, its eight waves split the columns, operands go
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
    int32_t blocks;          // of 64 columns
    int32_t tiles_m, tiles_n, tiles;
    int32_t splits, per_split;    // blocks of a split
    int32_t items, per_xcd;       // tiles times splits
};

constexpr int kGroup = 8;    // row tiles that neighbouring workgroups share column tiles over
constexpr int kBlock = 64;   // columns of a stage
constexpr int kRing  = 5;    // stages

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

// Piece c (16 bytes) of row r of a stage lies at c ^ swizzle(r).  The LDS serves 16-byte reads of 16 lanes at once, of each half wave the quads (4 lanes)
// {0, 3, 5, 6} and then {1, 2, 4, 7}; lane l reads piece l / 16 of row l % 16.  Rows of a quad differ in r % 4, that is in which 64 of 256
// bytes they use; of the quads of a set two are of the first piece and two of the second, and 0, 3, 2, 1 for the rows' r / 4 keeps all four apart.
__device__ __forceinline__ int swizzle(int r)
{
    const int q = (r >> 2) & 3;
    return (q ^ (q << 1)) & 3;
}
// a pointer that is the same in every lane, where the compiler does not see it
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p)
{
    const uint64_t v  = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
}

// WC x WR waves (features x tokens) of 64 features and 16 RT tokens each; SPLIT: partial sums
template <typename T, int WC, int WR, int RT, bool SPLIT>
__global__ __launch_bounds__(64 * WC * WR, 2) void linear_tile_kernel(LinearArgs a)
{
    constexpr int THREADS = 64 * WC * WR;
    constexpr int BN = 64 * WC, BM = 16 * RT * WR, CT = 4;
    constexpr int CB = BN * kBlock, STAGE = (BN + BM) * kBlock;
    constexpr int CL = BN * 4 / THREADS, RL = BM * 4 / THREADS, LOADS = CL + RL;    // 16-byte loads of a thread and block
    static_assert(CL * THREADS == BN * 4 && RL * THREADS == BM * 4 && (RT == 2 || RT >= CT), "a block must split evenly over the threads");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wc = wave % WC, wr = wave / WC;
    const int l16 = lane & 15, q4 = lane >> 4;

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

    // ---- what is requested: 16-byte unit u = j * THREADS + tid of either operand's part of a stage -----------------------------
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * 1024;
    uint32_t woff[CL], xoff[RL];    // from the running addresses
    const uint8_t *wat, *xat;
    int ahead_item = first_item, ahead, ahead_end, astage = 0;    // the block requested next, and its stage
    auto piece_of_unit = [&](int u) { return ((u & 3) ^ swizzle(u >> 2)) * 16; };
    // Rows past the last repeat it and are not stored.  Row 16 c + p of 64 holds feature 16 (p / 4) + 4 c + p % 4, so that a lane owns 16 neighbours.
    auto request_item = [&](int t) {
        const Item it = item_of(t);
#pragma unroll
        for (int j = 0; j < CL; j++)
        {
            const int u = j * THREADS + tid, r = u >> 2;
            const int64_t f = (r & ~63) + 16 * (r >> 2 & 3) + 4 * (r >> 4 & 3) + (r & 3), last = a.N - 1 - it.n0;
            woff[j] = (uint32_t)((f < last ? f : last) * a.ldw) + piece_of_unit(u);
        }
#pragma unroll
        for (int j = 0; j < RL; j++)
        {
            const int u = j * THREADS + tid;
            const int64_t r = u >> 2, last = a.M - 1 - it.m0;
            xoff[j] = (uint32_t)((r < last ? r : last) * a.ldx) + piece_of_unit(u);
        }
        ahead = it.block0, ahead_end = it.block1;
        wat = a.w + it.n0 * a.ldw + it.block0 * kBlock, xat = a.x + it.m0 * a.ldx + it.block0 * kBlock;
    };
    // load q of the block `ahead`; EDGE: the columns end in it, and zeros come from there on
    auto request = [&](int q, auto EDGE) {
        const bool is_w      = q < CL;
        const int j          = is_w ? q : q - CL;
        const uint32_t dst   = lds0 + astage * STAGE + (is_w ? 0 : CB) + j * THREADS * 16;
        const uint8_t* base  = is_w ? wat : xat;
        const uint32_t voff  = is_w ? woff[j] : xoff[j];
        if constexpr (decltype(EDGE)::value)
        {
            const bool inside  = ahead * kBlock + piece_of_unit(j * THREADS + tid) < a.K;
            const uint8_t* src = inside ? base + voff : a.zeros;
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(dst) : "memory");
        }
        else
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(uniform(base)), "s"(dst) : "memory");
    };
    // Past the last block it is requested again, into stages nobody reads: the loads in flight are then as many in every block.
    auto advance = [&]() {
        astage = astage + 1 < kRing ? astage + 1 : 0;
        if (++ahead < ahead_end)
            wat += kBlock, xat += kBlock;
        else if (ahead_item + per_turn < last_item)
            ahead_item += per_turn, request_item(ahead_item);
        else
            ahead = ahead_end - 1;
    };
    auto whole = [&]() { return (ahead + 1) * kBlock <= a.K; };

    // ---- what a lane reads: piece q4 of row l16 of a tile -------------------------------------------------------------------------
    const uint32_t waddr = (wc * 64 + l16) * 64 + ((q4 ^ swizzle(l16)) * 16), xaddr = CB + (wr * 16 * RT + l16) * 64 + ((q4 ^ swizzle(l16)) * 16);
    v4i acc[CT][RT];
    v4i fw[2][CT], fx[RT];
    auto read_w = [&](int set, const uint8_t* sb, int c) { fw[set][c] = *reinterpret_cast<const v4i*>(sb + waddr + c * 1024); };
    auto read_x = [&](const uint8_t* sb, int i) { fx[i] = *reinterpret_cast<const v4i*>(sb + xaddr + i * 1024); };

    // A block is one matrix instruction deep.  A wave takes it row tile by row tile; when a row tile is done its fragment is read from the next
    // block, a block ahead of its use, and the column tiles' fragments into a second set.  The barrier that publishes block n + 1 stands behind
    // the first row tile of block n; past it every wave is done with block n - 1, whose stage takes the loads of block n + 4.  Reads and
    // loads stand behind matrix instructions one by one, and are kept there: their wait for a slot passes while the matrix cores work.
    int cur = 0;
    auto one_block = [&](auto SET) {
        constexpr int P     = decltype(SET)::value;
        cur                 = cur + 1 < kRing ? cur + 1 : 0;
        const uint8_t* next = lds + cur * STAGE;
        const bool w        = whole();
#pragma unroll
        for (int i = 0; i < RT; i++)
        {
#pragma unroll
            for (int k = 0; k < CT; k++)
            {
                const int c = i & 1 ? CT - 1 - k : k;    // (one operand changes at a time)
                acc[c][i]   = mma_int8(fw[P][c], fx[i], acc[c][i]);
                if (i > 0 && k == 1)
#pragma unroll
                    for (int q = 0; q < LOADS; q++)
                        if (1 + q * (RT - 1) / LOADS == i)
                        {
                            if (w)
                                request(q, std::false_type());
                            else
                                request(q, std::true_type());
                        }
                if (i > 0 && (RT >= CT ? k == 2 && i < CT : k >= 1))
                    read_w(1 - P, next, RT >= CT ? i : k);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i == 0)
            {
                // (a bare barrier: the reads in flight are of the block in use)
                asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((kRing - 3) * LOADS) : "memory");
                read_w(1 - P, next, 0);
            }
            read_x(next, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        advance();
    };

    request_item(first_item);
#pragma unroll 1
    for (int b = 0; b < kRing - 1; b++)
    {
        if (whole())
#pragma unroll
            for (int q = 0; q < LOADS; q++)
                request(q, std::false_type());
        else
#pragma unroll
            for (int q = 0; q < LOADS; q++)
                request(q, std::true_type());
        advance();
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((kRing - 2) * LOADS) : "memory");
#pragma unroll
    for (int c = 0; c < CT; c++)
        read_w(0, lds, c);
#pragma unroll
    for (int i = 0; i < RT; i++)
        read_x(lds, i);
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
        int n = it.block0;
#pragma unroll 1
        for (; n + 1 < it.block1; n += 2)
        {
            one_block(std::integral_constant<int, 0>());
            one_block(std::integral_constant<int, 1>());
        }
        if (n < it.block1)
        {
            one_block(std::integral_constant<int, 0>());
#pragma unroll
            for (int c = 0; c < CT; c++)
                fw[0][c] = fw[1][c];
        }

        // ---- results: 16 neighbours of each of a lane's rows ------------------------------------------------------------------
        const int64_t n0 = it.n0 + wc * 64 + 16 * q4;
        float ws[16], bs[16];
        if constexpr (!SPLIT)
#pragma unroll
            for (int e = 0; e < 16; e++)
            {
                const int64_t f = n0 + e < a.N ? n0 + e : a.N - 1;
                ws[e] = a.w_scales[f], bs[e] = a.bias ? bias_at<T>(a.bias, f) : 0.0f;
            }
#pragma unroll
        for (int i = 0; i < RT; i++)
        {
            const int64_t m = it.m0 + (wr * RT + i) * 16 + l16;
            if (m >= a.M)
                continue;
            using Out = std::conditional_t<SPLIT, float, T>;    // (a partial sum is a word, as a float is)
            float y[16];
#pragma unroll
            for (int e = 0; e < 16; e++)
                y[e] = SPLIT ? __int_as_float(acc[e >> 2][i][e & 3]) : 0.0f;
            if constexpr (!SPLIT)
            {
                const float xs = a.x_scales[m];
#pragma unroll
                for (int e = 0; e < 16; e++)
                    y[e] = __builtin_fmaf((float)acc[e >> 2][i][e & 3] * ws[e], xs, bs[e]);
            }
            Out* row = SPLIT ? reinterpret_cast<Out*>(a.part) + ((int64_t)it.split * a.M + m) * a.N : static_cast<Out*>(a.out) + m * a.ldo;
#pragma unroll
            for (int p = 0; p < 16 / kPiece<Out>; p++)
                store_piece<Out, false>(row + n0, p * kPiece<Out>, (int)(a.N - n0 < 16 ? a.N - n0 : 16), piece_of<Out>(y + p * kPiece<Out>));
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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

// RT tiles of 16 tokens, CT of 16 features; a wave has every eighth pair of blocks, U pairs on their way at once
template <typename T, int RT, int CT, int U>
__global__ __launch_bounds__(512) void linear_rows_kernel(LinearArgs a)
{
    constexpr int WAVES = 8;
    __shared__ v4i met[WAVES][CT * RT * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, q4 = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * CT), m0 = (int64_t)blockIdx.y * (16 * RT);

    const uint8_t *w[CT], *x[RT];    // rows past the last repeat it
#pragma unroll
    for (int c = 0; c < CT; c++)
    {
        const int64_t n = n0 + c * 16 + l16;
        w[c]            = a.w + (n < a.N ? n : a.N - 1) * a.ldw;
    }
#pragma unroll
    for (int i = 0; i < RT; i++)
    {
        const int64_t m = m0 + i * 16 + l16;
        x[i]            = a.x + (m < a.M ? m : a.M - 1) * a.ldx;
    }
    v4i acc[CT][RT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int i = 0; i < RT; i++)
            acc[c][i] = v4i{ 0, 0, 0, 0 };

    const int pairs = (a.K + 127) / 128;
#pragma unroll 1
    for (int p = wave; p < pairs; p += WAVES * U)
    {
        v4i fw[U * 2][CT], fx[U * 2][RT];
        bool inside[U * 2];
#pragma unroll
        for (int u = 0; u < U * 2; u++)
        {
            const int k = (p + (u >> 1) * WAVES) * 128 + (u & 1) * 64 + q4 * 16;
            inside[u]   = k < a.K;
            const int at = inside[u] ? k : 0;
#pragma unroll
            for (int c = 0; c < CT; c++)
                fw[u][c] = *reinterpret_cast<const v4i*>(w[c] + at);
#pragma unroll
            for (int i = 0; i < RT; i++)
                fx[u][i] = *reinterpret_cast<const v4i*>(x[i] + at);
        }
#pragma unroll
        for (int u = 0; u < U * 2; u++)
#pragma unroll
            for (int c = 0; c < CT; c++)
            {
                const v4i f = inside[u] ? fw[u][c] : v4i{ 0, 0, 0, 0 };
#pragma unroll
                for (int i = 0; i < RT; i++)
                    acc[c][i] = mma_int8(f, fx[u][i], acc[c][i]);
            }
    }
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int i = 0; i < RT; i++)
            met[wave][(c * RT + i) * 64 + lane] = acc[c][i];
    __syncthreads();
#pragma unroll
    for (int u = tid; u < CT * RT * 64; u += 64 * WAVES)
    {
        v4i v = met[0][u];
#pragma unroll
        for (int k = 1; k < WAVES; k++)
            v += met[k][u];
        const int l = u & 63, tile = u >> 6;
        const int64_t m = m0 + (tile % RT) * 16 + (l & 15), n = n0 + (tile / RT) * 16 + 4 * (l >> 4);
        if (m >= a.M)
            continue;
        const float xs = a.x_scales[m];
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < a.N)
                store_one<T>(a.out, m * a.ldo + n + e, __builtin_fmaf((float)v[e] * a.w_scales[n + e], xs, a.bias ? bias_at<T>(a.bias, n + e) : 0.0f));
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

enum
{
    ROWS,        // linear_rows_kernel
    TILE_256,    // 256 x 256 results, eight waves
    TILE_128     // 128 x 128, eight waves, two workgroups a CU
};
struct Plan
{
    int kind;
    int splits, per_split;
};
constexpr int kMostSplits = 16, kLeastBlocks = 8;

Plan plan_of(const tmi_linear_int8_desc_t& d)
{
    Plan p{};
    const int blocks = (int)((whole16(d.in_features) + kBlock - 1) / kBlock);
    p.splits = 1, p.per_split = blocks;
    // (a lane's offset over a tile is held in 32 bits)
    const bool far = d.ld_x >= (int64_t(1) << 23) || d.ld_w >= (int64_t(1) << 23);
    if (d.rows <= 64 || far || blocks == 0)
    {
        p.kind = ROWS;
        return p;
    }
    const int64_t big = (((int64_t)d.rows + 255) / 256) * (((int64_t)d.out_features + 255) / 256);
    p.kind            = big >= 200 ? TILE_256 : TILE_128;
    if (p.kind == TILE_128)
    {
        const int64_t tiles = (((int64_t)d.rows + 127) / 128) * (((int64_t)d.out_features + 127) / 128);
        int want            = (int)(512 / tiles);
        want = want > kMostSplits ? kMostSplits : want;
        want = want > blocks / kLeastBlocks ? blocks / kLeastBlocks : want;
        if (want > 1)
        {
            p.per_split = (blocks + want - 1) / want;
            p.splits    = (blocks + p.per_split - 1) / p.per_split;
        }
    }
    return p;
}

template <typename T, int WC, int WR, int RT, bool SPLIT>
bool launch_tiles(hipStream_t st, LinearArgs a, int places)
{
    constexpr size_t lds = kRing * (64 * WC + 16 * RT * WR) * kBlock;
    constexpr auto kernel = linear_tile_kernel<T, WC, WR, RT, SPLIT>;
    if (!ensure_dynamic_lds<kernel>(lds))
        return false;
    a.tiles_m = (a.M + 16 * RT * WR - 1) / (16 * RT * WR), a.tiles_n = (a.N + 64 * WC - 1) / (64 * WC), a.tiles = a.tiles_m * a.tiles_n;
    a.items = a.tiles * a.splits, a.per_xcd = (a.items + 7) / 8;
    const int grid = a.per_xcd * 8 < places ? a.per_xcd * 8 : places;
    kernel<<<grid, 64 * WC * WR, lds, st>>>(a);
    return true;
}

template <typename T>
bool launch_typed(hipStream_t st, const LinearArgs& a, const Plan& p)
{
    if (p.kind == ROWS)
    {
        auto go = [&](auto kernel, int rt, int ct) { kernel<<<dim3((a.N + 16 * ct - 1) / (16 * ct), (a.M + 16 * rt - 1) / (16 * rt)), 512, 0, st>>>(a); };
        if (a.M <= 16)
            go(linear_rows_kernel<T, 1, 1, 4>, 1, 1);
        else if (a.M <= 32)
            go(linear_rows_kernel<T, 2, 1, 2>, 2, 1);
        else
            go(linear_rows_kernel<T, 4, 1, 2>, 4, 1);
        return true;
    }
    bool ok;
    if (p.kind == TILE_256)
        ok = launch_tiles<T, 4, 2, 8, false>(st, a, 256);
    else if (p.splits > 1)
        ok = launch_tiles<float, 2, 4, 2, true>(st, a, 512);
    else
        ok = launch_tiles<T, 2, 4, 2, false>(st, a, 512);
    if (ok && p.splits > 1)
        linear_join_kernel<T><<<dim3((a.N + 1023) / 1024, a.M < 32768 ? a.M : 32768), 256, 0, st>>>(a);
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
    const int blocks = (int)((whole16(d.in_features) + kBlock - 1) / kBlock);
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
