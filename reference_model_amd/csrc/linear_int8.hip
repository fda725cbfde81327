// The linear layer on 8-bit activations and weights, with a scale for each token and each output feature:
//
//   y[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n]
//
// The sum is exact: products of 8 bits in 32-bit integers, by the matrix instruction 16x16x64.  It becomes a 32-bit float (rounded to 24 bits), is
// multiplied by both scales, and rounded once.  Rows of x and w begin at multiples of 16 bytes and are filled up with zeros to the next one, so that
// every piece of 16 bytes goes as it lies into LDS or a matrix instruction.
//
// The weights are the first operand of the instruction and x the second, so that a lane owns neighbouring features of one token.  Out of registers alone it makes 4.9
// POP/s on zeros and 4.1 on random bits (power); 32x32x32 makes 4.9 and 3.5.
//
// linear_wide_kernel, linear_tile_kernel: many tokens.  Workgroups that stay go through a list of tiles.  Operands go straight from memory into LDS, 128 columns of
// 8 rows an instruction: whole cache lines (64 bytes of 16 rows bring 51 bytes a nanosecond and CU out of L2, 128 bytes of 8 rows 136).  They are requested a pair
// of matrix instruction depths ahead and more, across the borders of tiles: while a workgroup stores one tile's results the next one's operands are on their way.
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
// The list of tiles (times splits), and where a workgroup is in it.  Workgroups go round-robin to the 8 XCDs; each of those has a contiguous range of the
// list, along rows in groups of kGroup, which its workgroups go through side by side.
struct Item
{
    int64_t m0, n0;
    int split, block0, block1;
};
template <int BM, int BN, bool SPLIT>
struct Items
{
    int per_turn, first, last;
    __device__ __forceinline__ explicit Items(const LinearArgs& a)
    {
        per_turn = gridDim.x >> 3, first = (blockIdx.x & 7) * a.per_xcd + (blockIdx.x >> 3);
        const int of_xcd = ((int)(blockIdx.x & 7) + 1) * a.per_xcd;
        last = of_xcd < a.items ? of_xcd : a.items;
    }
    __device__ __forceinline__ Item at(const LinearArgs& a, int t) const
    {
        Item r;
        r.split        = SPLIT ? t / a.tiles : 0;
        const int tile = t - r.split * a.tiles, in_group = kGroup * a.tiles_n, group = tile / in_group, rest = tile - group * in_group;
        const int rows_here = a.tiles_m - group * kGroup < kGroup ? a.tiles_m - group * kGroup : kGroup;
        const int tn = rest / rows_here, tm = group * kGroup + rest - tn * rows_here;
        r.m0 = (int64_t)tm * BM, r.n0 = (int64_t)tn * BN;
        r.block0 = SPLIT ? r.split * a.per_split : 0;
        r.block1 = SPLIT && r.block0 + a.per_split < a.blocks ? r.block0 + a.per_split : a.blocks;
        return r;
    }
};

// For results of 16 bits row 16 c + p of 32 of a tile's weights holds feature 8 (p / 4) + 4 c + p % 4: a lane then owns eight neighbours, and four lanes 64 bytes in
// a row, as they do of 32 bits where row and feature are the same.  (Rows that differ in other bits add up.)
template <typename Out>
__device__ __forceinline__ int feature_of_row(int r)
{
    return sizeof(Out) == 4 ? r : (r & ~31) + 8 * (r >> 2 & 3) + 4 * (r >> 4 & 1) + (r & 3);
}
// 16 bytes a lane, straight into LDS: lane l's to `to` + 16 l
__device__ __forceinline__ void load_into_lds(const uint8_t* from, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(to) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const uint8_t* p)
{
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p;
}

// A lane's part of what a wave's CT x RT instruction tiles from feature n0 and token m0 on are multiplied by: asked for before their sum and used behind it (us
// asked for behind it 777 x 1111 x 2731 13.6, now 12.6; 1 x 4096 x 4096 6.7 and 6.4; 2048 x 4096 x 4096 37.5 and 36.8).
template <typename T, int CT, int RT>
struct Scales
{
    static constexpr int V = CT == 1 ? 4 : kPiece<T>, TILES = V / 4;    // (neighbours that a lane has, and column tiles that they come from)
    float of_row[RT], scale[CT * 4];
    using Bits = std::conditional_t<sizeof(T) == 4, float, uint16_t>;
    Bits bias[CT * 4];
    __device__ __forceinline__ void ask(const LinearArgs& a, int64_t n0, int64_t m0, int l16, int q4)
    {
#pragma unroll
        for (int i = 0; i < RT; i++)
        {
            const int64_t m = m0 + i * 16 + l16;
            of_row[i]       = a.x_scales[m < a.M ? m : a.M - 1];
        }
        // (no bias: other bits of that size, which are not used.  Loads in a branch would be waited for at its end)
        const Bits* from = static_cast<const Bits*>(a.bias ? a.bias : a.w_scales);
#pragma unroll
        for (int p = 0; p < CT / TILES; p++)
#pragma unroll
            for (int e = 0; e < V; e++)
            {
                const int64_t n = n0 + 16 * TILES * p + V * q4 + e, f = n < a.N ? n : a.N - 1;
                scale[p * V + e] = a.w_scales[f], bias[p * V + e] = from[f];
            }
    }
    __device__ __forceinline__ float of(const LinearArgs& a, int sum, int at, int i) const
    {
        float b;
        if constexpr (sizeof(T) == 4)
            b = bias[at];
        else
            b = from_bits16<T>(bias[at]);
        return __builtin_fmaf((float)sum * scale[at], of_row[i], a.bias ? b : 0.0f);
    }
};

// The results of those tiles: of each of a lane's rows pieces of 16 bytes
template <typename T, int CT, int RT, bool SPLIT>
__device__ __forceinline__ void store_tile(const LinearArgs& a, const v4i (&acc)[CT][RT], const Scales<T, CT, RT>& scales, int64_t n0, int64_t m0, int split, int l16,
                                           int q4)
{
    using Out       = std::conditional_t<SPLIT, float, T>;    // (a partial sum is a word, as a float is)
    constexpr int V = kPiece<Out>, TILES = V / 4;
#pragma unroll
    for (int p = 0; p < CT / TILES; p++)
    {
        const int64_t n = n0 + 16 * TILES * p + V * q4;
#pragma unroll
        for (int i = 0; i < RT; i++)
        {
            const int64_t m = m0 + i * 16 + l16;
            float y[V];
#pragma unroll
            for (int e = 0; e < V; e++)
            {
                const int sum = acc[TILES * p + e / 4][i][e & 3];
                if constexpr (SPLIT)
                    y[e] = __int_as_float(sum);
                else
                    y[e] = scales.of(a, sum, p * V + e, i);
            }
            Out* row = SPLIT ? reinterpret_cast<Out*>(a.part) + ((int64_t)split * a.M + m) * a.N : static_cast<Out*>(a.out) + m * a.ldo;
            if (m < a.M && n < a.N)
                store_piece<Out, false>(row + n, 0, (int)(a.N - n < V ? a.N - n : V), piece_of<Out>(y));
        }
    }
}

// What the waves that compute do with a pair of blocks.  A block is one matrix instruction deep; a wave takes it row tile by row tile.  When a row tile is done its
// fragment is read from the next block, a block ahead of its use, and the column tiles' fragments into a second set.  So behind the first row tile of
// a pair's second block all of the pair is read, and what `border` does there may say so.  Reads, and what `load` requests, stand behind matrix
// instructions one by one, and are kept there: their wait for a slot passes while the matrix cores work.
template <int CT, int RT>
struct Multiply
{
    static_assert(RT == 2 || RT >= CT, "where the weights' fragments are read");
    v4i acc[CT][RT], fw[2][CT], fx[RT];
    const uint8_t* lds;
    __device__ __forceinline__ void read_w(int set, uint32_t at, int c) { fw[set][c] = *reinterpret_cast<const v4i*>(lds + at + c * (16 * kPair)); }
    __device__ __forceinline__ void read_x(uint32_t at, int i) { fx[i] = *reinterpret_cast<const v4i*>(lds + at + i * (16 * kPair)); }
    __device__ __forceinline__ void first(uint32_t wat, uint32_t xat)
    {
#pragma unroll
        for (int c = 0; c < CT; c++)
            read_w(0, wat, c);
#pragma unroll
        for (int i = 0; i < RT; i++)
            read_x(xat, i);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int c = 0; c < CT; c++)
#pragma unroll
            for (int i = 0; i < RT; i++)
                acc[c][i] = v4i{ 0, 0, 0, 0 };
    }
    // Block P of a pair; wat and xat: where the next block's fragments are.  load(i): behind the second instruction of row tile i, from 1 on.
    template <int P, typename B, typename L>
    __device__ __forceinline__ void block(uint32_t wat, uint32_t xat, B&& border, L&& load)
    {
#pragma unroll
        for (int i = 0; i < RT; i++)
        {
#pragma unroll
            for (int k = 0; k < CT; k++)
            {
                const int c = i & 1 ? CT - 1 - k : k;    // (one operand changes at a time)
                acc[c][i]   = mma_int8(fw[P][c], fx[i], acc[c][i]);
                if (i > 0 && k == 1)
                    load(i);
                if (i > 0 && (RT >= CT ? k == 2 && i < CT : k >= 1))
                    read_w(1 - P, wat, RT >= CT ? i : k);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i == 0)
            {
                if constexpr (P == 1)
                    border();
                read_w(1 - P, wat, 0);
            }
            read_x(xat, i);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// 256 x 256 results, eight waves of 64 features x 128 tokens that load as well as compute.  LDS is a ring of five units: the weights of a pair, its x, the next
// pair's weights and so on.  At the barrier in the second block of pair p its units are free, and pair p + 1 has landed (all but the weights of p + 2);
// x of p + 2 goes in the place of p's weights, the weights of p + 3 in that of its x.  With the kernel below in tiles of 256 x 128
// 4096 x 4096 x 16384 took 262 us when this took 225 (half as much again of the operands' bytes), but 214 for 227 where the operands lay in the last cache.
// Operands from memory, on random bits: 239 to 250 us from run to run, 232 at the least; on zeros 201.  A dispatch is 447 thousand cycles: the matrix cores are busy 59 % of them,
// the LDS serves reads in 22 %, without conflicts; a wave waits 37 % of its time to issue anything and 3 % for LDS.  The clock falls from 2.2 GHz to 1.8 on random bits.
template <typename T>
__global__ __launch_bounds__(512, 2) void linear_wide_kernel(LinearArgs a)
{
    constexpr int CT = 4, RT = 8, B = 256, UNIT = B * kPair, RING = 5, LOADS = B * 8 / 512;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const Items<B, B, false> items(a);
    if (items.first >= items.last)
        return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wc = wave & 3, wr = wave >> 2, l16 = lane & 15, q4 = lane >> 4;

    // ---- what is requested: 16-byte piece u = j * 512 + tid of a unit, row u / 8 --------------------------------------------------
    const uint32_t lds0 = lds_address(lds) + wave * 1024;
    const int piece     = ((tid & 7) ^ swizzle(tid >> 3)) * 16;    // (64 rows are whole turns of the swizzle)
    const uint32_t woff = (uint32_t)(feature_of_row<T>(tid >> 3) * a.ldw), xoff = (uint32_t)((tid >> 3) * a.ldx);    // of this thread's first row
    // of the weights and of x: the item, its block that is requested next, where that lies, the last row's offset from there, and the unit it goes to
    struct Stream
    {
        int item, block, end, slot;
        const uint8_t* at;
        uint32_t last;
    };
    Stream ws, xs;
    auto begin = [&](auto W, int t) {
        constexpr bool IS_W = decltype(W)::value;
        Stream& s           = IS_W ? ws : xs;
        const Item it       = items.at(a, t);
        const int64_t ld = IS_W ? a.ldw : a.ldx, first = IS_W ? it.n0 : it.m0, last = (IS_W ? a.N : a.M) - 1 - first;
        s.item = t, s.block = it.block0, s.end = it.block1;
        s.at   = (IS_W ? a.w : a.x) + first * ld + it.block0 * kBlock;
        s.last = (uint32_t)((last < B - 1 ? last : B - 1) * ld);
    };
    // load j of a stream's next unit: rows past the last repeat it and are not stored; zeros where the columns end in it (without a branch: one to each side
    // of a load costs 50 to 100 cycles of a wave)
    auto request = [&](auto W, int j) {
        constexpr bool IS_W = decltype(W)::value;
        const Stream& s     = IS_W ? ws : xs;
        const uint32_t row  = IS_W ? woff + (uint32_t)(feature_of_row<T>(64 * j) * a.ldw) : xoff + (uint32_t)(64 * j * a.ldx);
        const uint32_t off  = (row < s.last ? row : s.last) + piece;
        load_into_lds(s.block * kBlock + piece < a.K ? s.at + off : a.zeros, lds0 + s.slot * UNIT + j * 8192);
    };
    // Past the last unit it is requested again, into places nobody reads: the loads in flight are then as many all the time.
    auto advance = [&](auto W) {
        Stream& s = decltype(W)::value ? ws : xs;
        s.slot    = s.slot + 2 < RING ? s.slot + 2 : s.slot + 2 - RING;
        s.block += 2, s.at += kPair;
        if (__builtin_expect(s.block >= s.end, 0))
        {
            if (s.item + items.per_turn < items.last)
                begin(W, s.item + items.per_turn);
            else
                s.block -= 2, s.at -= kPair;
        }
    };
    constexpr std::true_type of_w{};
    constexpr std::false_type of_x{};

    // ---- what a lane reads: piece q4 (and q4 + 4 in the second block) of row l16 of a tile -----------------------------------------
    const uint32_t place = (q4 ^ swizzle(l16)) * 16, waddr = (wc * 64 + l16) * kPair + place, xaddr = (wr * 128 + l16) * kPair + place;
    Multiply<CT, RT> m;
    m.lds     = lds;
    int wslot = 0, xslot = 1;    // the units of the pair in use
    auto pair = [&]() {
        auto loads = [&](auto W) {
            return [&](int i) {
#pragma unroll
                for (int j = 0; j < LOADS; j++)
                    if (1 + j * (RT - 1) / LOADS == i)
                        request(decltype(W){}, j);
            };
        };
        m.template block<0>(wslot * UNIT + (waddr ^ 64), xslot * UNIT + (xaddr ^ 64), []() {}, loads(of_w));
        advance(of_w);
        wslot = wslot + 2 < RING ? wslot + 2 : wslot + 2 - RING, xslot = xslot + 2 < RING ? xslot + 2 : xslot + 2 - RING;
        m.template block<1>(wslot * UNIT + waddr, xslot * UNIT + xaddr,
                            []() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory"); }, loads(of_x));
        advance(of_x);
    };

    begin(of_w, items.first), begin(of_x, items.first);
    ws.slot = 0, xs.slot = 1;
#pragma unroll 1
    for (int b = 0; b < 2; b++)
    {
#pragma unroll
        for (int j = 0; j < LOADS; j++)
            request(of_w, j);
#pragma unroll
        for (int j = 0; j < LOADS; j++)
            request(of_x, j);
        advance(of_w), advance(of_x);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
    m.first(waddr, UNIT + xaddr);
#pragma unroll 1
    for (int t = items.first; t < items.last; t += items.per_turn)
    {
        const Item it = items.at(a, t);
        m.clear();
#pragma unroll 1
        for (int n = it.block0; n < it.block1; n += 2)
            pair();
        Scales<T, CT, RT> scales;
        scales.ask(a, it.n0 + wc * 64, it.m0 + wr * 128, l16, q4);
        store_tile<T, CT, RT, false>(a, m.acc, scales, it.n0 + wc * 64, it.m0 + wr * 128, 0, l16, q4);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// WC x WR waves (features x tokens) that compute, of 64 features and 16 RT tokens each, and LW that load; LDS holds R pairs of blocks.  A wave that has loads to
// request waits for each of them (some 50 cycles; 110 where two share a SIMD), which those that compute need not do here, nor wait for the loads or for their own
// stores.  us with waves that do both 256 x 4096 x 4096 17.5 (now 10.6), 1024 x 4096 x 4096 23.7 (19.8), 512 x 8192 x 8192 40.8 (32.5).  Tiles of 64 with two waves
// that load and three workgroups a CU 13.4 at 256 x 4096 x 4096, one workgroup of eight pairs 11.2.  SPLIT: partial sums.
template <typename T, int WC, int WR, int RT, int LW, int R, bool SPLIT>
__global__ __launch_bounds__(64 * (WC * WR + LW), (WC * WR + LW) / 4) void linear_tile_kernel(LinearArgs a)
{
    constexpr int CT = 4, BN = 16 * CT * WC, BM = 16 * RT * WR;
    constexpr int PAIR = (BN + BM) * kPair;    // of LDS: the weights, then x
    using Out          = std::conditional_t<SPLIT, float, T>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const Items<BM, BN, SPLIT> items(a);
    if (items.first >= items.last)
        return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Barrier p (behind the first, which says that pair 0 is there) says that pair p + 1 is there and that nobody reads pair p any more.
    if (wave >= WC * WR)
    {
        // ---- waves that load: 16-byte piece u = j * 64 LW + tid of a pair, row u / 8, of the weights' rows and then of x's ------------
        constexpr int STEP = 8 * LW, WJ = BN / STEP, XJ = BM / STEP, LOADS = WJ + XJ;
        static_assert(WJ * STEP == BN && XJ * STEP == BM && STEP % 16 == 0, "all pieces of a thread have one place in their rows");
        static_assert(R >= 2 && (R - 1) * LOADS < 64, "loads in flight are counted in six bits");
        const int tid       = threadIdx.x - 64 * WC * WR, row0 = tid >> 3, piece = ((tid & 7) ^ swizzle(row0)) * 16;
        const uint32_t lds0 = lds_address(lds) + (wave - WC * WR) * 1024;
        const uint32_t woff = (uint32_t)(feature_of_row<Out>(row0) * a.ldw), xoff = (uint32_t)(row0 * a.ldx);
        // the item, its block that is requested next, where that lies, the last rows' offsets from there, and the place it goes to
        int item, block, end, slot = 0;
        const uint8_t *wat, *xat;
        uint32_t wlast, xlast;
        auto begin = [&](int t) {
            const Item it       = items.at(a, t);
            const int64_t lastw = a.N - 1 - it.n0, lastx = a.M - 1 - it.m0;
            item = t, block = it.block0, end = it.block1;
            wat = a.w + it.n0 * a.ldw + it.block0 * kBlock, xat = a.x + it.m0 * a.ldx + it.block0 * kBlock;
            wlast = (uint32_t)((lastw < BN - 1 ? lastw : BN - 1) * a.ldw), xlast = (uint32_t)((lastx < BM - 1 ? lastx : BM - 1) * a.ldx);
        };
        // (rows past the last, columns behind the last and pairs past the last as in the kernel above)
        auto request = [&]() {
            const bool inside = block * kBlock + piece < a.K;
#pragma unroll
            for (int j = 0; j < LOADS; j++)
            {
                const bool is_w    = j < WJ;
                const uint32_t row = is_w ? woff + (uint32_t)(feature_of_row<Out>(j * STEP) * a.ldw) : xoff + (uint32_t)((j - WJ) * STEP * a.ldx);
                const uint32_t off = (is_w ? (row < wlast ? row : wlast) : (row < xlast ? row : xlast)) + piece;
                load_into_lds(inside ? (is_w ? wat : xat) + off : a.zeros, lds0 + slot * PAIR + j * (STEP * kPair));
            }
            slot = slot + 1 < R ? slot + 1 : 0;
            block += 2, wat += kPair, xat += kPair;
            if (block >= end)
            {
                if (item + items.per_turn < items.last)
                    begin(item + items.per_turn);
                else
                    block -= 2, wat -= kPair, xat -= kPair;
            }
        };
        begin(items.first);
#pragma unroll 1
        for (int p = 0; p < R; p++)
            request();
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((R - 1) * LOADS) : "memory");
#pragma unroll 1
        for (int t = items.first; t < items.last; t += items.per_turn)
        {
            const Item it = items.at(a, t);
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
    const uint32_t place = (q4 ^ swizzle(l16)) * 16, waddr = (wc * 16 * CT + l16) * kPair + place, xaddr = (BN + wr * 16 * RT + l16) * kPair + place;
    Multiply<CT, RT> m;
    m.lds         = lds;
    uint32_t slot = 0;    // bytes
    auto pair     = [&]() {
        m.template block<0>(slot + (waddr ^ 64), slot + (xaddr ^ 64), []() {}, [](int) {});
        slot = slot + PAIR < R * PAIR ? slot + PAIR : 0;
        m.template block<1>(slot + waddr, slot + xaddr, []() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }, [](int) {});
    };
    asm volatile("s_barrier" ::: "memory");
    m.first(waddr, xaddr);
#pragma unroll 1
    for (int t = items.first; t < items.last; t += items.per_turn)
    {
        const Item it = items.at(a, t);
        Scales<T, CT, RT> scales;
        if constexpr (!SPLIT)
            scales.ask(a, it.n0 + wc * 16 * CT, it.m0 + wr * 16 * RT, l16, q4);
        m.clear();
#pragma unroll 1
        for (int n = it.block0; n < it.block1; n += 2)
            pair();
        store_tile<T, CT, RT, SPLIT>(a, m.acc, scales, it.n0 + wc * 16 * CT, it.m0 + wr * 16 * RT, it.split, l16, q4);
    }
}

// Results of a sum that was split into up to J parts, four of a row a thread: integers, so the order does not matter.  All parts are asked for at once (past the
// last one it again): one after the other 128 x 16384 x 1024 in eight parts took 13.3 us, now 11.6, 72 x 3646 x 201 in 15 11.1 and 7.6.
template <typename T, int J>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a)
{
    const int64_t own = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (own >= a.N)
        return;
    // (a row's last thread has its last four, some of which are its neighbour's; the buffer has room for four of a shorter row behind its end)
    const int64_t n = own + 4 <= a.N ? own : a.N >= 4 ? a.N - 4 : 0, plane = (int64_t)a.M * a.N;
    for (int64_t m = blockIdx.y; m < a.M; m += gridDim.y)
    {
        Scales<T, 1, 1> scales;
        scales.ask(a, n, m, 0, 0);
        v4i t[J], v = { 0, 0, 0, 0 };
#pragma unroll
        for (int s = 0; s < J; s++)
            __builtin_memcpy(&t[s], a.part + (s < a.splits ? s : a.splits - 1) * plane + m * a.N + n, 16);
#pragma unroll
        for (int s = 0; s < J; s++)
            if (s < a.splits)
                v += t[s];
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e >= own && n + e < a.N)
                store_one<T>(a.out, m * a.ldo + n + e, scales.of(a, v[e], e, 0));
    }
}

// RT tiles of 16 tokens against 16 features; a wave has every pair of blocks of WAVES, U pairs on their way at once.  SPLIT: partial sums.  Bound by the weights'
// bytes: 1 x 8192 x 8192 12.3 us, 5.4 TB/s; 1 x 4096 x 4096 5.6, of which 3.5 pass without any (a launch, two trips to memory, the sums' way through LDS)
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

    // (of the result that thread tid < 64 RT adds up)
    static_assert(RT <= WAVES, "a result a thread");
    const int64_t m = m0 + (wave < RT ? wave : 0) * 16 + l16, n = n0 + 4 * q4;
    Scales<T, 1, 1> scales;
    if constexpr (!SPLIT)
        scales.ask(a, n, m - l16, l16, 0);

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
    if (tid >= RT * 64)
        return;
    v4i v = met[0][tid];
#pragma unroll
    for (int k = 1; k < WAVES; k++)
        v += met[k][tid];
    if (m >= a.M)
        return;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (n + e < a.N)
        {
            if constexpr (SPLIT)
                a.part[((int64_t)blockIdx.z * a.M + m) * a.N + n + e] = v[e];
            else
                store_one<T>(a.out, m * a.ldo + n + e, scales.of(a, v[e], e, 0));
        }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

enum
{
    ROWS,        // linear_rows_kernel
    TILE_256,    // linear_wide_kernel
    TILE_BROAD,  // linear_tile_kernel: 128 tokens x 256 features, eight waves that compute and four that load
    TILE_128,    // 128 x 128, four and four
    TILE_LONG,   // 128 tokens x 64 features, four and four, two workgroups a CU
    TILE_64      // 64 x 64, two and four, two workgroups a CU
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

// What linear_rows_kernel takes, us: a CU's bytes, of x too, at 28 or 33 a nanosecond (45 where few CUs ask), or all weights out of memory, whichever is longer.  (1 x 16384 x 1024, 64
// workgroups: 11.2, split in four 7.6; 1 x 17776 x 5008, where some CUs have two: 22.5 and 18.0)
double rows_us(int64_t M, int64_t N, int blocks)
{
    const int64_t groups = tiles_of(N, 16) * tiles_of(M, 64);
    const double of_cu   = (double)tiles_of(groups, 256) * (16 + (M < 64 ? M : 64)) * blocks * 64 / (groups <= 32 ? 45e3 : M <= 16 ? 28e3 : 33e3);
    const double all     = (double)N * blocks * 64 * tiles_of(M, 64) / 6.2e6;
    return 2.0 + (of_cu > all ? of_cu : all);
}
double join_us(int64_t M, int64_t N, int splits)
{
    return splits > 1 ? 3.0 + (double)M * N * 8 * splits / 3.6e6 : 0;
}

// The kernel, and into how many parts its columns are split, with the least time by a model of each: a fixed part, and for each tile that a CU goes through its
// blocks' time and its border's.  Many tiles run at a lower clock, and share the L2s' bytes.  Of 81
// drawn sizes its choice is within 1.3 % of the best of all on average, and 17 % at most.  Measured, us rows x in_features x out_features:
//
//                         rows   tiles of 64, split in 1, 2, 4   128 x 64   128     128 x 256   256
//     16 x 4096 x 4096     6.4      9.6     9.5     9.4          11.8     13.5                 38
//     33 x 4096 x 4096     8.7     10.0     9.9    10.2          12.1     14.2                 38
//     64 x 4096 x 4096    11.9     10.0    10.0    10.5          12.3     14.4                 39
//    256 x 4096 x 4096    39.3     10.6    16.1    19.8          13.2     15.6                 41
//    512 x 4096 x 4096             16.6    24.5                  14.3     16.3                 41
//   1024 x 4096 x 4096             30.4    42.8                  23.3     20.1      25.0       43
//   1536 x 4096 x 4096             41.6    58.9                  33.6     31.8      28.2       45
//   2048 x 4096 x 4096             54.3    75.5                  44.8     36.0      34.1       47
//   4096 x 4096 x 4096            104                            84       65        62.6       57.5
//   1500 x 8192 x 8192            156                           128      100       110         89
//    300 x 1111 x 5003    17.7      8.6    18.5    20.9           7.8     10.1                 24
//   2048 x 1024 x 1024              7.9    20.5                   6.7      8.5                 17
//   1000 x 777 x 9000              23.4                          19.7     20.9                 18.2
//    300 x 16384 x 1024   65.7     27.7    20.0    19.3          37.4     42.8                141
//     64 x 4096 x 1024    11.4     10.0     9.4     8.2          10.8     14.3                 39      (rows, split in four: 7.9)
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
    const double memory = 3.6 + (double)(M + N) * blocks * 64 / 6e6;    // (tiles: no faster than their operands come)
    auto take           = [&](int kind, double us, int splits, int per) {
        if (kind != ROWS && us < memory)
            us = memory;
        us += join_us(M, N, splits);
        if (us * (splits > 1 ? 1.1 : 1.0) < least)    // (split where that is clearly less)
            least = us, p = Plan{ kind, splits, per };
    };
    auto tiles  = [&](int bm, int bn) { return tiles_of(M, bm) * tiles_of(N, bn); };
    auto per_cu = [](int64_t items) { return (double)((items + 255) / 256); };
    const int64_t t256 = tiles(256, 256), t_broad = tiles(128, 256), t128 = tiles(128, 128), t64 = tiles(64, 64);
    const double n_long = per_cu(tiles(128, 64));
    take(TILE_256, 4.0 + per_cu(t256) * (blocks * (t256 >= 200 ? 0.76 : 0.57) + 7.0), 1, blocks);
    take(TILE_BROAD, 3.6 + per_cu(t_broad) * (blocks * (t_broad >= 200 ? 0.41 : 0.3) + 3.6), 1, blocks);
    take(TILE_128, 3.6 + per_cu(t128) * (blocks * (t128 >= 200 ? 0.2 : 0.16) + 2.4), 1, blocks);
    take(TILE_LONG, 3.6 + n_long * (blocks * 0.13 + (n_long > 1 ? 1.4 : 1.0)), 1, blocks);
    for (int want = 1; want <= kMostSplits && want <= blocks / 2; want++)
    {
        const int per = (blocks / 2 + want - 1) / want * 2, splits = (blocks + per - 1) / per;
        const double n = per_cu(t64 * splits);
        take(TILE_64, 3.6 + per * (n > 1 ? 0.085 * n : 0.09) + 0.7 * n, splits, per);
        if (M <= 256 && splits > 1)
            take(ROWS, rows_us(M, N * splits, per), splits, per);
    }
    return p;
}

// `places`: workgroups that are there at once
template <auto Kernel>
bool launch_list(hipStream_t st, LinearArgs a, int bm, int bn, int threads, size_t lds, int places)
{
    if (!ensure_dynamic_lds<Kernel>(lds))
        return false;
    a.tiles_m = (a.M + bm - 1) / bm, a.tiles_n = (a.N + bn - 1) / bn, a.tiles = a.tiles_m * a.tiles_n;
    a.items = a.tiles * a.splits, a.per_xcd = (a.items + 7) / 8;
    const int grid = a.per_xcd * 8 < places ? a.per_xcd * 8 : places;
    Kernel<<<grid, threads, lds, st>>>(a);
    return true;
}
template <typename T, int WC, int WR, int RT, int LW, int R, bool SPLIT>
bool launch_tiles(hipStream_t st, const LinearArgs& a, int places)
{
    constexpr int BN = 64 * WC, BM = 16 * RT * WR;
    return launch_list<linear_tile_kernel<T, WC, WR, RT, LW, R, SPLIT>>(st, a, BM, BN, 64 * (WC * WR + LW), R * (BN + BM) * kPair, places);
}

template <int N>
constexpr std::integral_constant<int, N> number_of{};

template <typename T>
void launch_join(hipStream_t st, const LinearArgs& a)
{
    const dim3 grid((a.N + 1023) / 1024, a.M < 32768 ? a.M : 32768);
    if (a.splits > 8)
        linear_join_kernel<T, kMostSplits><<<grid, 256, 0, st>>>(a);
    else if (a.splits > 4)
        linear_join_kernel<T, 8><<<grid, 256, 0, st>>>(a);
    else if (a.splits > 1)
        linear_join_kernel<T, 4><<<grid, 256, 0, st>>>(a);
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
            // with four and eight 4.6; 1 x 8192 x 8192 14.4, 12.8 and 13.2.  With more tiles of tokens one pair and eight waves: 33 x 1111 x 5003 5.7, with two pairs
            // 7.2, with 16 waves 6.6; 24 x 4096 x 4096 8.5, 9.0 and 8.7; 48 x 4096 x 4096 11.0, 11.2 and 11.3; 64 x 4096 x 1024 in four 9.0, 10.5 and 9.2.
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
        ok = launch_list<linear_wide_kernel<T>>(st, a, 256, 256, 512, 5 * 256 * kPair, 256);
    else if (p.kind == TILE_BROAD)
        ok = launch_tiles<T, 4, 2, 4, 4, 3, false>(st, a, 256);
    else if (p.kind == TILE_128)
        ok = launch_tiles<T, 2, 2, 4, 4, 5, false>(st, a, 256);
    else if (p.kind == TILE_LONG)
        ok = launch_tiles<T, 1, 4, 2, 4, 3, false>(st, a, 512);
    else
        ok = p.splits > 1 ? launch_tiles<float, 1, 2, 2, 4, 4, true>(st, a, 512) : launch_tiles<T, 1, 2, 2, 4, 4, false>(st, a, 512);
    if (ok)
        launch_join<T>(st, a);
    return ok;
}

}    // namespace

void linear_int8_plan(const tmi_linear_int8_desc_t& d, int64_t* out3)
{
    const Plan p             = plan_of(d);
    constexpr int tokens[]   = { 0, 256, 128, 128, 128, 64 };
    constexpr int features[] = { 16, 256, 256, 128, 64, 64 };
    out3[0] = tokens[p.kind], out3[1] = features[p.kind], out3[2] = p.splits;
}

size_t linear_int8_scratch_bytes(const tmi_linear_int8_desc_t& d)
{
    const Plan p = plan_of(d);
    return p.splits > 1 ? (size_t)p.splits * d.rows * d.out_features * 4 + 16 : 0;
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
