// The gated feed-forward block on many rows, and its gradients, on the matrix cores:
//
//   forward    h[m][f]  = act(sum_d x[m][d] gate[f][d]) * (sum_d x[m][d] up[f][d])
//   slopes     dp[m]    = [ dh u act'(g) | dh act(g) ], 2 FP elements, FP = F up to whole blocks of 64, zeros behind F
//   d_x        dx[m][d] = sum_f dp[m][f] gate[f][d] + dp[m][FP + f] up[f][d]
//   d_w        dw[f][d] = sum_m dp[m][f] x[m][d], f over gate and up
//
// One kernel makes all three products.  The operand whose index runs along an output row ("columns": weights, weights, x) is the first of the
// 16x16x32 matrix instruction, so that a lane owns four neighbouring results of one row; the other ("rows": x, dp, dp) is the second.  (32x32x16
// does as many operations a clock, but takes more power for them: 1.82 PFLOP/s on random bf16 numbers and nothing else, against 2.03.)  An operand
// lies in memory with the summed index innermost (forward: both; d_x: dp) or outermost (d_x: the weights; d_w: both).  Either way 16-byte pieces
// go to LDS as they lie; an outermost one comes out through the transposing reads ds_read_b64_tr_b16.  So nothing is transposed in memory.
//
// The forward pass deals gate and up rows of the same 32 features to one wave as its four column tiles: activation and product are done on the
// accumulators, and the pre-activations leave the chip only if they are asked for.
//
// LDS is a ring of stages of 32 of the summed index (96 KB of operands in flight behind the one in use at 256 x 256).  Innermost: rows of 64
// bytes, their 16-byte pieces permuted by the row.  Outermost: 32 rows of the tile's width, their 32-byte segments permuted by the row.  Both keep
// the 16 (32) lanes that the LDS serves at once on banks of their own.  Pieces that are whole go from global memory straight into LDS; where
// rows begin at any element or end inside a piece they go through registers, two blocks ahead.
#include "tmi_ffn.h"

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
    const float* unit;         // gradients in fp16: what dp is held in units of
    int64_t ldc, ldr, ldo;     // elements
    int32_t M, N;              // results: rows and columns (features of h; d; d)
    int32_t K;                 // summed index (of one half, for d_x)
    int32_t width;             // elements of a row of an outermost columns operand: N, or of its copy
    int32_t half;              // FP, the columns of each half of dp
    int32_t features;          // F
    int32_t blocks;            // of 32 of the summed index
    int32_t tiles_m, tiles_n, tiles, per_xcd;
    int32_t splits, per_split; // blocks of a split
    int32_t act;
};

// Innermost: piece c of row r lies at c ^ swizzle_in(r).  The LDS serves 16-byte reads of 16 lanes at once, of each half wave the quads (4 lanes)
// {0, 3, 5, 6} and then {1, 2, 4, 7}; lane l reads piece l / 16 of row l % 16.  Rows of a quad differ in r % 4, that is in which 64 of 256
// bytes they use; of the quads of a set two are of the first piece and two of the second, and 0, 3, 2, 1 for the rows' r / 4 keeps all four apart.
__device__ __forceinline__ int swizzle_in(int r)
{
    const int q = (r >> 2) & 3;
    return (q ^ (q << 1)) & 3;
}
// Outermost: 32-byte segment c of row k lies at c ^ swizzle_out(k).  A transposing read serves 32 lanes at once: 32 bytes of the rows k % 8 = 0 ... 3
// (or 4 ... 7) of two neighbouring eights.
__device__ __forceinline__ int swizzle_out(int k)
{
    return (k & 3) | (k >> 1 & 4);
}

// whether dp of this type is held in units of a power of two (gated_slope_kernel)
template <typename T>
constexpr bool kInUnits = !__is_same(T, bf16_t);

constexpr int kGroup = 8;    // row tiles that neighbouring workgroups share column tiles over
constexpr int kBlock = 32;   // of the summed index

// stages of the ring: all of the LDS for one workgroup of eight waves or two of four; through registers, what that needs
template <bool DIRECT>
constexpr int kRing = DIRECT ? 5 : 4;

// a pointer that is the same in every lane, where the compiler does not see it
__device__ __forceinline__ const uint16_t* uniform(const uint16_t* p)
{
    const uint64_t v  = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const uint16_t*>((uint64_t)hi << 32 | lo);
}

// WC x WR waves (columns x rows) of 64 columns and 16 RT rows each
template <typename T, int OP, int WC, int WR, int RT, bool DIRECT>
__device__ __forceinline__ void gated_gemm(const GemmFfnArgs& a, int workgroup)
{
    constexpr int THREADS = 64 * WC * WR;
    constexpr int BN = 64 * WC, BM = 16 * RT * WR;
    constexpr int CT = 4;    // column tiles of a wave (forward: gate, gate, up, up)
    constexpr bool CIN = OP == OP_FORWARD;    // summed index innermost: columns operand
    constexpr bool RIN = OP != OP_DW;         // rows operand
    constexpr int CB = BN * 64, STAGE = (BN + BM) * 64, RING = kRing<DIRECT>;
    constexpr int CL = BN * 4 / THREADS, RL = BM * 4 / THREADS, LOADS = CL + RL;    // 16-byte loads of a thread and block
    constexpr int TN = CIN ? BN / 2 : BN;                                            // results a tile's columns make
    static_assert(CL * THREADS == BN * 4 && RL * THREADS == BM * 4 && (RT == 2 || RT >= CT), "a block must split evenly over the threads");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wc = wave % WC, wr = wave / WC;
    const int l16 = lane & 15, q4 = lane >> 4;

    // workgroups go round-robin to the 8 XCDs; each takes a contiguous range of the tile list, along rows in groups of kGroup
    const int t = (workgroup & 7) * a.per_xcd + (workgroup >> 3);
    if (t >= a.tiles * a.splits)
        return;
    const int split = t / a.tiles, tile = t - split * a.tiles;
    const int in_group = kGroup * a.tiles_n, group = tile / in_group, rest = tile - group * in_group;
    const int rows_here = a.tiles_m - group * kGroup < kGroup ? a.tiles_m - group * kGroup : kGroup;
    const int tn = rest / rows_here, tm = group * kGroup + rest - tn * rows_here;
    const int64_t n0 = (int64_t)tn * TN, m0 = (int64_t)tm * BM;
    const int block0 = split * a.per_split;
    const int block1 = block0 + a.per_split < a.blocks ? block0 + a.per_split : a.blocks;
    const int second = OP == OP_DX ? a.half / kBlock : INT32_MAX;    // first block of the second half
    auto block_k = [&](int n) { return (n >= second ? n - second : n) * kBlock; };    // its first index, within its half

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
            const int r     = u >> 2;
            const int64_t f = n0 + (r >> 6) * 32 + (r & 31);    // rows 0..31 of 64 are gate's, the others up's
            return Unit{ f < a.N ? f : a.N - 1, ((u & 3) ^ swizzle_in(r)) * 8 };
        }
        else
        {
            const int k = u / (BN / 8);
            return Unit{ k, ((u % (BN / 8)) ^ (swizzle_out(k) << 1)) * 8 };
        }
    };
    auto row_unit = [&](int j) {
        const int u = j * THREADS + tid;
        if constexpr (RIN)
        {
            const int r     = u >> 2;
            const int64_t m = m0 + r;
            return Unit{ m < a.M ? m : a.M - 1, ((u & 3) ^ swizzle_in(r)) * 8 };
        }
        else
        {
            const int k = u / (BM / 8);
            return Unit{ k, ((u % (BM / 8)) ^ (swizzle_out(k) << 1)) * 8 };
        }
    };
    // the column operand of load j of this wave (forward), or of block n (d_x)
    auto col_base = [&](int j, int n) { return CIN ? a.col[(j * THREADS + wave * 64) >> 7 & 1] : a.col[n >= second ? 1 : 0]; };

    // DIRECT: running addresses of the block to be requested next, and the thread's offsets from them
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * 1024;
    uint32_t cvoff[DIRECT ? CL : 1], rvoff[DIRECT ? RL : 1];
    const uint16_t *cat[DIRECT ? (CIN ? CL : 1) : 1], *rat = nullptr;
    int ahead = block0, astage = 0;    // the block, and the stage it goes to
    if constexpr (DIRECT)
    {
#pragma unroll
        for (int j = 0; j < CL; j++)
        {
            const Unit u = col_unit(j);
            if constexpr (CIN)
                cvoff[j] = (uint32_t)((u.row - n0) * a.ldc + u.col) * 2;
            else    // pieces past the row's end repeat the last one; never stored
                cvoff[j] = (uint32_t)(u.row * a.ldc + (u.col < a.width - 8 - n0 ? u.col : a.width - 8 - n0)) * 2;
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
#pragma unroll
        for (int j = 0; j < (CIN ? CL : 1); j++)
            cat[j] = col_base(j, block0) + (CIN ? n0 * a.ldc + block0 * kBlock : (int64_t)block_k(block0) * a.ldc + n0);
        rat = a.row + (RIN ? m0 * a.ldr + block0 * kBlock : (int64_t)block0 * kBlock * a.ldr + m0);
    }
    // load q of the block `ahead`; EDGE: the summed index ends in it, and zeros come from there on (dp holds its own)
    auto request = [&](int q, auto EDGE) {
        const bool is_c      = q < CL;
        const int j          = is_c ? q : q - CL;
        const uint32_t dst   = lds0 + astage * STAGE + (is_c ? 0 : CB) + j * THREADS * 16;
        const uint16_t* base = is_c ? cat[CIN ? j : 0] : rat;
        const uint32_t voff  = is_c ? cvoff[j] : rvoff[j];
        if constexpr (decltype(EDGE)::value)
        {
            if (is_c || OP != OP_DX)
            {
                const Unit u       = is_c ? col_unit(j) : row_unit(j);
                const bool inside  = block_k(ahead) + ((is_c ? CIN : RIN) ? u.col : (int)u.row) < a.K;
                const uint8_t* src = inside ? reinterpret_cast<const uint8_t*>(base) + voff : a.zeros;
                asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(dst) : "memory");
                return;
            }
        }
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(uniform(base)), "s"(dst) : "memory");
    };
    // Past the last block it is requested again, into stages nobody reads: the loads in flight are then as many in every block.
    auto advance = [&]() {
        astage = astage + 1 < RING ? astage + 1 : 0;
        if (++ahead < block1)
        {
#pragma unroll
            for (int j = 0; j < (CIN ? CL : 1); j++)
                cat[j] += CIN ? kBlock : kBlock * a.ldc;
            if (OP == OP_DX && ahead == second)
                cat[0] = a.col[1] + n0;
            rat += RIN ? kBlock : kBlock * a.ldr;
        }
        else
            ahead = block1 - 1;
    };

    // Otherwise through registers, in two sets
    v4i creg[DIRECT ? 1 : 2][DIRECT ? 1 : CL], rreg[DIRECT ? 1 : 2][DIRECT ? 1 : RL];
    // Pieces that their rows end in, and rows that are none, are put right on their way into LDS, when they are there; a block whose pieces all lie
    // inside needs no look at them.
    const bool inner = (CIN || n0 + BN <= a.width) && (RIN || m0 + BM <= a.M);
    struct Piece
    {
        const uint16_t* row;
        int64_t at, end;
        bool inside;
    };
    auto col_piece = [&](int j, int n) {
        const Unit u      = col_unit(j);
        const int k0      = block_k(n);
        const bool inside = CIN || k0 + u.row < a.K;
        return Piece{ col_base(j, n) + (CIN ? u.row : inside ? k0 + u.row : a.K - 1) * a.ldc, CIN ? k0 + u.col : n0 + u.col, CIN ? a.K : a.width, inside };
    };
    auto row_piece = [&](int j, int n) {
        const Unit u      = row_unit(j);
        const int k0      = block_k(n);
        const bool inside = RIN || k0 + u.row < a.K;
        return Piece{ a.row + (RIN ? u.row : inside ? k0 + u.row : a.K - 1) * a.ldr, OP == OP_DX ? n * kBlock + u.col : RIN ? k0 + u.col : m0 + u.col,
                      OP == OP_DX ? a.ldr : RIN ? a.K : a.M, inside };
    };
    auto fetch = [&](auto SET, int n) {
        constexpr int P = decltype(SET)::value;
#pragma unroll
        for (int j = 0; j < CL; j++)
        {
            const Piece p = col_piece(j, n);
            creg[P][j]    = load8_raw(p.row, p.at, p.end);
        }
#pragma unroll
        for (int j = 0; j < RL; j++)
        {
            const Piece p = row_piece(j, n);
            rreg[P][j]    = load8_raw(p.row, p.at, p.end);
        }
    };
    auto put = [&](auto SET, int n, int stage) {
        constexpr int P = decltype(SET)::value;
        if (!(inner && block_k(n) + kBlock <= a.K))
        {
#pragma unroll
            for (int j = 0; j < CL; j++)
            {
                const Piece p = col_piece(j, n);
                creg[P][j]    = settle8(creg[P][j], p.at, p.end, p.inside);
            }
#pragma unroll
            for (int j = 0; j < RL; j++)
                if (OP != OP_DX)
                {
                    const Piece p = row_piece(j, n);
                    rreg[P][j]    = settle8(rreg[P][j], p.at, p.end, p.inside);
                }
        }
        uint8_t* to = lds + stage * STAGE + tid * 16;
#pragma unroll
        for (int j = 0; j < CL; j++)
            *reinterpret_cast<v4i*>(to + j * THREADS * 16) = creg[P][j];
#pragma unroll
        for (int j = 0; j < RL; j++)
            *reinterpret_cast<v4i*>(to + CB + j * THREADS * 16) = rreg[P][j];
    };

    // ---- what a lane reads --------------------------------------------------------------------------------------------------
    // innermost: piece q4 of row l16 of a tile; outermost: as source lane, four columns of row l16 / 4 of the first four of the eight rows q4
    uint32_t caddr[CIN ? 1 : CT], raddr[RIN ? 1 : RT];    // (outermost: by tile)
    const int k8 = 8 * q4 + (l16 >> 2), seg = swizzle_out(k8);
    if constexpr (CIN)
        caddr[0] = (wc * 64 + l16) * 64 + ((q4 ^ swizzle_in(l16)) * 16);
    else
#pragma unroll
        for (int c = 0; c < CT; c++)
            caddr[c] = k8 * (BN * 2) + (((wc * CT + c) ^ seg) << 5) + 8 * (l16 & 3);
    if constexpr (RIN)
        raddr[0] = CB + (wr * 16 * RT + l16) * 64 + ((q4 ^ swizzle_in(l16)) * 16);
    else
#pragma unroll
        for (int i = 0; i < RT; i++)
            raddr[i] = CB + k8 * (BM * 2) + (((wr * RT + i) ^ seg) << 5) + 8 * (l16 & 3);
    auto transposed = [&](const uint8_t* at, int rows_apart) {
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
        const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + rows_apart)));
        return v4i{ lo.x, lo.y, hi.x, hi.y };
    };

    v4f acc[CT][RT];
#pragma unroll
    for (int c = 0; c < CT; c++)
#pragma unroll
        for (int i = 0; i < RT; i++)
            acc[c][i] = v4f{ 0.0f, 0.0f, 0.0f, 0.0f };

    // ---- main loop ------------------------------------------------------------------------------------------------------------
    // A block is one matrix instruction deep.  A wave takes it row tile by row tile; when a row tile is done its fragment is read from the next
    // block, a block ahead of its use, and the column tiles' fragments into a second set.  The barrier that publishes block n + 1 stands behind
    // the first row tile of block n; past it every wave is done with block n - 1, whose stage takes the loads of block n + RING - 1.  Reads and
    // loads stand behind matrix instructions one by one, and are kept there: their wait for a slot passes while the matrix cores work.
    v4i fc[2][CT], fr[RT];
    auto read_col = [&](int set, const uint8_t* sb, int c) {
        if constexpr (CIN)
            fc[set][c] = *reinterpret_cast<const v4i*>(sb + caddr[0] + c * 1024);
        else
            fc[set][c] = transposed(sb + caddr[c], 4 * (BN * 2));
    };
    auto read_row = [&](const uint8_t* sb, int i) {
        if constexpr (RIN)
            fr[i] = *reinterpret_cast<const v4i*>(sb + raddr[0] + i * 1024);
        else
            fr[i] = transposed(sb + raddr[i], 4 * (BM * 2));
    };
    // a block whose column fragments are in set P, with the reads of the next one from `next`; publish() behind the first row tile, and NL loads
    auto block = [&](auto SET, const uint8_t* next, auto&& publish, auto NL_tag, auto&& load) {
        constexpr int P = decltype(SET)::value, NL = decltype(NL_tag)::value;
#pragma unroll
        for (int i = 0; i < RT; i++)
        {
#pragma unroll
            for (int k = 0; k < CT; k++)
            {
                const int c = i & 1 ? CT - 1 - k : k;    // (one operand changes at a time)
                acc[c][i]   = mma16<T>(fc[P][c], fr[i], acc[c][i]);
                if (i > 0 && k == 1)
#pragma unroll
                    for (int q = 0; q < NL; q++)
                        if (1 + q * (RT - 1) / (NL ? NL : 1) == i)
                            load(q);
                if (i > 0 && (RT >= CT ? k == 2 && i < CT : k >= 1))
                    read_col(1 - P, next, RT >= CT ? i : k);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i == 0)
            {
                publish();
                read_col(1 - P, next, 0);
            }
            read_row(next, i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto first_reads = [&]() {
#pragma unroll
        for (int c = 0; c < CT; c++)
            read_col(0, lds, c);
#pragma unroll
        for (int i = 0; i < RT; i++)
            read_row(lds, i);
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr std::integral_constant<int, 0> zero{};
    constexpr std::integral_constant<int, 1> one{};
    auto next_of = [&](int s) { return s + 1 < RING ? s + 1 : 0; };

    if (block0 < block1)
    {
        int cur = 0;
        if constexpr (DIRECT)
        {
            auto whole = [&]() { return block_k(ahead) + kBlock <= a.K; };
#pragma unroll 1
            for (int b = 0; b < RING - 1; b++)
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
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((RING - 2) * LOADS) : "memory");
            first_reads();
            auto one_block = [&](auto SET) {
                cur          = next_of(cur);
                const bool w = whole();
                // (a bare barrier: the reads in flight are of the block in use)
                auto publish = [&]() { asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((RING - 3) * LOADS) : "memory"); };
                block(SET, lds + cur * STAGE, publish, std::integral_constant<int, LOADS>(), [&](int q) {
                    if (w)
                        request(q, std::false_type());
                    else
                        request(q, std::true_type());
                });
                advance();
            };
#pragma unroll 1
            for (int n = block0; n < block1; n += 2)
            {
                one_block(zero);
                if (n + 1 < block1)
                    one_block(one);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        else
        {
            // Blocks 0 and 1 in LDS, 2 and 3 in the registers; behind its barrier a block n writes block n + 2, and fetches n + 4.  Past the last block
            // that one is fetched again, so that no branch stands between the loads and the count of those to wait for.
            auto last = [&](int n) { return n < block1 ? n : block1 - 1; };
            fetch(zero, block0);
            fetch(one, last(block0 + 1));
            put(zero, block0, 0);
            put(one, last(block0 + 1), 1);
            fetch(zero, last(block0 + 2));
            fetch(one, last(block0 + 3));
            __syncthreads();
            first_reads();
            auto one_block = [&](auto SET, int n) {
                cur          = next_of(cur);
                auto publish = [&]() {
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    put(SET, last(n + 2), next_of(cur));
                    fetch(SET, last(n + 4));
                };
                block(SET, lds + cur * STAGE, publish, zero, [](int) {});
            };
            int n = block0;
#pragma unroll 1
            for (; n + 1 < block1; n += 2)
            {
                one_block(zero, n);
                one_block(one, n + 1);
            }
            if (n < block1)
                one_block(zero, n);
        }
    }

    // ---- results ------------------------------------------------------------------------------------------------------------
    // A lane has four neighbours of a row from each accumulator tile.  They go through LDS as a tile of whole rows (piece p of row r at p ^ r), and
    // from there in whole lines.  W words of 32 bits hold a lane's four results: 4 as floats (parts of a split sum), 2 rounded.
    auto through_lds = [&](int width, auto W_tag, auto&& words, auto&& store) {
        constexpr int W  = decltype(W_tag)::value;
        constexpr int TC = CIN && W == 2 ? CT / 2 : CT;    // tiles that results come from (forward: of gate and up together)
        const int pieces = width * W / 16;                  // 16-byte pieces of a row
        // what does not fit at once goes in two halves of each wave's row tiles
        constexpr int PASSES = BM * BN * W * (CIN && W == 2 ? 2 : 4) / 4 > RING * STAGE ? 2 : 1, RP = RT / PASSES;
#pragma unroll
        for (int i0 = 0; i0 < RT; i0 += RP)
        {
            __syncthreads();    // the ring, or the tile before, is read
#pragma unroll
            for (int i = 0; i < RP; i++)
#pragma unroll
                for (int c = 0; c < TC; c++)
                {
                    const int r = (wr * RP + i) * 16 + l16, col = (wc * TC + c) * 16 + 4 * q4;
                    uint32_t v[W];
                    words(c, i0 + i, v);
                    uint8_t* at = lds + (r * pieces + ((col * W / 16) ^ (r & (pieces - 1)))) * 16 + (W == 2 ? 8 * (q4 & 1) : 0);
                    if constexpr (W == 2)
                        *reinterpret_cast<v2i*>(at) = v2i{ (int)v[0], (int)v[1] };
                    else
                        *reinterpret_cast<v4i*>(at) = v4i{ (int)v[0], (int)v[1], (int)v[2], (int)v[3] };
                }
            __syncthreads();
#pragma unroll 2
            for (int u = tid; u < BM / PASSES * pieces; u += THREADS)
            {
                const int r = u / pieces, p = u % pieces;
                const int64_t m = m0 + (PASSES == 1 ? r : (r / (16 * RP) * RT + i0) * 16 + r % (16 * RP));
                if (m < a.M)
                    store(m, p, *reinterpret_cast<const v4i*>(lds + (r * pieces + (p ^ (r & (pieces - 1)))) * 16));
            }
        }
    };
    constexpr std::integral_constant<int, 2> rounded{};
    const float unit = kInUnits<T> && OP != OP_FORWARD ? *a.unit : 1.0f;
    auto round4 = [&](v4f v, uint32_t* w) { w[0] = pack16<T>(v[0], v[1]), w[1] = pack16<T>(v[2], v[3]); };
    if (a.splits > 1)
    {
        through_lds(BN, std::integral_constant<int, 4>(), [&](int c, int i, uint32_t* v) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[e] = __float_as_uint(acc[c][i][e]);
        }, [&](int64_t m, int p, v4i v) {
            // forward: of every 64 columns 32 are gate's sums, the others up's
            const int col   = 4 * p, which = CIN ? col >> 5 & 1 : 0;
            const int64_t n = n0 + (CIN ? (col >> 6) * 32 + (col & 31) : col);
            float* row      = a.part + (((int64_t)split * (CIN ? 2 : 1) + which) * a.M + m) * a.N;
            if (n + 4 <= a.N)
                __builtin_memcpy(row + n, &v, 16);
            else
#pragma unroll
                for (int e = 0; e < 3; e++)
                    if (n + e < a.N)
                        row[n + e] = __int_as_float(v[e]);
        });
        return;
    }
    if constexpr (OP == OP_FORWARD)
    {
        auto to = [&](uint16_t* out) { return [=](int64_t m, int p, v4i v) { store8(out + m * a.ldo, n0 + 8 * p, a.N, v); }; };
        if (a.pre_gate)
        {
            through_lds(TN, rounded, [&](int c, int i, uint32_t* w) { round4(acc[c][i], w); }, to(a.pre_gate));
            through_lds(TN, rounded, [&](int c, int i, uint32_t* w) { round4(acc[c + CT / 2][i], w); }, to(a.pre_up));
        }
        for_act(a.act, [&](auto ACT) {
            through_lds(TN, rounded, [&](int c, int i, uint32_t* w) {
                v4f v;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    v[e] = act_value<decltype(ACT)::value>(acc[c][i][e]) * acc[c + CT / 2][i][e];
                round4(v, w);
            }, to(a.out[0]));
        });
    }
    else
        through_lds(TN, rounded, [&](int c, int i, uint32_t* w) {
            if constexpr (kInUnits<T>)
            {
                const v4f v = acc[c][i];
                round4(v4f{ v[0] * unit, v[1] * unit, v[2] * unit, v[3] * unit }, w);
            }
            else
                round4(acc[c][i], w);
        }, [&](int64_t m, int p, v4i v) {
            uint16_t* out = a.out[0];
            if constexpr (OP == OP_DW)
            {
                // rows of dp's halves behind their F features are none of a gradient's
                if (m >= a.half)
                    m -= a.half, out = a.out[1];
                if (m >= a.features)
                    return;
            }
            store8(out + m * a.ldo, n0 + 8 * p, a.N, v);
        });
}

template <typename T, int OP, int WC, int WR, int RT, bool DIRECT>
__global__ __launch_bounds__(64 * WC * WR, 2) void gated_gemm_kernel(GemmFfnArgs a)
{
    gated_gemm<T, OP, WC, WR, RT, DIRECT>(a, blockIdx.x);
}

// d_x and the weights' gradients side by side in tiles of 128 x 128, where neither fills the chip: the first dx.per_xcd * 8 workgroups are d_x's.  us of both
// gradients together and one after the other: 509 x 722 x 1930 in fp16 31 and 50 (2 to 3 more on either side for the second pass over dp), 509 x 720 x 1930 26 and
// 38, 64 x 512 x 2048 16 and 22.
template <typename T, bool DIRECT>
__global__ __launch_bounds__(512, 2) void gated_gradients_kernel(GemmFfnArgs dx, GemmFfnArgs dw)
{
    const int of_dx = dx.per_xcd * 8;
    if ((int)blockIdx.x < of_dx)
        gated_gemm<T, OP_DX, 2, 4, 2, DIRECT>(dx, blockIdx.x);
    else
        gated_gemm<T, OP_DW, 2, 4, 2, DIRECT>(dw, blockIdx.x - of_dx);
}

// Results of a sum that was split, four of a row a thread: the parts in the order of the splits, then what the unsplit kernel does with a sum.
template <typename T, int OP>
__global__ __launch_bounds__(256) void gated_join_kernel(GemmFfnArgs a)
{
    const int64_t n = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, m = blockIdx.y;
    if (n >= a.N)
        return;
    constexpr int W     = OP == OP_FORWARD ? 2 : 1;
    const int64_t plane = (int64_t)a.M * a.N;
    const float* part   = a.part + m * a.N + n;
    const int live      = a.N - n < 4 ? (int)(a.N - n) : 4;
    v4f v[W];
#pragma unroll
    for (int w = 0; w < W; w++)
        v[w] = v4f{ 0.0f, 0.0f, 0.0f, 0.0f };
    for (int s = 0; s < a.splits; s++)
#pragma unroll
        for (int w = 0; w < W; w++)
        {
            v4f t = { 0.0f, 0.0f, 0.0f, 0.0f };
            const float* at = part + (s * W + w) * plane;
            if (live == 4)
                __builtin_memcpy(&t, at, 16);
            else
#pragma unroll
                for (int e = 0; e < 3; e++)
                    if (e < live)
                        t[e] = at[e];
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[w][e] += t[e];
        }
    auto store = [&](uint16_t* to, v4f r) {
        const v2i bits = { (int)pack16<T>(r[0], r[1]), (int)pack16<T>(r[2], r[3]) };
        if (live == 4)
            __builtin_memcpy(to, &bits, 8);
        else
#pragma unroll
            for (int e = 0; e < 3; e++)
                if (e < live)
                    to[e] = to_bits16<T>(r[e]);
    };
    if constexpr (OP == OP_FORWARD)
    {
        const int64_t at = m * a.ldo + n;
        if (a.pre_gate)
            store(a.pre_gate + at, v[0]), store(a.pre_up + at, v[W - 1]);
        for_act(a.act, [&](auto ACT) {
            v4f h;
#pragma unroll
            for (int e = 0; e < 4; e++)
                h[e] = act_value<decltype(ACT)::value>(v[0][e]) * v[W - 1][e];
            store(a.out[0] + at, h);
        });
    }
    else
    {
        const int half  = OP == OP_DW && m >= a.half ? 1 : 0;
        const int64_t r = m - (half ? a.half : 0);
        if constexpr (kInUnits<T>)
        {
            const float unit = *a.unit;
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[0][e] *= unit;
        }
        if (OP == OP_DX || r < a.features)
            store(a.out[half] + r * a.ldo + n, v[0]);
    }
}

// dp: eight features of a row a thread, of both halves, rounded to 16 bits because the matrix instructions take no more: each of its elements is then off
// by 2^-8 (bf16) or 2^-11 of itself at most, and a gradient by about sqrt(2) times what its own rounding costs.  Bound by memory: 335 MB in 64 us at 4096 x 8192.
//
// bf16 has the range of 32 bits, fp16 has not: dh u act'(g) may pass 65504, or lie below the least fp16 number, where the sums over it are numbers that fp16
// holds.  Where the largest of them lies between 2^-8 and 65504 they stand as they are, and what the least fp16 numbers cannot tell apart is less than 2^-17 of
// the largest, little beside the rounding.  Otherwise the second pass (AGAIN), which every call in fp16 launches and which returns at once (2 us) where the first one
// does, makes dp again in units of the power of two that brings the largest to 2^14 ... 2^15; the products' results are multiplied by it.  The largest is
// taken over finite elements; infinities and NaN stay what they are.
struct SlopeArgs
{
    const uint16_t *pre_gate, *pre_up, *dh;
    uint16_t* dp;
    float *most, *unit;        // fp16: the largest |dp| of every workgroup, and the unit
    int64_t ld, ldp, units;    // elements between rows of the inputs and of dp; units: rows * half / 8
    int32_t features, half, act;
    int32_t groups;            // workgroups of the first pass
};
constexpr int kSlopeGroups = 4096, kSlopeUnits = 2048, kSlopeAgain = 1024;   // workgroups at most: bf16, and fp16's two passes
constexpr size_t kUnitBytes = (kSlopeUnits + 16) * 4;                        // of most and unit

// the largest of the workgroup's (256 threads), in every thread
__device__ __forceinline__ float most_of_all(float v, float* of_wave)
{
#pragma unroll
    for (int d = 32; d; d >>= 1)
        v = fmaxf(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0)
        of_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(of_wave[0], of_wave[1]), fmaxf(of_wave[2], of_wave[3]));
}

template <typename T, bool AGAIN>
__global__ __launch_bounds__(256) void gated_slope_kernel(SlopeArgs a)
{
    static_assert(kInUnits<T> || !AGAIN, "bf16 has one pass");
    __shared__ float of_wave[4];
    float scale = 1.0f, most = 0.0f;    // (scale: a constant but in the second pass)
    if constexpr (AGAIN)
    {
        float of[kSlopeUnits / 256];    // (all on their way at once)
#pragma unroll
        for (int i = 0; i < kSlopeUnits / 256; i++)
            of[i] = a.most[i * 256 + (int)threadIdx.x < a.groups ? i * 256 + threadIdx.x : 0];
#pragma unroll
        for (int i = 0; i < kSlopeUnits / 256; i++)
            most = fmaxf(most, a.groups ? of[i] : 0.0f);
        most             = most_of_all(most, of_wave);
        const bool first = most == 0.0f || (most >= 0x1p-8f && most < 65520.0f);    // (65520 would round to infinity)
        const int bits   = (int)(__float_as_uint(most) >> 23), up = 141 - bits < 126 ? 141 - bits : 126;    // 2^14 / 2^(bits - 127); its reciprocal is no subnormal
        scale            = first ? 1.0f : __uint_as_float((uint32_t)(127 + up) << 23);
        if (blockIdx.x == 0 && threadIdx.x == 0)
            *a.unit = 1.0f / scale;
        if (first)
            return;
    }
    const int per_row = a.half / 8;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < a.units; u += (int64_t)gridDim.x * 256)
    {
        const int64_t m = u / per_row;
        const int f     = (int)(u - m * per_row) * 8;
        const v4i g = load8(a.pre_gate + m * a.ld, f, a.features), up = load8(a.pre_up + m * a.ld, f, a.features),
                  dh = load8(a.dh + m * a.ld, f, a.features);
        float x[8], y[8];
        for_act(a.act, [&](auto ACT) {
#pragma unroll
            for (int e = 0; e < 8; e++)
            {
                float value, slope;
                act_both<decltype(ACT)::value>(from_bits16<T>(half_of(g, e)), value, slope);
                const float d = from_bits16<T>(half_of(dh, e));
                x[e] = d * from_bits16<T>(half_of(up, e)) * slope;
                y[e] = d * value;
                if (f + e >= a.features)
                    x[e] = 0.0f, y[e] = 0.0f;
            }
        });
        if constexpr (kInUnits<T> && !AGAIN)
        {
            float here = 0.0f;    // (of a number and NaN the number)
#pragma unroll
            for (int e = 0; e < 8; e++)
                here = fmaxf(fmaxf(here, fabsf(x[e])), fabsf(y[e]));
            if (here == __builtin_huge_valf())
            {
                here = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    here = fmaxf(here, fmaxf(fabsf(x[e]) < __builtin_huge_valf() ? fabsf(x[e]) : 0.0f, fabsf(y[e]) < __builtin_huge_valf() ? fabsf(y[e]) : 0.0f));
            }
            most = fmaxf(most, here);
        }
        v4i dg, du;
#pragma unroll
        for (int p = 0; p < 4; p++)
        {
            dg[p] = (int)pack16<T>(x[2 * p] * scale, x[2 * p + 1] * scale);
            du[p] = (int)pack16<T>(y[2 * p] * scale, y[2 * p + 1] * scale);
        }
        uint16_t* row = a.dp + m * a.ldp + f;
        *reinterpret_cast<v4i*>(row)          = dg;
        *reinterpret_cast<v4i*>(row + a.half) = du;
    }
    if constexpr (kInUnits<T> && !AGAIN)
    {
        most = most_of_all(most, of_wave);
        if (threadIdx.x == 0)
            a.most[blockIdx.x] = most;
    }
}

// Rows filled up with zeros to whole pieces of eight elements: up to three matrices of one width
__global__ __launch_bounds__(256) void gated_widen_kernel(WidenRows a)
{
    const int per_row = (a.width + 7) / 8;
    const uint16_t* in = static_cast<const uint16_t*>(a.in[blockIdx.y]);
    const int64_t ld = a.ld[blockIdx.y], units = a.rows[blockIdx.y] * per_row, step = (int64_t)gridDim.x * 256;
    v4i* out = static_cast<v4i*>(a.out[blockIdx.y]);
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < units; u += step)
    {
        const int64_t m = u / per_row;
        out[u]          = load8(in + m * ld, (u - m * per_row) * 8, a.width);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

enum
{
    TILE_256,        // 256 x 256 results, eight waves
    TILE_256_128,    // 256 rows x 128 columns, eight waves
    TILE_128         // 128 x 128, eight waves, two workgroups a CU
};
struct Shape
{
    int tile;
    int splits, per_split;
    int tiles_m, tiles_n;
};
constexpr struct
{
    int bm, bn, slots;
    double empty, full, tile;    // us: of a block of 32 on an empty and on a full chip, and of a tile beside them
} kTiles[3] = { { 256, 256, 256, 0.62, 0.80, 12 }, { 256, 128, 256, 0.39, 0.48, 7 }, { 128, 128, 512, 0.33, 0.58, 6 } };
constexpr double kThroughRegisters = 1.4;
constexpr int kMostSplits = 16, kLeastBlocks = 16;    // parts of a sum, and blocks of a part

void split(Shape& s, int blocks, int parts)
{
    s.per_split = (blocks + parts - 1) / parts;
    s.splits    = s.per_split ? (blocks + s.per_split - 1) / s.per_split : 1;
}
// what splitting costs: the partial sums out and in, and a launch
double join_us(int op, int64_t M, int64_t N, int splits)
{
    return splits > 1 ? 3 + (double)M * N * (op == OP_FORWARD ? 2 : 1) * 4 * 2 * splits / 4.5e6 : 0;
}
bool may_split(int64_t M, int blocks, int parts)
{
    return parts == 1 || (blocks >= kLeastBlocks * parts && M < 65536);    // (a grid's second side)
}

// The tile, and into how many parts the sum is split, by the time that follows from what was measured (us, over 4096 x 2048 x 8192 and halves to
// eighths of each size): a block of 32 costs a workgroup of the three tiles 0.62, 0.39 and 0.33 on an empty chip and 0.80, 0.48 and 0.58 on
// a full one (the smaller ones ask L2 for more, the weights' gradients' least), a tile 12, 7 and 6 beside them, and a split its partial sums
// out and in at 4.5 TB/s and a launch.  Operands that go through
// registers cost 1.4 times as much, and take the smallest tile: the others' accumulators leave no room.  Both sides, us: d_x 4096 x 2048 x 8192 (128, 256 and 512 tiles) 240 with the largest tile and two parts, 332, 317
// and 359 in one part of each; of half the size 73 with four parts, 90 at best in one; forward 512 x 4096 x 2048 81, 52 and 43 in one part, 38, 32
// and 32 in the best number of parts; 4096 x 2048 x 8192 243, 301 and 328.
Shape shape_of(int op, int64_t M, int64_t N, int blocks, bool fast, double& least)
{
    const auto& of = kTiles;
    Shape best{};
    least = 0;
    for (int tile = fast ? TILE_256 : TILE_128; tile <= TILE_128; tile++)
    {
        const int tn = op == OP_FORWARD ? of[tile].bn / 2 : of[tile].bn;
        Shape s{};
        s.tile = tile, s.tiles_m = (int)((M + of[tile].bm - 1) / of[tile].bm), s.tiles_n = (int)((N + tn - 1) / tn);
        for (int want = 1; want <= kMostSplits && may_split(M, blocks, want); want++)
        {
            split(s, blocks, want);
            const int64_t n  = (int64_t)s.tiles_m * s.tiles_n * s.splits;
            const int64_t rounds = (n + of[tile].slots - 1) / of[tile].slots;
            // (of the smallest tile 256 have a CU each; of more some share one, and the last of those counts)
            const double busy = tile == TILE_128 ? n > 256 : n >= 256 ? 1 : n / 256.0;
            double us         = rounds * (s.per_split * (of[tile].empty + (of[tile].full - of[tile].empty) * busy) + of[tile].tile);
            us += join_us(op, M, N, s.splits);
            if (!best.tiles_m || us < least)
                least = us, best = s;
        }
        if (!best.tiles_m)    // no rows
            best = s;
    }
    least *= fast ? 1 : kThroughRegisters;
    return best;
}

size_t part_bytes(int op, const Shape& s, int64_t M, int64_t N)
{
    return s.splits > 1 ? (size_t)s.splits * (op == OP_FORWARD ? 2 : 1) * M * N * 4 : 0;
}

template <typename T, int OP, int WC, int WR, int RT, bool FAST>
bool launch_tiles(hipStream_t st, const GemmFfnArgs& a)
{
    constexpr size_t lds = kRing<FAST> * (64 * WC + 16 * RT * WR) * 64;
    if (!ensure_dynamic_lds<gated_gemm_kernel<T, OP, WC, WR, RT, FAST>>(lds))
        return false;
    gated_gemm_kernel<T, OP, WC, WR, RT, FAST><<<a.per_xcd * 8, 64 * WC * WR, lds, st>>>(a);
    return true;
}

// Tiles of 128 x 128 through registers: with two workgroups to a CU four waves are enough, and read LDS less (777 x 1111 x 2731 34.4 us with eight, 32.2)
bool four_waves(const Shape& s)
{
    return s.tiles_m * s.tiles_n * s.splits > 256;
}

void set_shape(GemmFfnArgs& a, const Shape& s)
{
    a.tiles_m = s.tiles_m, a.tiles_n = s.tiles_n, a.tiles = s.tiles_m * s.tiles_n;
    a.splits = s.splits, a.per_split = s.per_split;
    a.per_xcd = (a.tiles * a.splits + 7) / 8;
}

template <int OP>
void launch_join(hipStream_t st, int32_t dtype, const GemmFfnArgs& a)
{
    const dim3 grid((a.N + 1023) / 1024, a.M);
    if (a.splits > 1 && dtype == TMI_BF16)
        gated_join_kernel<bf16_t, OP><<<grid, 256, 0, st>>>(a);
    else if (a.splits > 1)
        gated_join_kernel<_Float16, OP><<<grid, 256, 0, st>>>(a);
}

bool launch_gradients(hipStream_t st, int32_t dtype, const GemmFfnArgs& dx, const GemmFfnArgs& dw, bool fast)
{
    auto typed = [&](auto type, auto FAST) {
        using T = decltype(type);
        constexpr bool DIRECT = decltype(FAST)::value;
        constexpr size_t lds  = kRing<DIRECT> * 256 * 64;
        if (!ensure_dynamic_lds<gated_gradients_kernel<T, DIRECT>>(lds))
            return false;
        gated_gradients_kernel<T, DIRECT><<<(dx.per_xcd + dw.per_xcd) * 8, 512, lds, st>>>(dx, dw);
        return true;
    };
    const bool ok = dtype == TMI_BF16 ? (fast ? typed(bf16_t{}, std::true_type()) : typed(bf16_t{}, std::false_type()))
                                      : (fast ? typed(_Float16{}, std::true_type()) : typed(_Float16{}, std::false_type()));
    if (ok)
        launch_join<OP_DX>(st, dtype, dx), launch_join<OP_DW>(st, dtype, dw);
    return ok;
}

template <int OP>
bool launch_product(hipStream_t st, int32_t dtype, const GemmFfnArgs& a, const Shape& s, bool fast)
{
    auto typed = [&](auto type) {
        using T = decltype(type);
        bool ok;
        if (s.tile == TILE_256)
            ok = launch_tiles<T, OP, 4, 2, 8, true>(st, a);
        else if (s.tile == TILE_256_128)
            ok = launch_tiles<T, OP, 2, 4, 4, true>(st, a);
        else
            // Eight waves, whose reads and matrix instructions hide each other's waits: us forward 1024 x 1024 x 1024 13.3 with eight and 15.2 with four, 500 x
            // 1111 x 2731 through registers 17.2 and 20.9.
            ok = fast ? launch_tiles<T, OP, 2, 4, 2, true>(st, a)
                      : four_waves(s) ? launch_tiles<T, OP, 2, 2, 4, false>(st, a) : launch_tiles<T, OP, 2, 4, 2, false>(st, a);
        return ok;
    };
    const bool ok = dtype == TMI_BF16 ? typed(bf16_t{}) : typed(_Float16{});
    if (ok)
        launch_join<OP>(st, dtype, a);
    return ok;
}

// Loads straight into LDS take a lane's offset from a tile's first element in 32 bits: over the 256 rows of the largest tile 2^31 bytes from here on.
constexpr int64_t kFarRows = int64_t(1) << 22;

// whether rows of `width` elements, `ld` apart, are whole 16-byte pieces, and near enough for those offsets
bool whole_pieces(const void* p, int64_t width, int64_t ld)
{
    return ((uintptr_t)p & 15) == 0 && width % 8 == 0 && ld % 8 == 0 && ld < kFarRows;
}

int64_t whole_of(int64_t n, int64_t per)
{
    return (n + per - 1) / per * per;
}

// A product's way: of operands that lie in whole pieces, as they are; of others through registers, or on copies that end in zeros, read and written at 3.5
// TB/s with 8 us for a launch more.  us forward 4096 x 2047 x 8192 460 through registers, 263 on copies, its gradients 905 and 536; 777 x 1111 x 2731 32 and
// 38, 512 x 4095 x 4096 61 and 87.  (Rows of less than eight elements are always copied: the loads through registers take eight.)  Where the rows of a copy,
// or of dp (`ldp`, 0 where it is no operand), lie too far apart for the offsets of the direct loads, the product takes the registers' 64-bit addresses.
struct Way
{
    bool fast, copies;
    size_t bytes;     // of the copies
    Shape shape;
};
Way way_of(int op, int64_t M, int64_t N, int blocks, bool whole, int64_t ldp, int64_t copied_rows, int64_t d, double& us)
{
    Way w{};
    double direct = 0, registers = 0;
    w.shape = shape_of(op, M, N, blocks, true, direct);
    w.fast  = true;
    us      = direct;
    const bool near = ldp < kFarRows;
    if (whole && near)
        return w;
    const Shape other  = shape_of(op, M, N, blocks, false, registers);
    const size_t bytes = (size_t)copied_rows * whole_of(d, 8) * 2;
    const double copy  = 2 * (double)bytes / 3.5e6 + 8;
    if (d < 8 || (near && whole_of(d, 8) < kFarRows && direct + copy < registers))
        w.copies = true, w.bytes = bytes, us += copy;
    if (!near || !w.copies)
        w.fast = false, w.shape = other, us = registers + (w.copies ? copy : 0);
    return w;
}

// Both gradients in one launch, if that takes less than `apart`, one after the other, and 4 us for the other launch: in tiles of 128 x 128, of which
// 512 have a place, with parts of the sums as long as those that are there together allow.
bool side_by_side(Way& dx, int64_t dx_rows, int dx_blocks, Way& dw, int64_t dw_rows, int dw_blocks, int64_t N, double apart)
{
    const auto& tile    = kTiles[TILE_128];
    const double slower = dx.fast ? 1 : kThroughRegisters;
    double least        = apart + 4;
    bool better         = false;
    Shape x{}, w{};
    x.tile = w.tile = TILE_128;
    x.tiles_m = (int)((dx_rows + tile.bm - 1) / tile.bm), w.tiles_m = (int)((dw_rows + tile.bm - 1) / tile.bm);
    x.tiles_n = w.tiles_n = (int)((N + tile.bn - 1) / tile.bn);
    if ((int64_t)(x.tiles_m + (int64_t)w.tiles_m) * x.tiles_n > 2 * tile.slots || !x.tiles_n || !x.tiles_m || !w.tiles_m)
        return false;
    for (int px = 1; px <= kMostSplits && may_split(dx_rows, dx_blocks, px); px++)
        for (int pw = 1; pw <= kMostSplits && may_split(dw_rows, dw_blocks, pw); pw++)
        {
            split(x, dx_blocks, px), split(w, dw_blocks, pw);
            const double nx = (double)x.tiles_m * x.tiles_n * x.splits, nw = (double)w.tiles_m * w.tiles_n * w.splits;
            const double block = (nx + nw > 256 ? tile.full : tile.empty) * slower;
            const double one_x = x.per_split * block + tile.tile, one_w = w.per_split * block + tile.tile;
            // the longest of them, and what all of them take from the places
            const double longest = one_x > one_w ? one_x : one_w, all = (nx * one_x + nw * one_w) / tile.slots;
            const double us = (nx + nw <= tile.slots ? longest : all + longest / 2) + join_us(OP_DX, dx_rows, N, x.splits) + join_us(OP_DW, dw_rows, N, w.splits);
            if (us < least)
                least = us, better = true, dx.shape = x, dw.shape = w;
        }
    return better;
}

// What a call launches, from its sizes, strides and addresses
struct ForwardPlan
{
    int blocks;
    Way way;
    double us;
};
ForwardPlan forward_plan(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up)
{
    ForwardPlan p;
    const bool whole = whole_pieces(x, d.in_features, d.ld_x) && whole_pieces(gate, d.in_features, d.ld_w) && whole_pieces(up, d.in_features, d.ld_w);
    p.blocks         = (int)(whole_of(d.in_features, kBlock) / kBlock);
    p.way            = way_of(OP_FORWARD, d.rows, d.hidden_features, p.blocks, whole, 0, (int64_t)d.rows + 2 * (int64_t)d.hidden_features, d.in_features, p.us);
    return p;
}
struct BackwardPlan
{
    int64_t half, ldp;
    size_t dp_bytes, unit_bytes;
    int dx_blocks, dw_blocks;
    Way dx, dw;
    bool together;    // in one launch
};
BackwardPlan backward_plan(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up, bool want_dx, bool want_dw)
{
    BackwardPlan p;
    p.half           = whole_of(d.hidden_features, 64);
    // Rows of dp lie 128 bytes further apart than they are long: the 256 rows that a tile reads 64 bytes of at a time would otherwise lie a power
    // of two apart where F is one, on few channels of the memory.
    p.ldp            = 2 * p.half + 64;
    p.dp_bytes       = (size_t)d.rows * p.ldp * 2;
    p.unit_bytes     = d.dtype == TMI_FP16 ? kUnitBytes : 0;
    p.dx_blocks      = (int)(2 * p.half / kBlock);
    p.dw_blocks      = (int)(whole_of(d.rows, kBlock) / kBlock);
    const int64_t D  = d.in_features, F = d.hidden_features;
    double us_dx, us_dw;
    p.dx             = way_of(OP_DX, d.rows, D, p.dx_blocks, whole_pieces(gate, D, d.ld_w) && whole_pieces(up, D, d.ld_w), p.ldp, 2 * F, D, us_dx);
    p.dw             = way_of(OP_DW, 2 * p.half, D, p.dw_blocks, whole_pieces(x, D, d.ld_x), p.ldp, d.rows, D, us_dw);
    p.together       = false;
    if (want_dx && want_dw && !p.dx.copies && !p.dw.copies && p.dx.fast == p.dw.fast)
        p.together = side_by_side(p.dx, d.rows, p.dx_blocks, p.dw, 2 * p.half, p.dw_blocks, D, us_dx + us_dw);
    return p;
}

}    // namespace

void launch_widen_rows(hipStream_t st, const WidenRows& a)
{
    int64_t most = 0;
    for (int i = 0; i < a.n; i++)
        most = most > a.rows[i] ? most : a.rows[i];
    const int64_t groups = (most * ((a.width + 7) / 8) + 255) / 256;
    if (groups > 0)
        gated_widen_kernel<<<dim3((int)(groups < 2048 ? groups : 2048), a.n), 256, 0, st>>>(a);
}

// The products of a few rows against the tiles here.  A workgroup of those takes 1024 columns of 16 weight rows and 32 rows of x in 3.6 us, 512 have a
// place, and the weights come in at 4.3 TB/s for each 32 rows; 1.4 times that from odd elements.  us few rows / tiles: 32 rows 512 x 512 4.9 / 8.3, 1024 x
// 4096 6.7 / 11.6, 4096 x 1024 16.6 / 13.9, 8000 x 500 30.9 / 16.4, 2048 x 8192 17.8 / 17.2; 48 rows 1024 x 2000 6.7 / 11.5; 40 rows 2048 x 8192 27.4 / 18.2.
bool gated_ffn_few_rows_lead(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up)
{
    if (d.rows <= 16 || d.in_features < 8)
        return true;
    if (d.rows > 64)
        return false;
    const double chunks = (d.rows + 31) / 32, workgroups = chunks * ((d.hidden_features + 15) / 16), places = workgroups > 512 ? workgroups / 512 : 1;
    const double chain  = ((d.in_features + 1023) / 1024) * 3.6 * places, bytes = chunks * 4.0 * d.in_features * d.hidden_features / 4.3e6;
    const bool odd      = ((d.ld_x | d.ld_w) & 1) || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(up)) & 2);
    return 1.7 + (chain > bytes ? chain : bytes) * (odd ? 1.4 : 1) < forward_plan(d, x, gate, up).us;
}

GatedFfnPlan gated_ffn_plan(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up, int product)
{
    GatedFfnPlan r{};
    if (product == OP_FORWARD && gated_ffn_few_rows_lead(d, x, gate, up))
        return r;
    Way w{};
    int64_t M = d.rows, col_rows = kBlock, row_rows = kBlock, ldc = product == OP_DW ? d.ld_x : d.ld_w, ldr = d.ld_x;
    if (product == OP_FORWARD)
        w = forward_plan(d, x, gate, up).way;
    else
    {
        const BackwardPlan p = backward_plan(d, x, gate, up, true, true);
        w = product == OP_DX ? p.dx : p.dw, ldr = p.ldp, r.together = p.together;
        M = product == OP_DX ? d.rows : 2 * p.half;
    }
    const auto& tile = kTiles[w.shape.tile];
    if (w.copies)
        ldc = whole_of(d.in_features, 8), ldr = product == OP_FORWARD ? ldc : ldr;
    if (product == OP_FORWARD)
        col_rows = d.hidden_features < tile.bn / 2 ? d.hidden_features : tile.bn / 2;
    if (product != OP_DW)
        row_rows = M < tile.bm ? M : tile.bm;
    r.bm = tile.bm, r.bn = tile.bn, r.fast = w.fast, r.copies = w.copies, r.splits = w.shape.splits;
    r.waves = !w.fast && !r.together && four_waves(w.shape) ? 4 : 8;
    // (a tile's rows are read 64 bytes at a time where the summed index is innermost, else whole)
    const int64_t of_col = (col_rows - 1) * ldc * 2 + (product == OP_FORWARD ? 2 * kBlock : 2 * tile.bn),
                  of_row = (row_rows - 1) * ldr * 2 + (product == OP_DW ? 2 * tile.bm : 2 * kBlock);
    r.span = w.fast ? (of_col > of_row ? of_col : of_row) : 0;
    return r;
}

size_t gated_ffn_scratch_bytes(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up)
{
    const Way w = forward_plan(d, x, gate, up).way;
    return w.bytes + part_bytes(OP_FORWARD, w.shape, d.rows, d.hidden_features);
}

const char* launch_gated_ffn(hipStream_t st, const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up, void* h, void* pre_gate,
                             void* pre_up, void* scratch, const void* zeros)
{
    ForwardPlan p = forward_plan(d, x, gate, up);
    if (!scratch && p.way.copies)
    {
        double us;
        p.way.copies = p.way.fast = false;
        p.way.shape = shape_of(OP_FORWARD, d.rows, d.hidden_features, p.blocks, false, us);
    }
    if (!scratch)
        p.way.shape.splits = 1, p.way.shape.per_split = p.blocks;
    GemmFfnArgs a{};
    a.col[0] = static_cast<const uint16_t*>(gate), a.col[1] = static_cast<const uint16_t*>(up), a.row = static_cast<const uint16_t*>(x);
    a.out[0] = static_cast<uint16_t*>(h);
    a.pre_gate = static_cast<uint16_t*>(pre_gate), a.pre_up = static_cast<uint16_t*>(pre_up);
    a.zeros = static_cast<const uint8_t*>(zeros);
    a.ldc = d.ld_w, a.ldr = d.ld_x, a.ldo = d.ld_h;
    a.M = d.rows, a.N = d.hidden_features, a.K = d.in_features, a.blocks = p.blocks, a.act = d.activation;
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + p.way.bytes);
    if (p.way.copies)
    {
        // (columns that fill up the last piece are zeros on both sides of the products)
        const int64_t wide = whole_of(d.in_features, 8);
        uint16_t *cx = static_cast<uint16_t*>(scratch), *cg = cx + d.rows * wide, *cu = cg + d.hidden_features * wide;
        launch_widen_rows(st, WidenRows{ 3, d.in_features, { x, gate, up }, { d.ld_x, d.ld_w, d.ld_w }, { d.rows, d.hidden_features, d.hidden_features }, { cx, cg, cu } });
        a.row = cx, a.col[0] = cg, a.col[1] = cu, a.ldr = a.ldc = wide, a.K = (int32_t)wide;
    }
    set_shape(a, p.way.shape);
    return launch_product<OP_FORWARD>(st, d.dtype, a, p.way.shape, p.way.fast) ? "gated_ffn" : nullptr;
}

// dp, then its unit, then copies, then the partial sums: of one product after the other, or of both
size_t gated_ffn_backward_scratch_bytes(const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up, bool dx, bool dw)
{
    const BackwardPlan p = backward_plan(d, x, gate, up, dx, dw);
    const size_t of_dx   = dx ? part_bytes(OP_DX, p.dx.shape, d.rows, d.in_features) : 0;
    const size_t of_dw   = dw ? part_bytes(OP_DW, p.dw.shape, 2 * p.half, d.in_features) : 0;
    return p.dp_bytes + p.unit_bytes + p.dx.bytes + p.dw.bytes + (p.together ? of_dx + of_dw : of_dx > of_dw ? of_dx : of_dw);
}

const char* launch_gated_ffn_backward(hipStream_t st, const tmi_gated_ffn_desc_t& d, const void* x, const void* gate, const void* up,
                                      const void* pre_gate, const void* pre_up, const void* d_h, void* d_x, void* d_gate, void* d_up, void* scratch,
                                      const void* zeros)
{
    const BackwardPlan p = backward_plan(d, x, gate, up, d_x, d_gate);
    SlopeArgs q{};
    q.pre_gate = static_cast<const uint16_t*>(pre_gate), q.pre_up = static_cast<const uint16_t*>(pre_up), q.dh = static_cast<const uint16_t*>(d_h);
    q.dp = static_cast<uint16_t*>(scratch), q.ld = d.ld_h, q.ldp = p.ldp, q.units = d.rows * (p.half / 8);
    q.features = d.hidden_features, q.half = (int32_t)p.half, q.act = d.activation;
    q.most = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + p.dp_bytes), q.unit = q.most + kSlopeUnits;
    const int64_t groups = (q.units + 255) / 256;
    const int64_t limit  = d.dtype == TMI_FP16 ? kSlopeUnits : kSlopeGroups;
    q.groups             = (int32_t)(groups < limit ? groups : limit);
    if (d.dtype == TMI_FP16)
    {
        if (q.groups > 0)
            gated_slope_kernel<_Float16, false><<<q.groups, 256, 0, st>>>(q);
        // (no rows or features: the unit of sums of nothing)
        gated_slope_kernel<_Float16, true><<<q.groups < 1 ? 1 : q.groups < kSlopeAgain ? q.groups : kSlopeAgain, 256, 0, st>>>(q);
    }
    else if (q.groups > 0)
        gated_slope_kernel<bf16_t, false><<<q.groups, 256, 0, st>>>(q);

    const int64_t wide = whole_of(d.in_features, 8);
    uint16_t* copies   = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(scratch) + p.dp_bytes + p.unit_bytes);
    GemmFfnArgs a{};
    a.row = q.dp, a.ldr = p.ldp, a.half = (int32_t)p.half, a.features = d.hidden_features;
    a.part  = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(copies) + p.dx.bytes + p.dw.bytes);
    a.zeros = static_cast<const uint8_t*>(zeros);
    a.unit  = q.unit;
    a.N     = d.in_features;
    GemmFfnArgs of_x = a, of_w = a;
    if (d_x)
    {
        of_x.col[0] = static_cast<const uint16_t*>(gate), of_x.col[1] = static_cast<const uint16_t*>(up), of_x.ldc = d.ld_w, of_x.width = d.in_features;
        if (p.dx.copies)
        {
            launch_widen_rows(st, WidenRows{ 2, d.in_features, { gate, up }, { d.ld_w, d.ld_w }, { d.hidden_features, d.hidden_features },
                                             { copies, copies + d.hidden_features * wide } });
            of_x.col[0] = copies, of_x.col[1] = copies + d.hidden_features * wide, of_x.ldc = wide, of_x.width = (int32_t)wide;
        }
        of_x.out[0] = static_cast<uint16_t*>(d_x), of_x.ldo = d.ld_x;
        of_x.M = d.rows, of_x.K = d.hidden_features, of_x.blocks = p.dx_blocks;
        set_shape(of_x, p.dx.shape);
    }
    if (d_gate)
    {
        of_w.col[0] = of_w.col[1] = static_cast<const uint16_t*>(x), of_w.ldc = d.ld_x, of_w.width = d.in_features;
        if (p.dw.copies)
        {
            uint16_t* cx = copies + p.dx.bytes / 2;
            launch_widen_rows(st, WidenRows{ 1, d.in_features, { x }, { d.ld_x }, { d.rows }, { cx } });
            of_w.col[0] = of_w.col[1] = cx, of_w.ldc = wide, of_w.width = (int32_t)wide;
        }
        of_w.out[0] = static_cast<uint16_t*>(d_gate), of_w.out[1] = static_cast<uint16_t*>(d_up), of_w.ldo = d.ld_w;
        of_w.M = (int32_t)(2 * p.half), of_w.K = d.rows, of_w.blocks = p.dw_blocks;
        set_shape(of_w, p.dw.shape);
    }
    bool ok = true;
    if (p.together)
    {
        of_w.part += part_bytes(OP_DX, p.dx.shape, d.rows, d.in_features) / 4;
        ok = launch_gradients(st, d.dtype, of_x, of_w, p.dx.fast);
    }
    else
    {
        if (d_x)
            ok = launch_product<OP_DX>(st, d.dtype, of_x, p.dx.shape, p.dx.fast);
        if (ok && d_gate)
            ok = launch_product<OP_DW>(st, d.dtype, of_w, p.dw.shape, p.dw.fast);
    }
    return ok ? "gated_ffn_backward" : nullptr;
}

}    // namespace tmi
