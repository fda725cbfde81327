// Gradients of the root-mean-square norm.  With n = s r and g = dy (offset + w), r = 1 / rms(s) from the forward pass:
//
//   d_x      = r (g - n mean(g n)) + d_sum        mean over a row; d_sum: what comes past the norm, where s is used elsewhere too
//   d_weight = sum over rows of dy n
//
// Bound by memory: a row of s, dy and d_sum is read once into registers, its mean is taken over the lanes, and d_x is written.  d_weight's terms of a lane's
// columns are added over the rows that its workgroup has, without leaving the registers; the workgroups' sums meet in the scratch buffer, [workgroup][width]
// in 32 bits, and a second kernel adds those in order, so that equal calls give equal bits.
//
// 8192 x 4096 in bf16 with d_weight: 46.6 us, 4.3 TB/s (the second kernel 4.8 of them), with d_sum too 55.3; without d_weight 38.1, 5.3 TB/s.  131072 x 128:
// 25.5.  A row's loads before the sum of the one ahead of it gave the same 46.2, and 1 us more where a workgroup has one or two rows; a wave for a whole row,
// whose registers then overflow, 59.4.  Rows of 4095 elements, read in words: 57.4 with d_weight, where 4096 take 45.5 in the same run.  1024 x 40000, read twice: 87.4, 2.8 TB/s of
// the bytes that one reading would take.
//
// A row has 8 to 64 lanes of a wave, 256 or 1024 of a workgroup, each with P pieces of 16 bytes.  Longer rows are read twice: once for the means, once by
// column tiles with the means given.
#include "tmi_rows.h"

namespace tmi
{
namespace
{

struct BackArgs
{
    const void *s, *weight, *dy, *d_sum;
    const float* rstd;
    void *dx, *dw;
    float *mean, *part;    // [rows] (long rows only) and [workgroups][width]
    int64_t ld_s, ld_y, ld_x;
    int64_t rows;
    int32_t width, groups;
    float offset;
};

constexpr int kMostGroups = 256;    // workgroups that leave sums

// THREADS / G rows at once.  GIVEN: the means are, and blockIdx.y is a column tile of G P pieces
template <typename T, int THREADS, int G, int P, bool WHOLE, bool GIVEN>
__global__ __launch_bounds__(THREADS) void norm_backward_kernel(BackArgs a)
{
    constexpr int ROWS = THREADS / G, V = kPiece<T>, COLUMNS = G * P * V;
    __shared__ uint32_t slots[2][ROWS][2 * (G > 64 ? G / 64 : 1)];
    __shared__ __align__(16) float met[ROWS > 1 ? THREADS * V : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G, width = a.width, first = GIVEN ? (int)blockIdx.y * COLUMNS : 0;
    auto at = [&](int p) { return first + (p * G + lane) * V; };

    v4i w[P];
    float dw[P][V];
#pragma unroll
    for (int p = 0; p < P; p++)
    {
        w[p] = load_piece<T, WHOLE>(static_cast<const T*>(a.weight), at(p), width);
#pragma unroll
        for (int e = 0; e < V; e++)
            dw[p][e] = 0.0f;
    }
    int slot = 0;
    // (the groups of a workgroup go round together, for its barriers; one whose rows are done takes the last row again, and drops what it makes)
    for (int64_t m0 = (int64_t)blockIdx.x * ROWS; m0 < a.rows; m0 += (int64_t)gridDim.x * ROWS)
    {
        const bool live = m0 + group < a.rows;
        const int64_t m = live ? m0 + group : a.rows - 1;
        // (with the means given no barrier stands between a row's reads and its writes)
        auto load = [&](const void* from, int64_t ld, int p) {
            const T* row = static_cast<const T*>(from) + m * ld;
            return GIVEN ? load_piece_alone<T, WHOLE>(row, at(p), width) : load_piece<T, WHOLE>(row, at(p), width);
        };
        v4i s[P], dy[P], past[P];
#pragma unroll
        for (int p = 0; p < P; p++)
            s[p] = load(a.s, a.ld_s, p);
#pragma unroll
        for (int p = 0; p < P; p++)
            dy[p] = load(a.dy, a.ld_y, p);
        const float r = a.rstd[m];
        if (a.d_sum)
#pragma unroll
            for (int p = 0; p < P; p++)
                past[p] = load(a.d_sum, a.ld_s, p);
        else
#pragma unroll
            for (int p = 0; p < P; p++)
                past[p] = v4i{ 0, 0, 0, 0 };

        float mean = 0.0f;
        if constexpr (GIVEN)
            mean = a.mean[m];
        else
        {
            uint32_t none = 0;
#pragma unroll
            for (int p = 0; p < P; p++)
            {
                float part = 0.0f;
#pragma unroll
                for (int e = 0; e < V; e++)
                    part = __builtin_fmaf(piece_get<T>(dy[p], e) * (a.offset + piece_get<T>(w[p], e)), piece_get<T>(s[p], e) * r, part);
                mean += part;
            }
            over_row<G, true, false>(mean, none, slots[slot][group]);
            slot = 1 - slot;
            mean /= (float)width;
            // (the pieces wait as they came: as floats they would take twice the registers)
#pragma unroll
            for (int p = 0; p < P; p++)
                asm volatile("" : "+v"(s[p]), "+v"(dy[p]), "+v"(w[p]));
        }
        if (!live)
            continue;
#pragma unroll
        for (int p = 0; p < P; p++)
        {
            float dx[V];
#pragma unroll
            for (int e = 0; e < V; e++)
            {
                const float n = piece_get<T>(s[p], e) * r, d = piece_get<T>(dy[p], e), g = d * (a.offset + piece_get<T>(w[p], e));
                dw[p][e] = __builtin_fmaf(d, n, dw[p][e]);
                dx[e]    = __builtin_fmaf(r, g - n * mean, piece_get<T>(past[p], e));
            }
            if (a.dx)
                store_piece<T, WHOLE>(static_cast<T*>(a.dx) + m * a.ld_x, at(p), width, piece_of<T>(dx));
        }
    }
    if (!a.dw)
        return;
    float* part = a.part + (int64_t)blockIdx.x * width;
    if constexpr (ROWS > 1)
    {
        // the groups' sums, in order
#pragma unroll
        for (int p = 0; p < P; p++)
        {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; e += 4)
                *reinterpret_cast<v4i*>(met + (group * G + lane) * V + e) = piece_of<float>(&dw[p][e]);
            __syncthreads();
            if constexpr (G * V < THREADS)
            {
                // V groups a thread, and then what those are (all of them one after the other took up to 0.5 us more)
                constexpr int PARTS = ROWS / V;
                const int k = threadIdx.x % (G * V), of = threadIdx.x / (G * V);
                float sum   = met[of * V * (G * V) + k];
#pragma unroll
                for (int g = 1; g < V; g++)
                    sum += met[(of * V + g) * (G * V) + k];
                __syncthreads();
                met[threadIdx.x] = sum;
                __syncthreads();
                if (of != 0 || p * G * V + k >= width)
                    continue;
#pragma unroll
                for (int i = 1; i < PARTS; i++)
                    sum += met[i * (G * V) + k];
                part[p * G * V + k] = sum;
            }
            else
                for (int k = threadIdx.x; k < G * V && p * G * V + k < width; k += THREADS)
                {
                    float sum = 0.0f;
#pragma unroll
                    for (int g = 0; g < ROWS; g++)
                        sum += met[g * G * V + k];
                    part[p * G * V + k] = sum;
                }
        }
    }
    else
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int e = 0; e < V; e += 4)
                store_piece<float, false>(part, at(p) + e, width, piece_of<float>(&dw[p][e]));
}

// The means of rows that are too long for the kernel above
template <typename T, bool WHOLE>
__global__ __launch_bounds__(1024) void norm_mean_kernel(BackArgs a)
{
    constexpr int G = 1024, V = kPiece<T>;
    __shared__ uint32_t slots[2][2 * (G / 64)];
    int slot = 0;
    for (int64_t m = blockIdx.x; m < a.rows; m += gridDim.x)
    {
        const T *s = static_cast<const T*>(a.s) + m * a.ld_s, *dy = static_cast<const T*>(a.dy) + m * a.ld_y, *w = static_cast<const T*>(a.weight);
        const float r = a.rstd[m];
        float mean    = 0.0f;
        uint32_t none = 0;
        for (int k = (int)threadIdx.x * V; k < a.width; k += G * V)
        {
            const v4i ps = load_piece<T, WHOLE>(s, k, a.width), pd = load_piece<T, WHOLE>(dy, k, a.width), pw = load_piece<T, WHOLE>(w, k, a.width);
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < V; e++)
                part = __builtin_fmaf(piece_get<T>(pd, e) * (a.offset + piece_get<T>(pw, e)), piece_get<T>(ps, e) * r, part);
            mean += part;
        }
        over_row<G, true, false>(mean, none, slots[slot]);
        slot = 1 - slot;
        if (threadIdx.x == 0)
            a.mean[m] = mean / (float)a.width;
    }
}

// The workgroups' sums: 32 columns and 32 parts of the list a workgroup (with 16 and 64 the same, with 8 and 128 2.5 us more at 8192 x 4096).  Of a grid's two
// dimensions none has more than kJoinGrid workgroups: the threads of one are counted in 32 bits, and 2^28 columns have 2^33.
constexpr int kJoinGrid = 1 << 20;
template <typename T>
__global__ __launch_bounds__(1024) void norm_join_kernel(BackArgs a)
{
    constexpr int COLUMNS = 32, SHARES = 1024 / COLUMNS;
    __shared__ float met[SHARES][COLUMNS + 1];
    const int column = threadIdx.x % COLUMNS, share = threadIdx.x / COLUMNS;
    const int64_t k  = ((int64_t)blockIdx.y * kJoinGrid + blockIdx.x) * COLUMNS + column;
    constexpr int MOST = kMostGroups / SHARES;
    const int each = (a.groups + SHARES - 1) / SHARES, first = share * each;
    const int64_t column_of = k < a.width ? k : a.width - 1;
    // (all of them asked for at once, past the last one it again: one after the other 509 x 1930 9.5 us, now 9.0)
    float sum = 0.0f;
    if (a.groups > 0)    // (no rows: zeros)
    {
        float t[MOST];
#pragma unroll
        for (int i = 0; i < MOST; i++)
        {
            const int g = i < each && first + i < a.groups ? first + i : a.groups - 1;
            t[i]        = a.part[(int64_t)g * a.width + column_of];
        }
#pragma unroll
        for (int i = 0; i < MOST; i++)
            if (i < each && first + i < a.groups)
                sum += t[i];
    }
    met[share][column] = sum;
    __syncthreads();
    if (share != 0 || k >= a.width)
        return;
#pragma unroll
    for (int i = 1; i < SHARES; i++)
        sum += met[i][column];
    if constexpr (sizeof(T) == 4)
        static_cast<T*>(a.dw)[k] = sum;
    else
        static_cast<uint16_t*>(a.dw)[k] = to_bits16<T>(sum);
}

// Lanes of a row (us with 16 at least 262144 x 64 bf16 34.0, with eight 25.8; with 64 instead of 32 44157 x 168 23.2 and 16.4), its pieces a lane, and how many
// workgroups share the rows.  Each of those leaves 4 bytes a column for the second kernel, against b bytes a
// column and tensor that it reads of its rows.
struct BackPlan
{
    int threads, lanes, pieces, groups, tiles;    // tiles > 1: long rows
};
BackPlan back_plan(int32_t dtype, int64_t rows, int64_t width, bool dw)
{
    const int v           = dtype == TMI_FP32 ? 4 : 8;
    const int64_t pieces  = (width + v - 1) / v;
    BackPlan p{};
    p.tiles = 1;
    if (pieces <= 8)
        p.lanes = 8, p.pieces = 1;
    else if (pieces <= 16)
        p.lanes = 16, p.pieces = 1;
    else if (pieces <= 32)
        p.lanes = 32, p.pieces = 1;
    else if (pieces <= 128)
        p.lanes = 64, p.pieces = pieces <= 64 ? 1 : 2;
    else if (pieces <= 512)
        p.lanes = 256, p.pieces = pieces <= 256 ? 1 : 2;
    else
    {
        p.lanes = 1024, p.pieces = pieces <= 1024 ? 1 : 2;
        p.tiles = (int)((pieces + 2047) / 2048);
    }
    // A workgroup's sums are written and read again, and few of them make a short second kernel: 256 workgroups of 1024 threads, one for a CU.  (us with them,
    // and with 512 of 256 threads: 8192 x 4096 bf16 46.6 and 48.4, 509 x 1930 fp32 9.0 and 11.9, 131072 x 128 bf16 25.5 and 27.5.)  Too few rows to give every
    // CU such a workgroup have ones of 256 threads: 64 x 4096 6.5 and with 1024 threads 8.1, 128 x 4096 7.5 and 8.3, but 256 x 4096 9.4 and 8.7.  Without
    // d_weight there are no sums, and each workgroup has its own rows: 8192 x 4096 38.1, with 256 workgroups 41.8.
    p.threads = p.lanes == 1024 || (dw && rows * p.lanes > 48 * 1024) ? 1024 : 256;
    const int at_once  = p.threads / p.lanes;
    const int64_t need = (rows + at_once - 1) / at_once, most = dw ? kMostGroups / (p.tiles < 4 ? p.tiles : 4) : 1 << 20;
    p.groups = (int)(need < most ? need : most);
    return p;
}

template <typename T, bool WHOLE>
void launch_typed(hipStream_t st, const BackArgs& a, const BackPlan& p)
{
    auto go = [&](auto kernel) { kernel<<<dim3(p.groups, p.tiles), p.threads, 0, st>>>(a); };
    if (p.groups > 0)
    {
        const bool many = p.threads == 1024;
        if (p.tiles > 1)
        {
            norm_mean_kernel<T, WHOLE><<<(int)(a.rows < (1 << 20) ? a.rows : 1 << 20), 1024, 0, st>>>(a);
            go(norm_backward_kernel<T, 1024, 1024, 2, WHOLE, true>);
        }
        else if (p.lanes == 8)
            many ? go(norm_backward_kernel<T, 1024, 8, 1, WHOLE, false>) : go(norm_backward_kernel<T, 256, 8, 1, WHOLE, false>);
        else if (p.lanes == 16)
            many ? go(norm_backward_kernel<T, 1024, 16, 1, WHOLE, false>) : go(norm_backward_kernel<T, 256, 16, 1, WHOLE, false>);
        else if (p.lanes == 32)
            many ? go(norm_backward_kernel<T, 1024, 32, 1, WHOLE, false>) : go(norm_backward_kernel<T, 256, 32, 1, WHOLE, false>);
        else if (p.lanes == 64 && p.pieces == 1)
            many ? go(norm_backward_kernel<T, 1024, 64, 1, WHOLE, false>) : go(norm_backward_kernel<T, 256, 64, 1, WHOLE, false>);
        else if (p.lanes == 64)
            many ? go(norm_backward_kernel<T, 1024, 64, 2, WHOLE, false>) : go(norm_backward_kernel<T, 256, 64, 2, WHOLE, false>);
        else if (p.lanes == 256 && p.pieces == 1)
            many ? go(norm_backward_kernel<T, 1024, 256, 1, WHOLE, false>) : go(norm_backward_kernel<T, 256, 256, 1, WHOLE, false>);
        else if (p.lanes == 256)
            many ? go(norm_backward_kernel<T, 1024, 256, 2, WHOLE, false>) : go(norm_backward_kernel<T, 256, 256, 2, WHOLE, false>);
        else
            p.pieces == 1 ? go(norm_backward_kernel<T, 1024, 1024, 1, WHOLE, false>) : go(norm_backward_kernel<T, 1024, 1024, 2, WHOLE, false>);
    }
    if (a.dw)
    {
        const int groups = (a.width + 31) / 32;
        norm_join_kernel<T><<<dim3(groups < kJoinGrid ? groups : kJoinGrid, (groups + kJoinGrid - 1) / kJoinGrid), 1024, 0, st>>>(a);
    }
}

size_t mean_bytes(const BackPlan& p, int64_t rows)
{
    return p.tiles > 1 ? (size_t)whole16(rows * 4) : 0;
}

}    // namespace

size_t rms_norm_backward_scratch_bytes(const tmi_rms_norm_desc_t& d, bool dw)
{
    const BackPlan p = back_plan(d.dtype, d.rows, d.width, dw);
    return mean_bytes(p, d.rows) + (dw ? (size_t)p.groups * d.width * 4 : 0);
}

const char* launch_rms_norm_backward(hipStream_t st, const tmi_rms_norm_desc_t& d, const void* s, const void* weight, const float* rstd, const void* d_y,
                                     const void* d_sum, void* d_x, void* d_weight, void* scratch)
{
    const BackPlan p = back_plan(d.dtype, d.rows, d.width, d_weight);
    float* mean      = static_cast<float*>(scratch);
    const BackArgs a{ s, weight, d_y, d_sum, rstd, d_x, d_weight, mean, mean + mean_bytes(p, d.rows) / 4, d.ld_sum, d.ld_y, d.ld_x, d.rows, d.width,
                      p.groups, d.weight_offset };
    auto typed = [&](auto type) {
        using T          = decltype(type);
        const bool whole = whole_rows<T>(s, d.width, d.ld_sum) && whole_rows<T>(weight, d.width, d.width) && whole_rows<T>(d_y, d.width, d.ld_y) &&
                           (!d_sum || whole_rows<T>(d_sum, d.width, d.ld_sum)) && (!d_x || whole_rows<T>(d_x, d.width, d.ld_x));
        whole ? launch_typed<T, true>(st, a, p) : launch_typed<T, false>(st, a, p);
    };
    if (d.dtype == TMI_FP16)
        typed(_Float16{});
    else if (d.dtype == TMI_BF16)
        typed(bf16_t{});
    else
        typed(float{});
    return "rms_norm_backward";
}

}    // namespace tmi
