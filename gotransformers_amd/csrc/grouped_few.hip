// Ragged products of few rows with an epilogue (grouped.hip has the others'): W
// streams from memory into MFMA operands, no LDS on its way, and the epilogue's
// thread has four columns of a row.
//
// A workgroup takes NC times 16 columns of one group's matrix and up to RT times 16
// of its rows, the waves splitting the reduction.  Its group is found on the
// device, as in grouped.hip; columns are dealt to the XCDs in turn, so that
// however few rows there are every XCD streams its share of W, and the row tiles of
// a group, a multiple of eight workgroups apart, find W in the same L2.
//
// What bounds it (MI355X): a launch and a wave's trips to memory one after the other.  32 rows of
// 1024 -> 2048 bf16 with bias, SiLU and factor 6.8 us, W's 4 MB alone 0.8: a wave has four steps of the
// reduction, too few for the batch of multiply_rows, and waits for each one's loads; then the factor's.
// 128 workgroups stream W, half of the CUs.  The same in fp32 10.  64 groups of 2048 -> 1024, a row
// each, 58.6, W's 268 MB at 4.6 TB/s.
#include "grouped_rows.h"

namespace gtmoe {

namespace {

constexpr int kWaves = 8;
constexpr int kMostRows = 256;

template <class T, int NC, int RT>
__global__ __launch_bounds__(64 * kWaves) void grouped_few_kernel(GroupedArgs a, int columns)
{
    __shared__ float part[kWaves][16 * RT][16 * NC + 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, i = lane & 15;
    const int tile = blockIdx.x / columns, n0 = (blockIdx.x - tile * columns) * (16 * NC);
    if (n0 >= a.outputs) return;
    // the tile's group: its rows in tiles of 16 RT
    int g = -1, t0 = 0, rows = 0, before = 0;
    for (int e0 = 0; e0 < a.groups; e0 += 64) {
        int lo = 0, hi = 0;
        if (e0 + lane < a.groups) group_rows(a, e0 + lane, lo, hi);
        const int n = (hi - lo + 16 * RT - 1) / (16 * RT);
        int total;
        const int first = before + wave_sum_before(n, total);
        const uint64_t hit = __ballot(tile >= first && tile < first + n);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            g = e0 + src;
            t0 = __builtin_amdgcn_readlane(lo, src) + (tile - __builtin_amdgcn_readlane(first, src)) * (16 * RT);
            rows = min(16 * RT, __builtin_amdgcn_readlane(hi, src) - t0);
            break;
        }
        before += total;
    }
    if (g < 0) return;
    typedef typename T::Store Store;
    f32x4 acc[NC][RT];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int p = 0; p < RT; ++p) acc[c][p] = f32x4{0.f, 0.f, 0.f, 0.f};
    // columns and rows past the last repeat it: their results are not kept
    const Store *w[NC], *x[RT];
#pragma unroll
    for (int c = 0; c < NC; ++c)
        w[c] = reinterpret_cast<const Store *>(a.b) + g * a.group_stride + min(n0 + 16 * c + i, a.outputs - 1) * a.ldb;
#pragma unroll
    for (int p = 0; p < RT; ++p) x[p] = reinterpret_cast<const Store *>(a.a) + (long long)(t0 + min(16 * p + i, rows - 1)) * a.lda;
    const Store *const(&wc)[NC] = w;
    const Store *const(&xc)[RT] = x;
    multiply_rows<T, kWaves, NC, RT>(wc, xc, a.inputs, wave, acc);
    // lane l: row l % 16 of each row tile, columns 4 (l / 16) .. of each column tile
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int p = 0; p < RT; ++p)
            *reinterpret_cast<f32x4 *>(&part[wave][16 * p + i][16 * c + 4 * q]) = acc[c][p];
    __syncthreads();
    for (int o = threadIdx.x; o < 16 * RT * 4 * NC; o += 64 * kWaves) {
        const int r = o / (4 * NC), c = (o - r * (4 * NC)) * 4;
        if (r >= rows || n0 + c >= a.outputs) continue;
        f32x4 s = *reinterpret_cast<const f32x4 *>(&part[0][r][c]);
#pragma unroll
        for (int v = 1; v < kWaves; ++v) s += *reinterpret_cast<const f32x4 *>(&part[v][r][c]);
        float y[4] = {s[0], s[1], s[2], s[3]};
        store_fused<T>(a, g, (long long)t0 + r, n0 + c, y, a.outputs - n0 - c);
    }
}

// Row tiles of a call: at most one partial tile per group.
long long row_tiles(const GroupedArgs &a, int rows) { return a.rows / rows + (a.groups < a.rows ? a.groups : a.rows); }
int columns_of(const GroupedArgs &a, int width) { return ((a.outputs + width - 1) / width + 7) / 8 * 8; }

template <class T, int NC, int RT>
hipError_t launch_shape(const GroupedArgs &a, hipStream_t s)
{
    const int columns = columns_of(a, 16 * NC);
    hipLaunchKernelGGL((grouped_few_kernel<T, NC, RT>), dim3((unsigned)(row_tiles(a, 16 * RT) * columns)), dim3(64 * kWaves), 0, s, a,
                       columns);
    return hipGetLastError();
}

template <class T>
hipError_t launch_values(const GroupedArgs &a, hipStream_t s)
{
    if (a.rows / a.groups <= 16) return launch_shape<T, 1, 1>(a, s);
    return launch_shape<T, 1, 2>(a, s);
}

}  // namespace

// When the few rows' kernel is taken, against tiles of grouped.hip, both with SiLU and a
// factor (us, MI355X):
//   one group: 32 rows always (2048 -> 2048 bf16 9.6 against 11.0, fp32 14.8 against 37.3);
//     more while 32 rows by 16 columns make at most one workgroup per CU (bf16, 128 rows of
//     2048 -> 1024 9.5 against 11.0, 192 14.8 against 11.0), or three in fp32, whose tiles
//     stream W worse (192 rows of 1024 -> 2048 20.2 against 22.3, 256 25.6 against 22.1)
//   groups: a row per group on average (16 of 1024 -> 2048 bf16, 8 rows 8.2 against 9.1, 16
//     rows 12.1 against 13.5, 32 rows 15.3 against 13.6; 64 of 2048 -> 1024, 64 rows, W
//     partly cached, 39.6 against 47.8), two in fp32 (32 rows 33.7 against 33.3, 2 rows 8.3 against 20.9)
//   16-bit rows that LDS-DMA cannot take: up to 192 (1201 -> 1000, 128 rows 12.0 against
//     19.4, 192 19.6 against 19.7; 14 groups of 1000 -> 1201, 64 rows 11.6 against 12.5)
//   more than 64 groups, with a bias and SiLU, rows dealt at random: 48 rows that make at most four
//     workgroups per CU, were each a group's only one (bf16: 128 of 2048 -> 1024, 4 rows 6.5 against 11.8, 16 rows 14.2
//     against 14.3, 24 rows 20.6 against 19.1; 256 of 1024 -> 512, 24 rows 8.5 against 9.9, 128 rows 27.2
//     against 23.4; 128 of 1001 -> 1201, 4 rows 9.2 against 18.2, 24 rows 23.9 against 20.4; 128 of 64 ->
//     8192, a row 4.1 against 6.8, 16 rows 22.5 against 14.3; of 16384 -> 64, 16 rows 22 against 54, 256
//     rows 98 against 76; fp32: 256 of 1024 -> 512, 32 rows 14.9
//     against 23.8, 64 rows 27.7 against 25.8; 1024 of 256 -> 256, 16 rows 9.8 against 19.0, 256 rows 42.0 against 28.5)
bool few_fits(const GroupedArgs &a, int value_bytes, bool staged)
{
    if (a.rows > kMostRows || row_tiles(a, 16) * columns_of(a, 16) > 1 << 22) return false;
    const bool wide = value_bytes == 4;
    if (a.groups > 64) return a.rows <= 48 && a.rows * ((a.outputs + 15) / 16) <= 1024;
    if (!wide && !staged) return a.rows <= 192;
    if (a.groups > 1) return a.rows <= a.groups * (wide ? 2 : 1);
    return a.rows <= 32 || (a.rows + 31) / 32 * ((a.outputs + 15) / 16) <= (wide ? 768 : 256);
}

hipError_t launch_few(const GroupedArgs &a, int values, hipStream_t s)
{
    switch (values) {
    case kValuesBf16: return launch_values<Bf16>(a, s);
    case kValuesF16: return launch_values<F16>(a, s);
    default: return launch_values<F32>(a, s);
    }
}

}  // namespace gtmoe
