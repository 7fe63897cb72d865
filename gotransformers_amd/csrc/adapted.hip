// A shared projection beside the adapters of many requests:
//   y[t] = W x[t] + b + s_a B_a (A_a x[t]),  a = adapter[t]
// The first kernel makes u[t] = s_a A_a x[t] in fp32; the second the product
// with W, to which it adds B_a u.  For few rows that is adapted_few_kernel here,
// which streams W; for many the tiles of grouped.hip and grouped_large.hip
// with their adapters' epilogue.
//
// The three kernels' times on an MI355X (us): one row of 2048 -> 2048, rank 16, bf16,
// 4.6 and 5.2, which is a launch and two dependent trips to memory each (W's
// 8 MiB alone: 1.6); 64 rows of 48 adapters 4.8 and 9.0, the gathered Up
// rows (2 MiB per 32 of them) in the epilogue; 8192 rows, 12 adapters of rank 64, fp16, sort
// 6.4, down 17.2 (17 MB of rows and, per 16 of them, 128 KiB of Down from L2),
// tiles 82 (grouped_large.hip).
#include "grouped_rows.h"

namespace gtmoe {

namespace {

constexpr int kWaves = 8;
// Up to this many rows the kernel that streams W without LDS: 256 rows of 1024 ->
// 2048 15.1 us against 24.3 with 64 x 64 tiles, 512 rows 29.5 against 16.5.
constexpr int kFewRows = 256;

// From this many rows times ranks on, with a shared matrix, whole 16-byte rows and up
// to kMaxSortedRank ranks, the rows are sorted by adapter (64 adapters, bf16, us;
// runs of 1, 7, 512 and 700 rows of one request):
//                                     sorted             in order
//   8192 rows, 1024 -> 2048, rank 64  97, 106, 73, 96    1269, 374, 95, 98
//   8192 rows, 1024 -> 2048, rank 16  78, 83, 62, 80     212, 133, 73, 75
//   8192 rows, 2048 -> 1024, rank 64  91, 109, 81, 93    760, 249, 85, 93
//   8192 rows, 512 -> 1024, rank 64   49, 52, 43, 48     403, 164, 40, 42
//   4096 rows, 1024 -> 2048, rank 64  72, 78, 50, 57     578, 193, 55, 60
//   2048 rows, 1024 -> 2048, rank 64  67, 72, 44, 50     260, 111, 35, 35
//   2048 rows, 512 -> 1024, rank 64   34, 36, 32, 34     100, 78, 18, 19
// and below it
//   4096 rows, 1024 -> 2048, rank 16  65, 67, 45, 49     101, 68, 41, 43
//   2048 rows, 1024 -> 2048, rank 32  63, 66, 42, 45     100, 59, 29, 29
//   1024 rows, 1024 -> 2048, rank 64  66, 74, 43, 47     190, 86, 28, 29
// Which order the rows come in is known on the device alone.  Near the limit the
// wrong form costs up to 1.8 times the better one when sorted (long runs) and up
// to three times in order (mixed rows).
constexpr long long kSortedValues = 1 << 17;
constexpr int kSortWaves = 16, kSortBins = 1024;

// Rows by adapter (bin `adapters`: none), by one workgroup: every wave counts
// the bins of its stretch of rows, the counts are summed over bins and waves,
// and every wave places its rows.  64 rows of one bin keep their order; rows of
// a bin among mixed ones take their places as they come, which changes no
// result: among sorted rows a row's sums do not depend on the rows beside it.
// (One workgroup: mixed rows of 64 adapters take 6.4 us at 8192 rows of runs of 700, 12
// with every row another's, 63 at 65536 and 224 at 262144.)
__global__ __launch_bounds__(64 * kSortWaves) void adapter_sort_kernel(const int32_t *__restrict__ adapter, int rows, int adapters,
                                                                       int32_t *__restrict__ index, int32_t *__restrict__ sorted,
                                                                       int32_t *__restrict__ offsets)
{
    __shared__ int place[kSortWaves][kSortBins];
    __shared__ int sums[kSortWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bins = adapters + 1;
    for (int i = threadIdx.x; i < kSortWaves * kSortBins; i += 64 * kSortWaves) (&place[0][0])[i] = 0;
    const int each = ((rows + kSortWaves - 1) / kSortWaves + 63) & ~63;
    const int begin = min(rows, wave * each), end = min(rows, begin + each);
    auto bin_of = [&](int t) {
        const int a = t < end ? adapter[t] : -1;
        return a < 0 || a >= adapters ? adapters : a;
    };
    __syncthreads();
    // eight times 64 rows of a wave's stretch are loaded together
    // (a wave's LDS operations stay in order; the fence keeps the compiler to it,
    // for lane 0's writes are the other lanes' next reads)
    auto each_chunk = [&](auto &&take) {
        for (int t = begin; t < end; t += 512) {
            int b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = bin_of(t + 64 * i + lane);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int n = min(64, end - (t + 64 * i));
                if (n <= 0) break;
                const int one = __builtin_amdgcn_readfirstlane(b[i]);
                take(t + 64 * i, b[i], n, one, __ballot(b[i] != one && lane < n) == 0);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
    };
    each_chunk([&](int t0, int b, int n, int one, bool same) {
        if (same) {
            if (lane == 0) place[wave][one] += n;
        } else if (lane < n) {
            atomicAdd(&place[wave][b], 1);
        }
    });
    __syncthreads();
    // a thread per bin: its rows before every wave's, then the bins before it
    int total = 0;
    if (threadIdx.x < bins)
        for (int w = 0; w < kSortWaves; ++w) {
            const int n = place[w][threadIdx.x];
            place[w][threadIdx.x] = total;
            total += n;
        }
    int all;
    int before = wave_sum_before(total, all);
    if (lane == 0) sums[wave] = all;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before += sums[w];
    if (threadIdx.x < bins) {
        offsets[threadIdx.x] = before;
        for (int w = 0; w < kSortWaves; ++w) place[w][threadIdx.x] += before;
        if (threadIdx.x == bins - 1) offsets[bins] = before + total;
    }
    __syncthreads();
    each_chunk([&](int t0, int b, int n, int one, bool same) {
        if (same) {
            const int at = place[wave][one];
            if (lane < n) {
                index[at + lane] = t0 + lane;
                sorted[at + lane] = one;
            }
            if (lane == 0) place[wave][one] = at + n;
        } else if (lane < n) {
            const int at = atomicAdd(&place[wave][b], 1);
            index[at] = t0 + lane;
            sorted[at] = b;
        }
    });
}

template <class T>
__device__ __forceinline__ void load_whole_ranks(const typename T::Store *p, float (&v)[8])
{
    typename T::Store w[8];
    __builtin_memcpy(w, p, sizeof w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = T::load(w[e]);
}

// A workgroup takes `tile` (at most 16) rows and NR times 16 ranks
// (blockIdx.y): every adapter among the rows in turn, its ranks times all the
// rows, the waves splitting the reduction; a row keeps its own adapter's
// products only.
template <class T, int NR>
__global__ __launch_bounds__(64 * kWaves) void adapter_down_kernel(AdapterDownArgs a, int tile)
{
    __shared__ float part[kWaves][16][16 * NR + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, i = lane & 15;
    const int t0 = blockIdx.x * tile, j0 = blockIdx.y * (16 * NR);
    const int rows = min(tile, a.rows - t0);
    typedef typename T::Store Store;
    int mine = -1;
    const int at = t0 + min(i, rows - 1), row = a.index ? a.index[at] : at;
    if (i < rows) {
        mine = a.adapter[at];
        if (mine >= a.adapters) mine = -1;
    }
    const Store *const x[1] = {reinterpret_cast<const Store *>(a.x) + (long long)row * a.ldx};
    f32x4 acc[NR];
#pragma unroll
    for (int p = 0; p < NR; ++p) acc[p] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint64_t todo = __ballot(mine >= 0);
    while (todo) {
        const int cur = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
        const bool here = mine == cur;
        todo &= ~__ballot(here);
        // ranks past the last repeat it: their results are not kept
        const Store *d[NR];
        f32x4 sum[NR][1];
#pragma unroll
        for (int p = 0; p < NR; ++p) {
            d[p] = reinterpret_cast<const Store *>(a.down) +
                   ((long long)cur * a.rank + min(j0 + 16 * p + i, a.rank - 1)) * a.inputs;
            sum[p][0] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const Store *const(&dc)[NR] = d;
        multiply_rows<T, kWaves, NR, 1>(dc, x, a.inputs, wave, sum);
        if (here) {
#pragma unroll
            for (int p = 0; p < NR; ++p) acc[p] = sum[p][0];
        }
    }
    // lane l: row l % 16, ranks 4 (l / 16) ..
#pragma unroll
    for (int p = 0; p < NR; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[wave][i][16 * p + 4 * q + e] = acc[p][e];
    __syncthreads();
    for (int o = threadIdx.x; o < 16 * 16 * NR; o += 64 * kWaves) {
        const int r = o / (16 * NR), c = o - r * (16 * NR);
        if (r < rows && j0 + c < a.ldu) {
            const int ad = a.adapter[t0 + r], to = a.index ? a.index[t0 + r] : t0 + r;
            float v = 0.f;
            if (ad >= 0 && ad < a.adapters && j0 + c < a.rank) {
#pragma unroll
                for (int w = 0; w < kWaves; ++w) v += part[w][r][c];
                v *= a.scales[ad];
            }
            a.u[(long long)to * a.ldu + j0 + c] = v;
        }
    }
}

// NC times 16 columns of W (blockIdx.x) times RT times 16 rows (blockIdx.y), the
// waves splitting the reduction; then a thread per value adds the waves'
// sums, the bias and its row's adapter.  W is read once per RT * 16 rows and x
// once per NC * 16 columns, from memory into MFMA operands without LDS.
template <class T, int NC, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void adapted_few_kernel(GroupedArgs a)
{
    __shared__ float part[WAVES][16 * RT][16 * NC + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, i = lane & 15;
    const int n0 = blockIdx.x * (16 * NC), t0 = blockIdx.y * (16 * RT);
    const int rows = min(16 * RT, a.rows - t0);
    typedef typename T::Store Store;
    f32x4 acc[NC][RT];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int p = 0; p < RT; ++p) acc[c][p] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (a.b) {
        // columns and rows past the last repeat it: their results are not kept
        const Store *w[NC], *x[RT];
#pragma unroll
        for (int c = 0; c < NC; ++c)
            w[c] = reinterpret_cast<const Store *>(a.b) + (long long)min(n0 + 16 * c + i, a.outputs - 1) * a.ldb;
#pragma unroll
        for (int p = 0; p < RT; ++p)
            x[p] = reinterpret_cast<const Store *>(a.a) + (long long)(t0 + min(16 * p + i, rows - 1)) * a.lda;
        const Store *const(&wc)[NC] = w;
        const Store *const(&xc)[RT] = x;
        multiply_rows<T, WAVES, NC, RT>(wc, xc, a.inputs, wave, acc);
    }
    // lane l: row l % 16 of each row tile, columns 4 (l / 16) .. of each column tile
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int p = 0; p < RT; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[wave][16 * p + i][16 * c + 4 * q + e] = acc[c][p][e];
    __syncthreads();
    const AdapterTerm &t = a.term;
    for (int o = threadIdx.x; o < 16 * RT * 16 * NC; o += 64 * WAVES) {
        const int r = o / (16 * NC), c = o % (16 * NC), col = n0 + c;
        if (r >= rows || col >= a.outputs) continue;
        const int row = t0 + r, mine = t.adapter[row];
        const bool has = mine >= 0 && mine < t.adapters;
        Store *out = reinterpret_cast<Store *>(a.out) + row * a.ldo + col;
        if (!a.b && !a.bias && !has) continue;  // nothing to add: left as it is
        float v = a.b ? 0.f : T::load(*out);
        if (a.b) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) v += part[w][r][c];
        }
        if (a.bias) v += T::load(reinterpret_cast<const Store *>(a.bias)[col]);
        if (has) {
            const float *u = t.u + (long long)row * t.ldu;
            const Store *up = reinterpret_cast<const Store *>(t.up) + ((long long)mine * a.outputs + col) * t.rank;
            float d = 0.f;
            int k = 0;
            for (; k + 16 <= t.rank; k += 16) {  // 16 ranks' loads together
                f32x4 uv[4];
                float b[2][8];
#pragma unroll
                for (int e = 0; e < 4; ++e) uv[e] = *reinterpret_cast<const f32x4 *>(u + k + 4 * e);
                load_whole_ranks<T>(up + k, b[0]);
                load_whole_ranks<T>(up + k + 8, b[1]);
#pragma unroll
                for (int e = 0; e < 16; ++e) d = fmaf(uv[e >> 2][e & 3], b[e >> 3][e & 7], d);
            }
            for (; k < t.rank; k += 8) {
                const f32x4 u0 = *reinterpret_cast<const f32x4 *>(u + k), u1 = *reinterpret_cast<const f32x4 *>(u + k + 4);
                float b[8];
                load_ranks<T>(up, k, t.rank, b);
#pragma unroll
                for (int e = 0; e < 4; ++e) d = fmaf(u0[e], b[e], d);
#pragma unroll
                for (int e = 0; e < 4; ++e) d = fmaf(u1[e], b[4 + e], d);
            }
            v += d;
        }
        *out = T::round(v);
    }
}

template <class T, int NR>
hipError_t launch_down(const AdapterDownArgs &a, int tile, hipStream_t s)
{
    const dim3 grid((a.rows + tile - 1) / tile, (a.ldu + 16 * NR - 1) / (16 * NR));
    hipLaunchKernelGGL((adapter_down_kernel<T, NR>), grid, dim3(64 * kWaves), 0, s, a, tile);
    return hipGetLastError();
}

template <class T>
hipError_t launch_down_values(const AdapterDownArgs &a, hipStream_t s)
{
    if (a.index) {
        if (a.rank <= 16) return launch_down<T, 1>(a, 16, s);
        return a.rank <= 32 ? launch_down<T, 2>(a, 16, s) : launch_down<T, 4>(a, 16, s);
    }
    const int tile = a.rows <= 512 ? 1 : a.rows >= 8192 ? 16 : (a.rows + 511) / 512;
    if (a.rows < 512 || a.rank <= 16) return launch_down<T, 1>(a, tile, s);
    return a.rank <= 32 ? launch_down<T, 2>(a, tile, s) : launch_down<T, 4>(a, tile, s);
}

template <class T, int NC, int RT, int WAVES>
hipError_t launch_few_tiles(const GroupedArgs &a, hipStream_t s)
{
    const dim3 grid((a.outputs + 16 * NC - 1) / (16 * NC), (a.rows + 16 * RT - 1) / (16 * RT));
    hipLaunchKernelGGL((adapted_few_kernel<T, NC, RT, WAVES>), grid, dim3(64 * WAVES), 0, s, a);
    return hipGetLastError();
}

// Rows and columns per workgroup by how many workgroups 16 columns of 32 rows
// would give (K = 2048, N = 2048, rank 16, a different adapter per row, bf16, both
// kernels): 64 rows, 256 of them, 16 x 32 13.0 us against 15.6 with 32 x 32 and
// 17.4 with 16 columns of 64 rows; 256 rows, 1024 of them, 31.3, 24.8 and, 32
// columns of 64 rows by 16 waves, 22.2; 128 rows of K = 1024, 512 of them, 13.0, 11.7
// and 14.5.  Up to 16 rows 16 x 16 (one row: 9.2 us).
template <class T>
hipError_t launch_few(const GroupedArgs &a, hipStream_t s)
{
    if (a.rows <= 16) return launch_few_tiles<T, 1, 1, 8>(a, s);
    const long long groups = (long long)((a.outputs + 15) / 16) * ((a.rows + 31) / 32);
    if (groups <= 256) return launch_few_tiles<T, 1, 2, 8>(a, s);
    if (groups <= 512) return launch_few_tiles<T, 2, 2, 8>(a, s);
    return launch_few_tiles<T, 2, 4, 16>(a, s);
}

}  // namespace

hipError_t launch_adapter_down(const AdapterDownArgs &a, int values, hipStream_t s)
{
    if (a.rows == 0) return hipSuccess;
    switch (values) {
    case kValuesBf16: return launch_down_values<Bf16>(a, s);
    case kValuesF16: return launch_down_values<F16>(a, s);
    default: return launch_down_values<F32>(a, s);
    }
}

bool adapted_fits(const GroupedArgs &a, int values)
{
    // launch_down's 16 rows per workgroup; a grid holds 2^32 - 1 threads
    return ((long long)a.rows + 15) / 16 * (64 * kWaves) < 1ll << 32 && grouped_fits(a, kGroupedForward, values);
}

bool adapted_sorts(const GroupedArgs &a, int values)
{
    if (values == kValuesF32 || !a.b || (long long)a.rows * a.term.rank < kSortedValues || a.term.adapters >= kSortBins) return false;
    const AdapterTerm &t = a.term;
    auto whole = [](const void *p, long long stride) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0; };
    return whole(a.a, a.lda) && whole(a.b, a.ldb) && whole(t.up, t.rank) && a.inputs % 8 == 0 && t.rank <= kMaxSortedRank &&
           (long long)a.rows * a.lda < 1 << 30 && (long long)a.rows * t.ldu < 1 << 29;
}

hipError_t launch_adapter_sort(const int32_t *adapter, int rows, int adapters, int32_t *index, int32_t *sorted,
                               int32_t *offsets, hipStream_t s)
{
    hipLaunchKernelGGL(adapter_sort_kernel, dim3(1), dim3(64 * kSortWaves), 0, s, adapter, rows, adapters, index, sorted,
                       offsets);
    return hipGetLastError();
}

hipError_t launch_adapted(const GroupedArgs &a, int values, hipStream_t s)
{
    if (a.rows == 0) return hipSuccess;
    if (a.term.index) return launch_large(a, kGroupedForward, values, s);
    if (a.rows > kFewRows) return launch_grouped(a, kGroupedForward, values, s);
    switch (values) {
    case kValuesBf16: return launch_few<Bf16>(a, s);
    case kValuesF16: return launch_few<F16>(a, s);
    default: return launch_few<F32>(a, s);
    }
}

}  // namespace gtmoe
