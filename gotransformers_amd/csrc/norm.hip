// Root-mean-square norm over plain rows with the residual's addition
// (normalization/rmsnorm.go:33-53 around transformer/block.go:76-77):
//   s = x + residual, rounded to the values' type as it is kept
//   y = s r w, r = 1 / sqrt(mean(s^2) + epsilon), in the values' type and / or in 8 bits
// its gradients, from s:
//   n = s r, g = dy w
//   dx = r (g - n mean(g n)) + ds       (ds: what reaches s past the norm)
//   dw = sum over the rows of dy n
// and the packing of rows that need no norm.
//
// A row stays in registers between its sum and its use: 16 lanes, a wave or a
// workgroup hold one (`TEAM` threads of `NV` times eight values), rows wider than
// 16384 are read again.  The gradient keeps dw's sums in registers over the rows
// of a team, one partial row per workgroup, which a second kernel adds in a fixed
// order; few rows are one workgroup's, which writes dw itself.
//
// What bounds it (MI355X): memory.  8192 x 2048 bf16, residual and sums: forward 28.6 us (134 MB
// at 4.7 TB/s, a large copy reaches 5.0), gradient 31.5 (4.5 TB/s) and its partial rows' sums 4.9,
// which read their lines two to three times over, sixteen columns a workgroup.  2331 x 1201 fp32,
// rows that begin anywhere: 13.2 (3.5 TB/s), 12.4 and 4.3.  Into 8 bits 8192 x 2048 bf16: int8 with
// a scale per 128 columns 20.7, E4M3 with one per row 22.2.  512 rows of 40000, read again: 19.6, gradient 36.7
// and, for the weights, 39 and 5.  One row: 4.0, a launch and two trips to memory.  The gradient's
// gap is the work between a row's loads and its store; the next row's loads ahead of it, or two
// rows at a time, took more registers and fewer waves: 40 to 53 and 54 us.
#include "rows.h"

#include <algorithm>
#include <type_traits>

namespace gtmoe {

namespace {

constexpr int kThreads = 256;

// Totals over a team: 16 lanes, a wave, or the waves of a workgroup that hold a row.
// Waves exchange by LDS, one barrier a total: two totals in turn use two places,
// so that a place is written again only when a barrier has passed since its last
// reading.  Every thread of the workgroup calls them together.
template <int TEAM, int TEAMS>
struct Totals {
    static constexpr int kTeamWaves = TEAM > 64 ? TEAM / 64 : 1, kWaves = kTeamWaves * TEAMS;
    double (*place)[kWaves];
    int turn = 0;

    template <class T>
    __device__ __forceinline__ T *exchange(T v)
    {
        T *p = reinterpret_cast<T *>(place[turn & 1]);
        ++turn;
        if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = v;
        __syncthreads();
        return p;
    }
    // any: whether a team of the workgroup (TEAM <= 64: of the wave) has a total outside [least, most]
    __device__ __forceinline__ float sum(float v, float least, float most, bool &any)
    {
        if constexpr (TEAM <= 64) {
            v = TEAM == 16 ? sixteen_sum(v) : wave_sum(v);
            any = __ballot(!(v >= least && v <= most)) != 0;
            return v;
        } else {
            const float *p = exchange(wave_sum(v));
            float mine = 0.f;
            any = false;
#pragma unroll
            for (int t = 0; t < TEAMS; ++t) {
                float total = 0.f;
#pragma unroll
                for (int w = 0; w < kTeamWaves; ++w) total += p[t * kTeamWaves + w];
                any = any || !(total >= least && total <= most);
                if (TEAMS == 1 || t == (int)(threadIdx.x / TEAM)) mine = total;
            }
            return mine;
        }
    }
    __device__ __forceinline__ float sum(float v)
    {
        if constexpr (TEAM <= 64) {
            return TEAM == 16 ? sixteen_sum(v) : wave_sum(v);
        } else {
            const float *p = exchange(wave_sum(v)) + threadIdx.x / TEAM * kTeamWaves;
            v = 0.f;
#pragma unroll
            for (int w = 0; w < kTeamWaves; ++w) v += p[w];
            return v;
        }
    }
    __device__ __forceinline__ uint32_t most(uint32_t v)
    {
        if constexpr (TEAM <= 64) {
            return TEAM == 16 ? lanes_max(v, 16) : wave_max(v);
        } else {
            const uint32_t *p = exchange(wave_max(v)) + threadIdx.x / TEAM * kTeamWaves;
            v = 0;
#pragma unroll
            for (int w = 0; w < kTeamWaves; ++w) v = max(v, p[w]);
            return v;
        }
    }
    // in 64 bits, for squares that fp32 does not hold
    __device__ double sum64(double v)
    {
#pragma unroll
        for (int d = 1; d < (TEAM < 64 ? TEAM : 64); d <<= 1) v += __shfl_xor(v, d);
        if constexpr (TEAM > 64) {
            const double *p = exchange(v) + threadIdx.x / TEAM * kTeamWaves;
            v = 0;
            for (int w = 0; w < kTeamWaves; ++w) v += p[w];
        }
        return v;
    }
};

constexpr int team_threads(int team) { return team > kThreads ? team : kThreads; }

// A row in a team's registers (NV > 0) or read again each time.
template <int VALUES, int TEAM, int NV>
struct Row {
    Eight<VALUES> v[NV ? NV : 1];
    const void *base;
    long long at;
    int columns, thread;
    float times = 1.f;  // of what is read again

    __device__ __forceinline__ Row(const void *base_, long long at_, int columns_)
        : base(base_), at(at_), columns(columns_), thread(threadIdx.x % TEAM)
    {
    }
    __device__ __forceinline__ int chunks() const { return NV ? NV : ((columns + 7) / 8 + TEAM - 1) / TEAM; }
    __device__ __forceinline__ int column(int i) const { return 8 * (i * TEAM + thread); }
    __device__ __forceinline__ void fill(const void *from, long long row)
    {
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) load_eight(v[i], from, row, column(i), columns);
        }
    }
    // whether the thread has columns in its i-th group
    __device__ __forceinline__ bool any(int i) const { return any_column<VALUES>(column(i), columns); }
    __device__ __forceinline__ Eight<VALUES> get(int i) const
    {
        if constexpr (NV > 0) {
            return v[i];
        } else {
            Eight<VALUES> e;
            load_eight(e, base, at, column(i), columns);
            if (times != 1.f) scale(e, times);
            return e;
        }
    }
    static __device__ __forceinline__ void scale(Eight<VALUES> &e, float by)
    {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = e.get(j) * by;
        e.set(y);
    }
    __device__ __forceinline__ void scale(float by)
    {
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) scale(v[i], by);
        } else {
            times = by;
        }
    }
    // f(i) for every group of eight of the thread; i is a constant of the compiler's
    // where the row is in registers
    template <class F>
    __device__ __forceinline__ void each(F &&f) const
    {
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) f(i);
        } else {
            for (int i = 0; i < chunks(); ++i) f(i);
        }
    }
};

// r = 1 / sqrt(mean(s^2) + epsilon) of a row, as value * times, times a power of two.
struct Inverse {
    float value, times = 1.f;
};
// Squares beyond fp32, or all below it beside no epsilon, are added in 64 bits.  r itself
// may then be none of fp32's normal numbers (rows of size 2^-128 and less, or 2^126 and more):
// the row is left times a power of two, so that s r is what it holds times value.
template <int VALUES, int TEAM, int NV, class T>
__device__ __forceinline__ Inverse inverse_size(Row<VALUES, TEAM, NV> &row, int columns, double epsilon, T &totals)
{
    float sum = 0.f;
    row.each([&](int i) {
        const Eight<VALUES> e = row.get(i);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(e.get(j), e.get(j), sum);
    });
    const float least = epsilon >= 1e-15 ? 0.f : 1e-25f;
    bool any;
    sum = totals.sum(sum, least, 1e37f, any);
    Inverse r{1.f / sqrtf(sum / (float)columns + (float)epsilon)};
    if (any) {
        double wide = 0;
        row.each([&](int i) {
            const Eight<VALUES> e = row.get(i);
#pragma unroll
            for (int j = 0; j < 8; ++j) wide += (double)e.get(j) * (double)e.get(j);
        });
        wide = totals.sum64(wide);
        if (!(sum >= least && sum <= 1e37f)) {
            const double exact = 1.0 / sqrt(wide / columns + epsilon);
            r.times = exact > 0x1p64 ? 0x1p64f : exact < 0x1p-64 ? 0x1p-32f : 1.f;
            r.value = (float)(exact / (double)r.times);
        }
        row.scale(r.times);
    }
    return r;
}

template <int VALUES, int TEAM, int NV>
__global__ __launch_bounds__(team_threads(TEAM)) void norm_forward_kernel(NormArgs a)
{
    constexpr int TEAMS = team_threads(TEAM) / TEAM;
    __shared__ double place[2][Totals<TEAM, TEAMS>::kWaves];
    Totals<TEAM, TEAMS> totals{place};
    for (long long r0 = (long long)blockIdx.x * TEAMS; r0 < a.rows; r0 += (long long)gridDim.x * TEAMS) {
        // teams past the last row work on a row of no columns
        const long long r = r0 + threadIdx.x / TEAM;
        const bool have = r < a.rows;
        const int columns = have ? a.columns : 0;
        Row<VALUES, TEAM, NV> row(a.sums ? a.sums : a.x, r * (a.sums ? a.ldsums : a.ldx), columns);
        if (a.residual || a.sums) {
            row.fill(a.x, r * a.ldx);
            row.each([&](int i) {
                const int c = row.column(i);
                if (!row.any(i)) return;
                Eight<VALUES> e;
                if constexpr (NV > 0) e = row.v[i];
                else load_eight(e, a.x, r * a.ldx, c, columns);
                if (a.residual) {
                    Eight<VALUES> b;
                    load_eight(b, a.residual, r * a.ldresidual, c, columns);
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = e.get(j) + b.get(j);
                    e.set(v);
                }
                if constexpr (NV > 0) row.v[i] = e;
                store_eight(e, a.sums, r * a.ldsums, c, columns);
            });
        } else {
            row.fill(a.x, r * a.ldx);
        }
        float inverse = 1.f;
        if (a.norm) inverse = inverse_size(row, a.columns, a.epsilon, totals).value;
        auto value = [&](int i, float (&y)[8]) {
            const Eight<VALUES> e = row.get(i);
            if (a.norm) {
                Eight<VALUES> w;
                if (a.w) load_eight(w, a.w, 0, row.column(i), columns);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = a.w ? e.get(j) * inverse * w.get(j) : e.get(j) * inverse;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = e.get(j);
            }
        };
        uint32_t most = 0;
        if (a.kept.codes && !a.kept.scale_columns) {
            row.each([&](int i) {
                float y[8];
                value(i, y);
                most = max(most, max(largest_of_four(y), largest_of_four(y + 4)));
            });
            most = totals.most(most);
        }
        row.each([&](int i) {
            float y[8];
            value(i, y);
            if (a.out && row.any(i)) {
                Eight<VALUES> e;
                e.set(y);
                store_eight(e, a.out, r * a.ldo, row.column(i), columns);
            }
            if (a.kept.codes) keep_eight<VALUES>(y, r, row.column(i), columns, a.kept, most);
        });
    }
}

// out[g][c] (+)= sum, rounded once.
template <int VALUES>
__device__ __forceinline__ void store_sum(const AddPartialsArgs &a, int g, int c, double sum)
{
    const long long at = g * a.ldo + c;
    if (a.out_f32) {
        float *o = reinterpret_cast<float *>(a.out) + at;
        *o = (float)(a.accumulate ? *o + sum : sum);
    } else {
        typedef typename Eight<VALUES>::Store Store;
        Eight<VALUES> e;
        Store *o = reinterpret_cast<Store *>(a.out) + at, w[8] = {};
        if (a.accumulate) {
            w[0] = *o;
            __builtin_memcpy(e.raw, w, sizeof w);
            sum += e.get(0);
        }
        const float v[8] = {(float)sum, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        e.set(v);
        __builtin_memcpy(w, e.raw, sizeof w);
        *o = w[0];
    }
}

// One partial row of dw per workgroup (a.partial); of few rows one workgroup, which
// writes dw itself (a.into.out); or none.
template <int VALUES, int TEAM, int NV>
__global__ __launch_bounds__(team_threads(TEAM)) void norm_gradient_kernel(NormGradientArgs a)
{
    constexpr int THREADS = team_threads(TEAM), TEAMS = THREADS / TEAM;
    __shared__ double place[2][Totals<TEAM, TEAMS>::kWaves];
    Totals<TEAM, TEAMS> totals{place};
    __shared__ float part[TEAMS > 1 ? TEAMS : 1][TEAMS > 1 ? TEAM * NV * 8 : 1];
    float dw[NV ? NV : 1][8];
#pragma unroll
    for (int i = 0; i < (NV ? NV : 1); ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
    const float mean = 1.f / (float)a.columns;
    Row<VALUES, TEAM, NV> w(a.w, 0, a.columns);
    if (a.w) w.fill(a.w, 0);
    for (long long r0 = (long long)blockIdx.x * TEAMS; r0 < a.rows; r0 += (long long)gridDim.x * TEAMS) {
        const long long r = r0 + threadIdx.x / TEAM;
        const bool have = r < a.rows;
        const int columns = have ? a.columns : 0;
        // all of a row's loads go out together
        Row<VALUES, TEAM, NV> s(a.s, r * a.lds, columns), dy(a.dy, r * a.lddy, columns), ds(a.ds, r * a.ldds, columns);
        s.fill(a.s, r * a.lds);
        dy.fill(a.dy, r * a.lddy);
        if (a.ds) ds.fill(a.ds, r * a.ldds);
        Inverse size = inverse_size(s, a.columns, a.epsilon, totals);
        // a team past the last row adds nothing to dw (without epsilon its row of zeros has no inverse)
        if (!have) size.value = 0.f;
        const float inverse = size.value;
        if (NV == 0 && a.inverse && threadIdx.x == 0) {
            a.inverse[2 * r] = size.value;
            a.inverse[2 * r + 1] = size.times;
        }
        float dot = 0.f;
        s.each([&](int i) {
            const Eight<VALUES> v = s.get(i), g = dy.get(i), f = a.w ? w.get(i) : v;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float t = g.get(j) * (v.get(j) * inverse);
                dot = a.w ? fmaf(f.get(j), t, dot) : dot + t;
                if constexpr (NV > 0) dw[i][j] += t;
            }
        });
        dot = totals.sum(dot) * mean;
        s.each([&](int i) {
            if (!s.any(i)) return;
            const Eight<VALUES> v = s.get(i), g = dy.get(i), f = a.w ? w.get(i) : v, p = a.ds ? ds.get(i) : v;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float m = v.get(j) * inverse, t = a.w ? g.get(j) * f.get(j) : g.get(j);
                y[j] = fmaf(inverse * fmaf(-m, dot, t), size.times, a.ds ? p.get(j) : 0.f);
            }
            Eight<VALUES> e;
            e.set(y);
            store_eight(e, a.dx, r * a.lddx, s.column(i), columns);
        });
    }
    if constexpr (NV > 0) {
        if (!a.partial && !a.into.out) return;
        const int thread = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
        auto keep = [&](int c, float v) {
            if (a.partial) a.partial[(long long)blockIdx.x * a.columns + c] = v;
            else store_sum<VALUES>(a.into, 0, c, v);
        };
        if constexpr (TEAMS > 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) part[team][column_of<VALUES>(8 * (i * TEAM + thread), j)] = dw[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < a.columns; c += THREADS) {
                float v = 0.f;
#pragma unroll
                for (int t = 0; t < TEAMS; ++t) v += part[t][c];
                keep(c, v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = column_of<VALUES>(8 * (i * TEAM + thread), j);
                    if (c < a.columns) keep(c, dw[i][j]);
                }
        }
    }
}

// Sums over rows by group, in fp64 (fp32 sums of terms that cancel lose the difference's bits; 16
// uneven groups of 16384 x 2048 bf16 16.8 -> 17.7 us, 14 of 2331 x 1201 fp32 12.1 -> 13.6), in two
// steps: a workgroup adds `each` consecutive rows of 512 columns, one partial row for every group
// among them; the pair (workgroup b, group g) has slot b + g, and no other pair has it, since
// rows are in group order.  With v: of the rows' values times v's times r's two inverses.  All
// rows by one workgroup per 512 columns (few rows): it writes the sums themselves (a.into.out),
// zero for the groups without rows.
constexpr int kSumColumns = 512;

template <int VALUES>
__global__ __launch_bounds__(kThreads) void column_sums_kernel(ColumnSumsArgs a)
{
    __shared__ double part[kThreads / 64][kSumColumns];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = blockIdx.x * kSumColumns + 8 * lane;
    const bool any = any_column<VALUES>(c, a.columns), whole = column_of<VALUES>(c, 7) < a.columns;
    const int first = blockIdx.y * a.each, last = min(first + a.each, a.rows);
    for (int g0 = 0; g0 < a.groups; g0 += 64) {
        int lo = 0, hi = 0;
        if (g0 + lane < a.groups) {
            lo = a.offsets ? min(max(a.offsets[g0 + lane], 0), a.rows) : 0;
            hi = a.offsets ? min(max(a.offsets[g0 + lane + 1], lo), a.rows) : a.rows;
        }
        lo = max(lo, first);
        hi = min(hi, last);
        const bool own = a.into.out != nullptr;
        uint64_t todo = __ballot(lo < hi || (own && !a.into.accumulate && g0 + lane < a.groups));
        while (todo) {
            const int src = __builtin_ctzll(todo);
            todo &= todo - 1;
            const int begin = __builtin_amdgcn_readlane(lo, src), end = __builtin_amdgcn_readlane(hi, src);
            double sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            // eight rows' loads of a wave go out together
            constexpr int WAVES = kThreads / 64, AHEAD = 8;
            int r = begin + wave;
            if (whole && !a.v)
                for (; r + (AHEAD - 1) * WAVES < end; r += AHEAD * WAVES) {
                    Eight<VALUES> e[AHEAD];
#pragma unroll
                    for (int x = 0; x < AHEAD; ++x) load_whole_eight(e[x], a.x, (r + x * WAVES) * a.ldx, c);
#pragma unroll
                    for (int x = 0; x < AHEAD; ++x)
#pragma unroll
                        for (int j = 0; j < 8; ++j) sum[j] += (double)e[x].get(j);
                }
            // and the rest's of them, the last row in the place of those past the end, which are not
            // added (16 uneven groups of 16384 x 2048 bf16 with sums in fp32 19.9 -> 16.7 us, fp32
            // 34.2 -> 30.3; 14 of 2331 x 1201 fp32 10.8 -> 11.9)
            if (whole && !a.v && r < end) {
                Eight<VALUES> e[AHEAD];
#pragma unroll
                for (int x = 0; x < AHEAD; ++x) load_whole_eight(e[x], a.x, min(r + x * WAVES, end - 1) * a.ldx, c);
#pragma unroll
                for (int x = 0; x < AHEAD; ++x) {
                    if (r + x * WAVES >= end) continue;
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum[j] += (double)e[x].get(j);
                }
                r = end;
            }
            if (any)
                for (; r < end; r += WAVES) {
                    Eight<VALUES> e;
                    load_eight(e, a.x, r * a.ldx, c, a.columns);
                    if (a.v) {
                        Eight<VALUES> v;
                        load_eight(v, a.v, r * a.ldv, c, a.columns);
                        const float inverse = a.inverse[2 * (long long)r], times = a.inverse[2 * (long long)r + 1];
#pragma unroll
                        for (int j = 0; j < 8; ++j) sum[j] += (double)e.get(j) * (double)(v.get(j) * times * inverse);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) sum[j] += (double)e.get(j);
                    }
                }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j) part[wave][column_of<VALUES>(8 * lane, j)] = sum[j];
            __syncthreads();
            double *out = a.partial + (long long)(blockIdx.y + g0 + src) * a.columns + blockIdx.x * kSumColumns;
            for (int i = threadIdx.x; i < min(kSumColumns, a.columns - blockIdx.x * kSumColumns); i += kThreads) {
                double v = 0;
#pragma unroll
                for (int w = 0; w < kThreads / 64; ++w) v += part[w][i];
                if (own) store_sum<VALUES>(a.into, g0 + src, blockIdx.x * kSumColumns + i, v);
                else out[i] = v;
            }
        }
    }
}

// out[g][c] (+)= the sum of partial rows: 16 columns per workgroup, EACH threads each.
// The partial rows of group g are those of the row ranges it touches.
template <int VALUES, int EACH, class Partial>
__global__ __launch_bounds__(16 * EACH) void add_partials_kernel(AddPartialsArgs a)
{
    __shared__ double part[EACH][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4, g = blockIdx.y;
    const int c = blockIdx.x * 16 + x;
    int begin = 0, end = a.count;
    if (a.each) {
        int lo = a.offsets ? min(max(a.offsets[g], 0), a.rows) : 0;
        int hi = a.offsets ? min(max(a.offsets[g + 1], lo), a.rows) : a.rows;
        begin = lo < hi ? lo / a.each + g : 0;
        end = lo < hi ? (hi - 1) / a.each + g + 1 : 0;
    }
    double sum = 0;
    if (c < a.columns) {
        const Partial *partial = reinterpret_cast<const Partial *>(a.partial) + c;
#pragma unroll 8
        for (int p = begin + y; p < end; p += EACH) sum += (double)partial[(long long)p * a.columns];
    }
    part[y][x] = sum;
    __syncthreads();
    if constexpr (EACH == 64) {
        // the 64 sums of a column, four at a time, then the sixteen of them
        if (y < 16) part[y][x] = (part[y][x] + part[y + 16][x]) + (part[y + 32][x] + part[y + 48][x]);
        __syncthreads();
    }
    if (y == 0 && c < a.columns) {
        sum = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += part[i][x];
        if (begin == end && a.accumulate) return;
        store_sum<VALUES>(a, g, c, sum);
    }
}

// Threads and groups of eight values per thread that hold a row: 16 lanes up to 128
// columns, a wave up to 1024, from there, and while there are few rows, a workgroup.
// (2048 columns by a wave, four groups a lane: the gradient 47.5 us without dw against
// 29.5, fewer waves with so many registers; the forward 29.7 against 29.1, fp32 37.4
// against 34.6.)
constexpr int kFewRows = 512;
struct Shape {
    int team, nv;
};
Shape shape_of(int rows, int columns)
{
    const int eights = (columns + 7) / 8;
    if (eights <= 16) return {16, 1};
    if (eights <= 64) return {64, 1};
    if (rows > kFewRows && eights <= 128) return {64, 2};
    if (eights <= 256) return {256, 1};
    if (eights <= 512) return {256, 2};
    if (eights <= 1024) return {1024, 1};
    if (eights <= 2048) return {1024, 2};
    return {1024, 0};
}

// f(team, nv) as constants
template <class F>
hipError_t with_shape(Shape s, F &&f)
{
#define GTMOE_SHAPE(T, N) \
    if (s.team == T && s.nv == N) return f(std::integral_constant<int, T>(), std::integral_constant<int, N>());
    GTMOE_SHAPE(16, 1)
    GTMOE_SHAPE(64, 1)
    GTMOE_SHAPE(64, 2)
    GTMOE_SHAPE(256, 1)
    GTMOE_SHAPE(256, 2)
    GTMOE_SHAPE(1024, 1)
    GTMOE_SHAPE(1024, 2)
#undef GTMOE_SHAPE
    return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 0>());
}
template <class F>
hipError_t with_values(int values, F &&f)
{
    switch (values) {
    case kValuesBf16: return f(std::integral_constant<int, kValuesBf16>());
    case kValuesF16: return f(std::integral_constant<int, kValuesF16>());
    default: return f(std::integral_constant<int, kValuesF32>());
    }
}

constexpr int kMostBlocks = 1 << 20;

int blocks_of(long long rows, int team)
{
    const int teams = team_threads(team) / team;
    return (int)std::min<long long>((rows + teams - 1) / teams, kMostBlocks);
}

// Workgroups of the gradient with dw, as many partial rows: sixteen waves per CU (8192 x
// 2048 in bf16, us, both kernels: 50.9 with 512 workgroups of four waves, 37.8 with 1024,
// 47.7 with 2048, whose partial rows take longer; 1024 x 16384: 50.7 with 256 of sixteen
// waves, 66 with 512).
constexpr int kGradientWaves = 4096;
int gradient_blocks(int rows, int columns)
{
    const Shape s = shape_of(rows, columns);
    return std::min(blocks_of(rows, s.team), kGradientWaves / (team_threads(s.team) / 64));
}

}  // namespace

hipError_t launch_norm_forward(const NormArgs &a, int values, hipStream_t s)
{
    const Shape shape = shape_of(a.rows, a.columns);
    return with_values(values, [&](auto v) {
        return with_shape(shape, [&](auto team, auto nv) {
            constexpr int T = decltype(team)::value;
            hipLaunchKernelGGL((norm_forward_kernel<decltype(v)::value, T, decltype(nv)::value>), dim3(blocks_of(a.rows, T)),
                               dim3(team_threads(T)), 0, s, a);
            return hipGetLastError();
        });
    });
}

namespace {

// many: partial rows of a group.
template <int V, class Partial>
hipError_t launch_add(const AddPartialsArgs &a, int many, hipStream_t s)
{
    const dim3 grid((a.columns + 15) / 16, a.groups);
    if (many > 32) hipLaunchKernelGGL((add_partials_kernel<V, 64, Partial>), grid, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((add_partials_kernel<V, 16, Partial>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

// (64 rows of 2048 columns in 16 groups 15.1 us by one workgroup per 512 columns, 9.8 by two kernels; 32 rows
// of one group 7.5 and 9.8)
static bool few_sums(int rows, int groups) { return rows <= 64 && groups <= 4; }

int sum_rows_each(int rows, int groups, int columns)
{
    // few rows one range, whose sums need no second kernel; else a workgroup per CU, of 32 rows
    // at least (16384 x 2048 bf16 both kernels, us: 15.2 with
    // 256 workgroups, 16.7 with 512, 18.2 with 1024)
    const int strips = (columns + kSumColumns - 1) / kSumColumns;
    const int slices = std::max(1, 256 / std::min(strips, 256));
    return few_sums(rows, groups) ? 64 : std::max(32, (rows + slices - 1) / slices);
}
size_t sum_bytes(int rows, int groups, int columns)
{
    const int each = sum_rows_each(rows, groups, columns);
    return (size_t)((rows + each - 1) / each + groups) * columns * sizeof(double);
}

hipError_t launch_column_sums(ColumnSumsArgs a, const AddPartialsArgs &add, int values, hipStream_t s)
{
    const bool one = a.rows > 0 && few_sums(a.rows, a.groups);
    if (one) a.into = add;
    return with_values(values, [&](auto v) {
        constexpr int V = decltype(v)::value;
        if (a.rows > 0)
            hipLaunchKernelGGL(column_sums_kernel<V>, dim3((a.columns + kSumColumns - 1) / kSumColumns, (a.rows + a.each - 1) / a.each),
                               dim3(kThreads), 0, s, a);
        return one ? hipGetLastError() : launch_add<V, double>(add, a.rows / a.each / a.groups, s);
    });
}

size_t norm_gradient_bytes(int rows, int columns)
{
    if (rows == 0) return 0;
    if (shape_of(rows, columns).nv) return (size_t)gradient_blocks(rows, columns) * columns * sizeof(float);
    return 2 * (size_t)rows * sizeof(float) + sum_bytes(rows, 1, columns);
}

hipError_t launch_norm_gradient(NormGradientArgs a, float *workspace, const AddPartialsArgs &into, int values, hipStream_t s)
{
    const Shape shape = shape_of(a.rows, a.columns);
    const bool weights = into.out != nullptr;
    int blocks = weights && shape.nv ? gradient_blocks(a.rows, a.columns) : blocks_of(a.rows, shape.team);
    // few rows, four for each of a workgroup's teams: a second launch would take longer
    const bool one = weights && shape.nv && shape.team <= 256 && a.rows > 0 && blocks <= 4;
    if (one) {
        blocks = 1;
        a.into = into;
    } else if (weights) {
        (shape.nv ? a.partial : a.inverse) = workspace;
    }
    return with_values(values, [&](auto v) -> hipError_t {
        constexpr int V = decltype(v)::value;
        if (a.rows > 0) {
            const hipError_t e = with_shape(shape, [&](auto team, auto nv) {
                constexpr int T = decltype(team)::value;
                hipLaunchKernelGGL((norm_gradient_kernel<V, T, decltype(nv)::value>), dim3(blocks), dim3(team_threads(T)), 0, s, a);
                return hipGetLastError();
            });
            if (e != hipSuccess) return e;
        }
        if (!weights || one) return hipSuccess;
        AddPartialsArgs add = into;
        add.columns = a.columns;
        add.groups = 1;
        if (shape.nv || a.rows == 0) {
            add.partial = workspace;
            add.count = a.rows ? blocks : 0;
            return launch_add<V, float>(add, add.count, s);
        }
        ColumnSumsArgs c;
        c.x = a.dy;
        c.ldx = a.lddy;
        c.v = a.s;
        c.ldv = a.lds;
        c.inverse = a.inverse;
        c.partial = reinterpret_cast<double *>(workspace + 2 * (size_t)a.rows);
        c.rows = add.rows = a.rows;
        c.columns = a.columns;
        c.groups = 1;
        c.each = add.each = sum_rows_each(a.rows, 1, a.columns);
        add.partial = c.partial;
        return launch_column_sums(c, add, V, s);
    });
}

}  // namespace gtmoe
