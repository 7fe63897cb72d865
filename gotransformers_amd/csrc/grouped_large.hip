// The ragged products of grouped.hip for many tiles of 16-bit values.
//
// A workgroup of eight waves takes tiles of up to 256 x 256 one after the other
// (one workgroup per CU, the grid at most the chip): wave (wm, wn) of 2 x 4
// owns the 32-row blocks wm, wm + 2, ... of the tile and 64 of its columns, so
// that a tile of m rows costs ceil(m / 64) block rows, not four.  The steps of
// consecutive tiles are one stream: while a tile's last two steps multiply,
// the next tile's first two are on their way into LDS, and they land while
// the tile's results leave through 4 KiB of LDS per wave as whole 128-byte
// row pieces.
//
// What bounds it (MI355X, bf16): a step's 64 KiB per CU on their way from L2
// into LDS take about 1.5 us however few of the tile's rows exist, which is
// about what the 256 x 256 tile's MFMAs take (kRowCost).  Long tiles reach 880 to
// 1050 TFLOP/s (8 groups of 2048 x 2048, 16384 rows: weight gradient 131 us,
// forward 148, input gradient 156; a large library product 1010 to 1296), skewed
// small groups 640 to 980 (fp16, 131072 rows over 128 matrices of 768 x 2048:
// forward 421 us, input gradient 483, weight gradient 640).  A last round of tiles
// that does not fill the chip costs as much as a full one: 16 groups of 1024 rows,
// 2048 -> 1024, are 384 tiles for 256 CUs, 85 us in which a CU has work 65 % of the
// time.  The weight gradient of short groups is bound by its results' bytes: 64 fp32
// matrices of 2048 x 1024 from 16384 rows 174 us, 3.6 TB/s, the four steps of a
// tile and the stores of its 256 KiB mostly one after the other, in all CUs at about
// the same time.
//
// ADAPTED costs more than the product beside it (8192 rows of 1024 -> 2048 with
// 12 adapters of rank 64, fp16, 82 us; the plain product 38): thirteen
// groups' rows make some 380 tiles where 256 would do, two rounds of them, rows
// are gathered, and two steps are added to sixteen, whose MFMAs are five times (bf16:
// three) a plain product's of as many ranks.  (With u in two fp16 parts 76 us, but
// a rank far below the row's largest lost its bits.)
//
// Tiles: rows of a group by bm, every XCD an eighth of them in order (the
// hardware hands block b to XCD b % 8), its blocks taking them in turn, so
// that the tiles an XCD works on at a time share rows and columns in its L2.
// bm is the multiple of 64 with the least time for the whole product by the
// rounds of tiles an XCD's CUs go through (kRowCost cycles per step, measured
// against each other, and kTileCost per tile).  The weight gradient's XCDs take
// eighths of the work instead: groups differ in their rows.
#include "grouped_tile.h"

namespace gtmoe {

namespace {

constexpr int SB = 128;       // bytes of reduction per step
constexpr int kThreads = 512;
constexpr int kBm = 256, kBn = 256;
constexpr int kXcds = 8, kCus = 256;

// Cycles of LDS and matrix cores per 128-byte step of a tile of 64 i rows, and
// per tile besides.
__device__ constexpr int kRowCost[5] = {0, 1060, 1380, 1720, 2050};
constexpr int kTileCost = 3000;

// Workgroups of an XCD and this one's place among them.
__device__ __forceinline__ int xcd() { return blockIdx.x & (kXcds - 1); }
__device__ __forceinline__ int place() { return blockIdx.x / kXcds; }
__device__ __forceinline__ int places() { return gridDim.x / kXcds; }

// Tiles of rows: group g's rows in ceil(rows / bm) tiles of equal multiples of
// 64 rows (the last takes what is left).
struct RowTiles {
    const GroupedArgs &a;
    int bm, columns, total;
    // the 64 groups from e0 on, a lane each: first row, end, tiles, rows of
    // a tile, tiles before
    int e0, before, count, lo, hi, n, per, first;

    __device__ __forceinline__ void load(int from)
    {
        e0 = from;
        const int e = e0 + (threadIdx.x & 63);
        lo = hi = 0;
        if (e < a.groups) group_rows(a, e, lo, hi);
    }
    __device__ __forceinline__ void cut(int by)
    {
        n = (hi - lo + by - 1) / by;
        per = n ? ((hi - lo + n - 1) / n + 63) & ~63 : 64;
    }
    __device__ __forceinline__ void place_tiles()
    {
        cut(bm);
        first = before + wave_sum_before(n, count);
    }
    __device__ __forceinline__ RowTiles(const GroupedArgs &a_, int columns_, int steps) : a(a_), columns(columns_)
    {
        // rounds of tiles times a tile's mean cost, for every bm
        int tiles[4] = {0, 0, 0, 0};
        float cycles[4] = {0.f, 0.f, 0.f, 0.f};
        for (int from = 0; from < a.groups; from += 64) {
            load(from);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                cut(64 * (i + 1));
                float c = (float)n * (per == 64 ? kRowCost[1] : per == 128 ? kRowCost[2] : per == 192 ? kRowCost[3] : kRowCost[4]);
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) c += __shfl_xor(c, d);
                cycles[i] += c;
                int t;
                wave_sum_before(n, t);
                tiles[i] += t;
            }
        }
        float best = 0.f;
#pragma unroll
        for (int i = 3; i >= 0; --i) {
            const float each = (float)tiles[i] * columns / kXcds;
            const float cost = tiles[i] ? ceilf(each / places()) * (cycles[i] / tiles[i] * steps + kTileCost) : 0.f;
            if (i == 3 || cost < best) {
                best = cost;
                bm = 64 * (i + 1);
                total = tiles[i];
            }
        }
        bm = __builtin_amdgcn_readfirstlane(bm);
        total = __builtin_amdgcn_readfirstlane(total);
        before = 0;
        load(0);
        place_tiles();
    }
    // tile t of the product (never below one asked for before): its group,
    // first row, rows and column
    __device__ __forceinline__ void find(int t, int &g, int &p0, int &m, int &column)
    {
        const int tile = t / columns;
        column = t - tile * columns;
        while (tile >= before + count && e0 + 64 < a.groups) {
            before += count;
            load(e0 + 64);
            place_tiles();
        }
        const uint64_t hit = __ballot(tile >= first && tile < first + n);
        const int src = hit ? __builtin_ctzll(hit) : 0;
        g = e0 + src;
        const int rows = __builtin_amdgcn_readlane(per, src);
        p0 = __builtin_amdgcn_readlane(lo, src) + (tile - __builtin_amdgcn_readlane(first, src)) * rows;
        m = min(rows, __builtin_amdgcn_readlane(hi, src) - p0);
    }
    __device__ __forceinline__ void range(int &begin, int &end) const
    {
        // (more than the 2^30 tiles a launch is held to: only of offsets that descend)
        const long long all = min((long long)total * columns, 1ll << 30);
        begin = (int)(all * xcd() / kXcds);
        end = (int)(all * (xcd() + 1) / kXcds);
    }
};

// The weight gradient's tiles: `each` per group, of the group's steps plus
// kGroupCost.
constexpr int kGroupCost = 4;
struct MatrixTiles {
    const GroupedArgs &a;
    int each;
    __device__ __forceinline__ long long cost_of(int e) const
    {
        if (e >= a.groups) return 0;
        int lo, hi;
        group_rows(a, e, lo, hi);
        return (long long)each * ((hi - lo + 63) / 64 + kGroupCost);
    }
    static __device__ __forceinline__ long long sum_before(long long v, long long &total)
    {
        const int lane = threadIdx.x & 63;
        long long s = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const long long o = __shfl_up(s, d);
            if (lane >= d) s += o;
        }
        total = __shfl(s, 63);
        return s - v;
    }
    // first tile whose start in the groups' costs is at least `bound`
    __device__ __forceinline__ int tile_at(long long bound) const
    {
        long long before = 0;
        for (int e0 = 0; e0 < a.groups; e0 += 64) {
            const int e = e0 + (threadIdx.x & 63);
            const long long c = cost_of(e);
            long long t;
            const long long first = before + sum_before(c, t);
            const uint64_t hit = __ballot(c > 0 && bound >= first && bound < first + c);
            if (hit) {
                const long long unit = c / each;
                const int tile = e * each + (int)((bound - first + unit - 1) / (unit > 0 ? unit : 1));
                return __builtin_amdgcn_readlane(tile, __builtin_ctzll(hit));
            }
            before += t;
        }
        return a.groups * each;
    }
    // A bound between two XCDs moved to whole rounds of an XCD's workgroups where that is near: with 65 tiles
    // for 32 CUs one tile more would take as long as 32
    __device__ __forceinline__ int whole_rounds(int tile) const
    {
        const int near = min((tile + places() / 2) / places() * places(), a.groups * each);
        return abs(near - tile) <= places() / 8 ? near : tile;
    }
    __device__ __forceinline__ void range(int &begin, int &end) const
    {
        long long all = 0;
        for (int e0 = 0; e0 < a.groups; e0 += 64) {
            long long t;
            sum_before(cost_of(e0 + (threadIdx.x & 63)), t);
            all += t;
        }
        begin = xcd() == 0 ? 0 : whole_rounds(tile_at(all * xcd() / kXcds));
        end = xcd() == kXcds - 1 ? a.groups * each : whole_rounds(tile_at(all * (xcd() + 1) / kXcds));
    }
};

__device__ __forceinline__ const char *scalar(const char *p)
{
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const char *>((uint64_t)hi << 32 | lo);
}

// 16 bytes of a row's results as they were staged: eight values of a 16-bit type S
// = O, or four fp32 ones, to which `add` adds what out holds before the one
// rounding to O.  `left` of them exist.
template <class S, class O>
__device__ __forceinline__ void store_unit(typename O::Store *p, u32x4 v, int left, bool aligned, bool add)
{
    constexpr int unit = 16 / S::kBytes;
    if (left >= unit && aligned) {
        if constexpr (S::kBytes == 2) {
            *reinterpret_cast<u32x4 *>(p) = v;
        } else {
            f32x4 w = __builtin_bit_cast(f32x4, v);
            if constexpr (O::kBytes == 4) {
                if (add) w += *reinterpret_cast<const f32x4 *>(p);
                // not kept in L2, which the operands want (64 matrices of 2048 x 1024,
                // 16384 rows: 176 us against 182)
                __builtin_nontemporal_store(w, reinterpret_cast<f32x4 *>(p));
            } else {
                if (add) {
                    const uint2 o = *reinterpret_cast<const uint2 *>(p);
                    w += f32x4{O::load((uint16_t)o.x), O::load((uint16_t)(o.x >> 16)), O::load((uint16_t)o.y),
                               O::load((uint16_t)(o.y >> 16))};
                }
                *reinterpret_cast<uint2 *>(p) = make_uint2(O::pack(w[0], w[1]), O::pack(w[2], w[3]));
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < unit; ++e)
            if (e < left) {
                if constexpr (S::kBytes == 2) p[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
                else p[e] = O::round((add ? O::load(p[e]) : 0.f) + __uint_as_float(v[e]));
            }
    }
}

// ADAPTED (forward, one matrix for all groups): the groups are the adapters, their
// rows at the places of a.term.index.  The adapter's term is two steps more of
// the same stream, u's parts against the adapter's up matrix.
template <class T, int DIR, bool ADAPTED>
__global__ __launch_bounds__(kThreads) void grouped_large_kernel(GroupedArgs a)
{
    typedef Operand<T, DIR != kGroupedWeightGradient, kBm, kThreads, SB, ADAPTED> A;
    typedef Operand<T, DIR == kGroupedForward, kBn, kThreads, SB> B;
    typedef Operand<F32, true, kBm, kThreads, SB, ADAPTED> U;  // of an adapter's term
    typedef typename T::Store Store;
    constexpr int NJ = 2, KK = SB / 32, L = A::kLoads + B::kLoads;
    __shared__ __attribute__((aligned(1024))) char s0[(kBm + kBn) * SB];
    __shared__ __attribute__((aligned(1024))) char s1[(kBm + kBn) * SB];
    __shared__ __attribute__((aligned(1024))) char so[8 * 4096];

    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave >> 2) * 32, wn = (wave & 3) * 64;
    const int width = DIR == kGroupedForward ? a.outputs : a.inputs;
    const int columns = (width + kBn - 1) / kBn;

    // A tile: rows m0 .. + m of the output buffer (weight gradient: of the
    // group's matrix), columns n0 .. + n, its operands and steps.
    struct Tile {
        int g, m0, n0, m, n, length, steps, extra;  // extra: steps of an adapter's term
    };
    RowTiles rows_of(a, columns, (DIR == kGroupedForward ? a.inputs : a.outputs) * T::kBytes / SB + 1);
    const int strips = (a.outputs + kBm - 1) / kBm;
    const MatrixTiles matrices{a, strips * columns};
    auto find = [&](int t) {
        Tile x;
        if constexpr (DIR == kGroupedWeightGradient) {
            x.g = t / matrices.each;
            const int q = t - x.g * matrices.each;
            x.m0 = q / columns * kBm;
            x.n0 = (q - q / columns * columns) * kBn;
            int lo, hi;
            wave_group_rows(a, x.g, lo, hi);
            x.length = hi - lo;
            x.m = min(kBm, a.outputs - x.m0);
        } else {
            int column;
            rows_of.find(t, x.g, x.m0, x.m, column);
            x.n0 = column * kBn;
            x.length = DIR == kGroupedForward ? a.inputs : a.outputs;
        }
        x.n = min(kBn, width - x.n0);
        x.g = __builtin_amdgcn_readfirstlane(x.g);
        x.m0 = __builtin_amdgcn_readfirstlane(x.m0);
        x.m = __builtin_amdgcn_readfirstlane(x.m);
        x.length = __builtin_amdgcn_readfirstlane(x.length);
        x.steps = max(2, ((x.length + A::kStep - 1) / A::kStep + 1) / 2 * 2);
        x.extra = ADAPTED && x.g < a.term.adapters ? 2 : 0;
        return x;
    };
    auto operand_a = [&](const Tile &x) {
        const Store *p = reinterpret_cast<const Store *>(a.a);
        if constexpr (DIR == kGroupedWeightGradient) {
            int lo, hi;
            wave_group_rows(a, x.g, lo, hi);
            p += __builtin_amdgcn_readfirstlane(lo) * a.lda + x.m0;
        } else if constexpr (!ADAPTED) {
            p += x.m0 * a.lda;
        }
        if constexpr (ADAPTED) return A(p, a.lda, a.rows, a.term.index + x.m0, x.m, x.length);
        else return A(p, a.lda, x.m, x.length);
    };
    auto operand_u = [&](const Tile &x) {
        if constexpr (ADAPTED) return U(a.term.u, a.term.ldu, a.rows, a.term.index + x.m0, x.m, a.term.rank);
        else return 0;
    };
    // step e of the adapter's up matrix: as many ranks as a step of u has
    auto operand_up = [&](const Tile &x, int e) {
        const Store *p = reinterpret_cast<const Store *>(a.term.up) +
                         ((long long)min(x.g, max(a.term.adapters - 1, 0)) * a.outputs + x.n0) * a.term.rank + e * U::kStep;
        return B(p, a.term.rank, x.n, min(U::kStep, a.term.rank - e * U::kStep));
    };
    auto operand_b = [&](const Tile &x) {
        const Store *p = reinterpret_cast<const Store *>(a.b);
        if constexpr (DIR == kGroupedWeightGradient) {
            int lo, hi;
            wave_group_rows(a, x.g, lo, hi);
            p += __builtin_amdgcn_readfirstlane(lo) * a.ldb + x.n0;
        } else {
            p += x.g * a.group_stride + (DIR == kGroupedForward ? x.n0 * a.ldb : (long long)x.n0);
        }
        return B(p, a.ldb, x.n, x.length);
    };

    int begin, end;
    if constexpr (DIR == kGroupedWeightGradient) matrices.range(begin, end);
    else rows_of.range(begin, end);
    begin = __builtin_amdgcn_readfirstlane(begin);
    end = __builtin_amdgcn_readfirstlane(end);
    int t = begin + place();
    if (t >= end) return;

    // the request stream: the tile whose steps are being requested, and the next of them
    Tile rt = find(t);
    A oa = operand_a(rt);
    B ob = operand_b(rt);
    auto ou = operand_u(rt);
    int rk = 0, next_t = t + places();
    auto advance = [&]() {
        if (rk < rt.steps + rt.extra) return;
        rk = 0;
        if (next_t < end) {
            rt = find(next_t);
            next_t += places();
            oa = operand_a(rt);
            ob = operand_b(rt);
            ou = operand_u(rt);
        } else {
            oa.length = ob.length = 0;  // nothing more: requests of no bytes
            rt.steps = 1 << 30;
            rt.extra = 0;
        }
    };
    // step rk of the request stream: of the operands, then of u and the adapter's
    // up matrix (every field that is one for the wave kept scalar)
    auto request_a = [&]() {
        auto q = oa.request(rk);
        if constexpr (ADAPTED) {
            const bool more = rk >= rt.steps;
            static_assert(U::kLoads == A::kLoads, "");
            const auto e = ou.request(more ? rk - rt.steps : 0);
            q.p = scalar(more ? e.p : q.p);
            q.bytes = __builtin_amdgcn_readfirstlane(more ? e.bytes : q.bytes);
#pragma unroll
            for (int i = 0; i < A::kLoads; ++i) q.off[i] = more ? e.off[i] : q.off[i];
        }
        return q;
    };
    auto request_b = [&]() {
        auto q = ob.request(rk);
        if constexpr (ADAPTED) {
            const bool more = rk >= rt.steps;
            const auto e = operand_up(rt, more ? rk - rt.steps : 0).request(0);
            q.p = scalar(more ? e.p : q.p);
            q.bytes = __builtin_amdgcn_readfirstlane(more ? e.bytes : q.bytes);
            q.row = __builtin_amdgcn_readfirstlane(more ? e.row : q.row);
            q.off[0] = more ? e.off[0] : q.off[0];
        }
        return q;
    };

    u32x4 fa[2][4], fb[2][NJ];
    const uint32_t la = A::lane_offset(wm), lb = B::lane_offset(wn);
    // the lane's first eight ranks of u in a step: units 2 h and 2 h + 1 of its row
    const int ur = wm + (lane & 31);
    const uint32_t lu = ur * SB + ((2 * h) ^ swizzle<F32, true, kBm, SB>(ur)) * 16;
    auto landed = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    A::issue(s0, oa.request(0));
    B::issue(s0 + kBm * SB, ob.request(0));
    A::issue(s1, oa.request(1));
    B::issue(s1 + kBm * SB, ob.request(1));
    rk = 2;
    landed();

    Tile x = rt;
    auto run = [&](auto blocks) {
        constexpr int MI = decltype(blocks)::value;
        f32x16 acc[MI][NJ];
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        auto read = [&](const char *s, int kk, int p) {
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[p][i] = A::template read<2>(s, la, i, kk);
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[p][j] = B::read(s + kBm * SB, lb, j, kk);
        };
        auto interleave = [&](auto loads) {
            constexpr int mfmas = MI * NJ, vm = decltype(loads)::value;
            constexpr int ds = MI * A::kReads + NJ * B::kReads;
            constexpr int early = mfmas > 4 ? mfmas - mfmas / 4 : mfmas;  // the last quarter covers the reads' latency
            constexpr int dn = (ds + early - 1) / early, vn = (vm + mfmas - 1) / mfmas;
#pragma unroll
            for (int i = 0; i < mfmas; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                if (i * dn < ds) __builtin_amdgcn_sched_group_barrier(0x100, dn, 0);
                if (i * vn < vm) __builtin_amdgcn_sched_group_barrier(0x20, vn, 0);
            }
        };
        // as in grouped_kernel; the requests run two steps ahead, into the next tile
        auto body = [&](char *cur, const char *next) {
            advance();
            const auto qa = request_a();
            const auto qb = request_b();
            ++rk;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                if (kk + 1 < KK) {
                    read(cur, kk + 1, (kk + 1) & 1);
                } else {
                    landed();
                    A::issue(cur, qa);
                    B::issue(cur + kBm * SB, qb);
                    read(next, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = T::mfma(fb[kk & 1][j], fa[kk & 1][i], acc[i][j]);
                if (kk + 1 < KK) interleave(std::integral_constant<int, 0>());
                else interleave(std::integral_constant<int, L>());
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // a step of the adapter's term: 32 ranks of u, split as they leave LDS
        auto ranks = [&](char *cur, int e) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (e * U::kStep + 16 * g >= a.term.rank) break;
                UpRow<T> b[NJ];
#pragma unroll
                for (int j = 0; j < NJ; ++j) b[j].split(B::read(cur + kBm * SB, lb, j, g));
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    f32x4 v[2];
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                        v[p] = *reinterpret_cast<const f32x4 *>(cur + ((lu ^ (64 * g + 16 * p)) + i * (64 * SB)));
                    RankRow u;
                    u.split(v);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = multiply_ranks<T>(b[j], u, acc[i][j]);
                }
            }
            advance();
            const auto qa = request_a();
            const auto qb = request_b();
            ++rk;
            landed();
            A::issue(cur, qa);
            B::issue(cur + kBm * SB, qb);
        };
        // ADAPTED, asked for now and used at the end: the places of the wave's rows
        // (lane l: rows l and 64 + l of them)
        int at_rows[2];
        if constexpr (ADAPTED) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int row = 64 * (2 * q + h) + wm + (lane & 31);
                at_rows[q] = row < x.m ? a.term.index[x.m0 + row] : 0;
            }
        }
        read(s0, 0, 0);
        for (int k = 0; k < x.steps; k += 2) {
            body(s0, s1);
            body(s1, s0);
        }
        if constexpr (ADAPTED) {
            if (x.extra) {
                ranks(s0, 0);
                ranks(s1, 1);
            }
            if (a.bias) add_bias<T>(acc, a.bias, x.n0 + wn, a.outputs);
        }
        // results: lane l holds row 64 i + wm + l % 32 and, in register r of
        // block (i, j), column wn + 32 j + 8 (r / 4) + 4 (l / 32) + r % 4.  Through
        // LDS (rows of 128 bytes, 16-byte unit u of row r in slot u ^ (r / 2) % 8) to
        // 16 bytes per lane, eight rows of 128 bytes at a time.
        // What the epilogue uses of the lane is made again here, hidden from the
        // compiler: made ahead it was spilled over the steps, and every reload waited
        // for the stores before it (24576 rows over 64 matrices of 512 x 1024 44.8
        // -> 40.5 us, with 12 adapters 114 -> 94).
        char *stage = so + wave * 4096;
        int el = lane;
        asm volatile("" : "+v"(el));
        const int er = el & 31, slot = er * 128 + ((er >> 1) & 7) * 16;
        int places_of[2] = {0, 0};
        if constexpr (ADAPTED) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                places_of[q] = at_rows[q];
                asm volatile("" : "+v"(places_of[q]));
            }
        }
        if (DIR == kGroupedWeightGradient && a.accumulate && x.length == 0) return;
        auto leave = [&](auto staged, auto type) {
            typedef decltype(staged) S;  // the values' type in LDS
            typedef decltype(type) O;
            constexpr int unit = 16 / S::kBytes, each = S::kBytes == 2 ? 2 : 1;  // column blocks per pass
            typename O::Store *out = reinterpret_cast<typename O::Store *>(a.out) +
                                     (DIR == kGroupedWeightGradient ? x.g * a.group_stride : 0) +
                                     (ADAPTED ? 0 : x.m0 * a.ldo) + x.n0;
            const bool aligned = a.ldo % unit == 0 && (reinterpret_cast<uintptr_t>(out) & (unit * O::kBytes - 1)) == 0;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j0 = 0; j0 < NJ; j0 += each) {
#pragma unroll
                    for (int j = j0; j < j0 + each; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const f32x16 &v = acc[i][j];
                            if constexpr (S::kBytes == 2) {
                                *reinterpret_cast<uint2 *>(stage + ((slot ^ (4 * (j - j0) + q) * 16) + (el >> 5) * 8)) =
                                    make_uint2(S::pack(v[4 * q], v[4 * q + 1]), S::pack(v[4 * q + 2], v[4 * q + 3]));
                            } else {
                                *reinterpret_cast<float4 *>(stage + (slot ^ (2 * q + (el >> 5)) * 16)) =
                                    make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                            }
                        }
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const int rr = 8 * p + (el >> 3), u = el & 7;
                        const u32x4 v = *reinterpret_cast<const u32x4 *>(stage + rr * 128 + (u ^ ((rr >> 1) & 7)) * 16);
                        const int row = 64 * i + wm + rr, col = wn + 32 * j0 + unit * u;
                        int to = row;
                        if constexpr (ADAPTED) to = __builtin_amdgcn_ds_bpermute(4 * (32 * (i & 1) + rr), places_of[i >> 1]);
                        if (row < x.m && col < x.n) store_unit<S, O>(out + to * a.ldo + col, v, x.n - col, aligned, a.accumulate);
                    }
                    __builtin_amdgcn_wave_barrier();
                }
        };
        // (a weight gradient in fp32 up to its one rounding, for what it may be added to)
        if (DIR == kGroupedWeightGradient && a.out_f32) leave(F32(), F32());
        else if (DIR == kGroupedWeightGradient) leave(F32(), T());
        else leave(T(), T());
    };
    for (;;) {
        switch ((x.m + 63) / 64) {
        case 1: run(std::integral_constant<int, 1>()); break;
        case 2: run(std::integral_constant<int, 2>()); break;
        case 3: run(std::integral_constant<int, 3>()); break;
        default: run(std::integral_constant<int, 4>()); break;
        }
        t += places();
        if (t >= end) break;
        x = rt;  // the requests have moved to this tile
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // nothing may still be on its way into LDS
}

template <class T>
hipError_t launch_values(const GroupedArgs &a, int direction, hipStream_t s)
{
    const dim3 grid(kCus), block(kThreads);
    switch (direction) {
    case kGroupedForward:
        if (a.term.index) hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedForward, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedForward, false>), grid, block, 0, s, a);
        break;
    case kGroupedInputGradient: hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedInputGradient, false>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedWeightGradient, false>), grid, block, 0, s, a); break;
    }
    return hipGetLastError();
}

}  // namespace

// The weight gradient from 128 tiles on (16 experts of 2048 x 1024, 512 tiles: 64
// rows 32.1 -> 26.7 us, 4096 rows 43.4 -> 35.1; 8 of 512 x 256, 16 tiles: 5.9
// against 10.7), the others from 112 rows per group on average and, by the
// rows' average, more than 128 tiles (64 experts of 2048 -> 1024: 64 rows each
// 54.0 against 66.0, 128 rows 92.3 -> 78.3; 16 of 1024 -> 2048: 128 rows, 128 tiles,
// 21.4 against 23.4, 256 rows, 192 tiles, 37.5 -> 28.1; input gradient of the
// latter, 96 tiles, 28.7 against 33.8).  bf16, against 128 x 128 tiles.
bool large_fits(const GroupedArgs &a, int direction, int value_bytes)
{
    if (value_bytes != 2) return false;
    const long long columns = ((direction == kGroupedForward ? a.outputs : a.inputs) + kBn - 1) / kBn;
    if (direction == kGroupedWeightGradient) {
        const long long tiles = (a.outputs + kBm - 1) / kBm * columns * a.groups;
        return tiles >= 128 && tiles < 1 << 30;
    }
    const long long most = (a.rows / 64 + a.groups) * columns, likely = (a.rows / 256 + a.groups / 2) * columns;
    return a.rows / 112 >= a.groups && likely > 128 && most < 1 << 30;
}

hipError_t launch_large(const GroupedArgs &a, int direction, int values, hipStream_t s)
{
    return values == kValuesBf16 ? launch_values<Bf16>(a, direction, s) : launch_values<F16>(a, direction, s);
}

}  // namespace gtmoe
