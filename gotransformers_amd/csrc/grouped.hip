// Ragged matrix products grouped by expert over plain rows (bf16, fp16 or
// fp32), in the three directions of a projection's training step:
//   forward          y[r]  = W_g x[r]               rows [off_g, off_{g+1})
//   input gradient   dx[r] = W_g^T dy[r]
//   weight gradient  dW_g (+)= sum_r dy[r] x[r]^T
// and, for one group of all rows, the shared projection beside many requests'
// adapters, whose second half (B_a u) the epilogue adds.
//
// One workgroup of four waves computes a BM x BN tile of one group's product on
// the matrix cores, fp32 accumulation: v_mfma_f32_32x32x16 for 16-bit values,
// v_mfma_f32_32x32x2_f32 for fp32.  A step takes 128 bytes of reduction (64
// 16-bit values, 32 fp32) of both operands into LDS; two stages, the next
// step's loads in flight while this one multiplies, or four where few
// workgroups share a CU and the loads' latency would show.  Tiles by the rules
// above launch_direction; many 16-bit rows go to grouped_large.hip.
//
// What bounds it (MI355X): a decode batch, the matrices' bytes: 64 rows over 16
// matrices of 2048 x 1024 in bf16 13.0 us, 67 MB at 5.1 TB/s, what a large copy
// reaches.  Fewer row tiles than that leave XCDs idle, each tile's columns being
// one XCD's: two rows of two matrices (8.4 MB, 1.6 us) take 8.4 us, ten of ten
// (42 MB, 8.2 us) 13.5.  fp32, the matrix cores and the tiles' shares: 2331 rows over
// 14 matrices of 1201 x 1000 83, 80 and 89 us (forward, input and weight
// gradient), 63 to 70 TFLOP/s of the 154 a large product reaches.  By the
// counters 28 % of the products are of ragged tiles' missing rows and columns,
// the matrix cores are busy 82, 77 and 68 % of the time their CU has work, and CUs
// have work for 72 to 81 % of the kernel: of 42 to 44 row tiles seven XCDs take six
// each and the last what is left.
//
// Row groups are found on the device: the grid holds the most tiles the rows
// can need, every wave scans the offsets for its tile, surplus workgroups end.
#include "grouped_rows.h"

namespace gtmoe {

namespace {

constexpr int kThreads = 256;                               // of every grouped_kernel
constexpr long long kMaxBlocks = (1ll << 32) / kThreads - 1;  // a grid holds 2^32 - 1 threads
constexpr int SB = 128;                                   // bytes of reduction per step
constexpr int kCus = 256;

// Tile of rows of block b (the hardware hands block b to XCD b % 8): XCD x
// takes the x-th eighth of the row tiles (rounded up: the last XCDs may get less or
// none) in order, each with its `columns` column tiles back to back, so that a
// group's matrix and a tile's rows are fetched once per XCD.  False for the blocks
// past the last tile.
__device__ __forceinline__ bool find_row_tile(const GroupedArgs &a, int bm, int columns, int &g, int &p0, int &m,
                                              int &column)
{
    const int lane = threadIdx.x & 63;
    auto tiles_of = [&](int e) {
        if (e >= a.groups) return 0;
        int lo, hi;
        group_rows(a, e, lo, hi);
        return (hi - lo + bm - 1) / bm;
    };
    int total = 0;
    for (int e0 = 0; e0 < a.groups; e0 += 64) {
        int t;
        wave_sum_before(tiles_of(e0 + lane), t);
        total += t;
    }
    const int j = blockIdx.x >> 3, per = (total + 7) >> 3;
    const int tile = (int)(blockIdx.x & 7) * per + j / columns;
    column = j % columns;
    if (j / columns >= per || tile >= total) return false;
    int before = 0;
    for (int e0 = 0; e0 < a.groups; e0 += 64) {
        const int n = tiles_of(e0 + lane);
        int t;
        const int first = before + wave_sum_before(n, t);
        const uint64_t hit = __ballot(n > 0 && tile >= first && tile < first + n);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            g = e0 + src;
            int lo, hi;
            group_rows(a, g, lo, hi);
            p0 = lo + (tile - __builtin_amdgcn_readlane(first, src)) * bm;
            m = min(bm, hi - p0);
            g = __builtin_amdgcn_readfirstlane(g);
            p0 = __builtin_amdgcn_readfirstlane(p0);
            m = __builtin_amdgcn_readfirstlane(m);
            return true;
        }
        before += t;
    }
    return false;
}

// out (+)= acc for the wave's MI x NJ blocks of 32 x 32 whose first row and
// column are m0 and n0: lane l holds row m0 + 32 i + l % 32 and, in register r
// of block (i, j), column n0 + 32 j + 8 (r / 4) + 4 (l / 32) + r % 4.
// skip: rows of it to leave as they are (bit i: the lane's row of block i).
template <class O, int MI, int NJ>
__device__ __forceinline__ void store_tile(const f32x16 (&acc)[MI][NJ], void *out, long long ldo, int m0, int n0, int m,
                                           int n, bool add, uint32_t skip)
{
    const int lane = threadIdx.x & 63, h = lane >> 5;
    typename O::Store *o = reinterpret_cast<typename O::Store *>(out);
    const bool aligned = ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * O::kBytes - 1)) == 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = m0 + 32 * i + (lane & 31);
        if (row >= m || (skip >> i & 1)) continue;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = n0 + 32 * j + 8 * q + 4 * h;
                if (col >= n) continue;
                typename O::Store *p = o + row * ldo + col;
                float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                if (add) {
                    float w[4];
                    load4<O>(p, w, n - col, aligned);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += w[e];
                }
                store4<O>(p, v, n - col, aligned);
            }
    }
}

// BM x BN tile by WM x WN waves; NS: stages; DA, DB: the operands staged by
// LDS-DMA (both of them with more than two stages).
template <class T, int DIR, int BM, int BN, int WM, int WN, int NS, bool DA, bool DB, bool ADAPTED, bool FUSED>
__global__ __launch_bounds__(64 * WM * WN) void grouped_kernel(GroupedArgs a)
{
    constexpr int THREADS = 64 * WM * WN;
    static_assert(THREADS == kThreads, "");
    constexpr int MI = BM / WM / 32, NJ = BN / WN / 32;
    typedef Operand<T, DIR != kGroupedWeightGradient, BM, THREADS, SB> A;
    typedef Operand<T, DIR == kGroupedForward, BN, THREADS, SB> B;
    // one array per stage, so that the compiler tells their accesses apart
    __shared__ __attribute__((aligned(1024))) char s0[(BM + BN) * SB];
    __shared__ __attribute__((aligned(1024))) char s1[(BM + BN) * SB];
    __shared__ __attribute__((aligned(1024))) char s2[NS > 2 ? (BM + BN) * SB : 16];
    __shared__ __attribute__((aligned(1024))) char s3[NS > 2 ? (BM + BN) * SB : 16];
    constexpr int L = (DA ? A::kLoads : 0) + (DB ? B::kLoads : 0);
    static_assert(NS == 2 || (NS == 4 && DA && DB && 3 * L < 64), "");

    typedef typename T::Store Store;
    const Store *pa = reinterpret_cast<const Store *>(a.a), *pb = reinterpret_cast<const Store *>(a.b);
    int g, m, n, length, tile_m, tile_n;
    char *out = reinterpret_cast<char *>(a.out);
    if constexpr (DIR == kGroupedWeightGradient) {
        // strips of a group's output rows go to the XCDs in turn, each with
        // its column tiles back to back
        const int strips = (a.outputs + BM - 1) / BM, columns = (a.inputs + BN - 1) / BN;
        const int j = blockIdx.x >> 3, strip = (j / columns) * 8 + (blockIdx.x & 7);
        if (strip >= strips * a.groups) return;
        g = strip / strips;
        int lo, hi;
        group_rows(a, g, lo, hi);
        lo = __builtin_amdgcn_readfirstlane(lo);
        length = __builtin_amdgcn_readfirstlane(hi) - lo;
        tile_m = (strip % strips) * BM;
        tile_n = (j % columns) * BN;
        m = a.outputs - tile_m;
        n = a.inputs - tile_n;
        if (a.accumulate && length == 0) return;
        pa += lo * a.lda + tile_m;
        pb += lo * a.ldb + tile_n;
        out += (g * a.group_stride + tile_m * a.ldo + tile_n) * (a.out_f32 ? 4 : T::kBytes);
    } else {
        const int width = DIR == kGroupedForward ? a.outputs : a.inputs;
        int column, p0;
        if (!find_row_tile(a, BM, (width + BN - 1) / BN, g, p0, m, column)) return;
        tile_m = p0;
        tile_n = column * BN;
        n = width - tile_n;
        length = DIR == kGroupedForward ? a.inputs : a.outputs;
        pa += p0 * a.lda;
        pb += g * a.group_stride + (DIR == kGroupedForward ? tile_n * a.ldb : (long long)tile_n);
        out += (p0 * a.ldo + tile_n) * T::kBytes;
    }
    if constexpr (ADAPTED)
        if (!a.b) length = 0;  // the shared product is in out already
    const A oa(pa, a.lda, min(m, BM), length);
    const B ob(pb, a.ldb, min(n, BN), length);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);

    f32x16 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int steps = (length + A::kStep - 1) / A::kStep;
    constexpr int KK = SB / 32;
    u32x4 fa[2][MI], fb[2][NJ];
    const uint32_t la = A::lane_offset(wm), lb = B::lane_offset(wn);
    auto read = [&](const char *s, int kk, int p) {
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[p][i] = A::read(s, la, i, kk);
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[p][j] = B::read(s + BM * SB, lb, j, kk);
    };
    auto multiply = [&](int p) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = T::mfma(fb[p][j], fa[p][i], acc[i][j]);
    };
    // All stages are filled up front, a stage again with step k + NS once step
    // k has been read from it.  A step's MFMA groups run with the next
    // group's operands already on their way from LDS; before its last group every
    // wave has read all of the step and step k + 1 has landed (the loads of at
    // most NS - 2 later steps are still pending), so that the
    // next step's first operands, too, load under MFMAs.  Steps past the end
    // read zeros, and the loop takes NS steps at a time without a way out
    // between them (with one, the accumulators were copied at the join).  An
    // operand staged through registers is loaded at the start of step k and
    // written where LDS-DMA loads are issued.
    u32x4 qa[DA ? 1 : A::kLoads], qb[DB ? 1 : B::kLoads];
    auto fetch = [&](int k) {
        if constexpr (!DA) oa.fetch(qa, k);
        if constexpr (!DB) ob.fetch(qb, k);
    };
    auto fill = [&](char *s, int k) {
        if constexpr (DA) oa.issue(s, oa.request(k));
        else oa.put(s, qa);
        if constexpr (DB) ob.issue(s + BM * SB, ob.request(k));
        else ob.put(s + BM * SB, qb);
    };
    constexpr auto vm_wait = [](int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4); };  // vmcnt(n) lgkmcnt(0)
    auto landed = [&](auto pending) {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(vm_wait(decltype(pending)::value));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    // asks for one MFMA, then its share of the group's LDS reads and memory
    // loads, in turn
    auto interleave = [&](auto loads) {
        constexpr int mfmas = MI * NJ * (T::kBytes == 4 ? 4 : 1), vm = decltype(loads)::value;
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
    auto body = [&](char *cur, const char *next, int k) {
        fetch(k + NS);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            if (kk + 1 < KK) {
                read(cur, kk + 1, (kk + 1) & 1);
            } else {
                landed(std::integral_constant<int, (NS - 2) * L>());
                fill(cur, k + NS);
                read(next, 0, 0);
            }
            multiply(kk & 1);
            if (kk + 1 < KK) interleave(std::integral_constant<int, 0>());
            else interleave(std::integral_constant<int, L>());
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (steps > 0) {
        fetch(0);
        fill(s0, 0);
        fetch(1);
        fill(s1, 1);
        if constexpr (NS > 2) {
            fill(s2, 2);
            fill(s3, 3);
        }
        landed(std::integral_constant<int, NS == 2 ? 0 : (NS - 1) * L>());
        read(s0, 0, 0);
    }
    for (int k = 0; k < steps; k += NS) {
        body(s0, s1, k);
        body(s1, NS > 2 ? s2 : s0, k + 1);
        if constexpr (NS > 2) {
            body(s2, s3, k + 2);
            body(s3, s0, k + 3);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // nothing may still be on its way into LDS

    uint32_t skip = 0;
    if constexpr (ADAPTED) {
        if (a.bias) add_bias<T>(acc, a.bias, tile_n + wn, a.outputs);
        const uint32_t without = add_adapters<T>(acc, a, tile_m + wm, tile_n + wn, tile_m + m);
        if (!a.b && !a.bias) skip = without;
    }
    if constexpr (FUSED) {
        static_assert((BM + BN) * SB >= THREADS * 64, "4 KiB for every wave");
        __syncthreads();  // every wave has read its last operands
        finish_blocks<T, MI, NJ, 32, -1, false>(acc, a, g, tile_m, wm, min(m, BM), tile_n, wn, min(n, BN), s0 + wave * 4096,
                                                threadIdx.x & 63);
        return;
    }
    if (DIR == kGroupedWeightGradient && a.out_f32)
        store_tile<F32>(acc, out, a.ldo, wm, wn, m, n, a.accumulate, skip);
    else
        store_tile<T>(acc, out, a.ldo, wm, wn, m, n, a.accumulate, skip);
}

bool aligned16(const void *p, long long stride_bytes)
{
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride_bytes & 15) == 0;
}

// Whether every row an epilogue of 16-bit values reads or writes is whole 16 bytes.
bool whole_epilogue(const GroupedArgs &a)
{
    const Epilogue &e = a.epilogue;
    auto whole = [](const void *p, long long stride) { return !p || aligned16(p, stride * 2); };
    return !e.on || (a.outputs % 8 == 0 && whole(a.out, a.ldo) && whole(e.factor, e.ldfactor) && whole(e.residual, e.ldresidual) &&
                     whole(e.products, e.ldproducts));
}

// Workgroups of a product in bm x bn tiles: at most one partial tile per group.
long long tile_blocks(const GroupedArgs &a, int direction, int bm, int bn)
{
    if (direction == kGroupedWeightGradient) {
        const long long strips = (long long)((a.outputs + bm - 1) / bm) * a.groups;
        return (strips + 7) / 8 * 8 * ((a.inputs + bn - 1) / bn);
    }
    const int width = direction == kGroupedForward ? a.outputs : a.inputs;
    const long long tiles = a.rows / bm + (a.groups < a.rows ? a.groups : a.rows);
    return (tiles + 7) / 8 * 8 * ((width + bn - 1) / bn);
}

template <class T, int DIR, int BM, int BN, int WM, int WN, int NS, bool DA, bool DB, bool ADAPTED, bool FUSED>
hipError_t launch_tiles(const GroupedArgs &a, hipStream_t s)
{
    const long long blocks = tile_blocks(a, DIR, BM, BN);
    hipLaunchKernelGGL((grouped_kernel<T, DIR, BM, BN, WM, WN, NS, DA, DB, ADAPTED, FUSED>), dim3((unsigned)blocks),
                       dim3(64 * WM * WN), 0, s, a);
    return hipGetLastError();
}

// NS: stages where both operands take LDS-DMA loads.
template <class T, int DIR, int BM, int BN, int WM, int WN, int NS, bool ADAPTED = false, bool FUSED = false>
hipError_t launch_staged(const GroupedArgs &a, bool da, bool db, hipStream_t s)
{
    if constexpr (DIR == kGroupedForward && !ADAPTED && !FUSED)
        if (a.epilogue.on) return launch_staged<T, DIR, BM, BN, WM, WN, NS, false, true>(a, da, db, s);
    if (da && db) return launch_tiles<T, DIR, BM, BN, WM, WN, NS, true, true, ADAPTED, FUSED>(a, s);
    return db ? launch_tiles<T, DIR, BM, BN, WM, WN, 2, false, true, ADAPTED, FUSED>(a, s)
              : launch_tiles<T, DIR, BM, BN, WM, WN, 2, false, false, ADAPTED, FUSED>(a, s);
}

// The tile by type, rows per group and number of tiles (times in us, MI355X):
//   fp32  64 x 64: the matrix cores are so much slower here that small tiles lose
//     nothing and waste less (14 experts of 1000 -> 1201, 2331 rows: forward 71
//     against 126 with 128 x 128; 16 of 1024 -> 2048, 4096 rows: 159 against 230).
//     Up to 32 rows per group 32 x 128 with four stages, to stream the weights
//     (64 of 2048 -> 1024, 1024 rows: 107 against 150).
//   16 bits, large tiles where large_fits says so; else
//     64 x 64 up to 48 rows per group (16 of 1024 -> 2048, 512 rows: 14.2 against
//     17.5 with 128 x 128) or while 128 x 128 would give fewer than 128 tiles
//     (8 of 256 -> 512, 2048 rows: 6.0 against 7.7); with four stages while
//     the tiles are at most two per CU, where the loads in flight bound it (16
//     of 1024 -> 2048, 64 rows, input gradient: 13.5 against 20.0; 64 of 1024 ->
//     512, 100 rows, 1024 tiles: 15.0 against 13.2),
//     64 x 128 up to 192 rows per group (14 of 1000 -> 1201, 2331 rows: 25.8
//     against 28.2), and for the weight gradient (12000 rows: 71 against 80),
//     128 x 128 beyond (the same, input gradient: 61 against 69).
template <class T, int DIR>
hipError_t launch_direction(const GroupedArgs &a, hipStream_t s)
{
    // LDS-DMA: 16-byte aligned rows, and no unit partly outside a row
    constexpr int unit = 16 / T::kBytes;
    const bool groups = a.groups == 1 || a.group_stride % unit == 0;
    const int width_a = DIR == kGroupedForward ? a.inputs : a.outputs;
    const bool da = aligned16(a.a, a.lda * T::kBytes) && width_a % unit == 0;
    const bool db = aligned16(a.b, a.ldb * T::kBytes) && a.inputs % unit == 0 && (DIR == kGroupedWeightGradient || groups);
    if constexpr (DIR == kGroupedForward)
        if (a.term.adapter) {
            // 64 x 64: the adapters' term wants many waves (512 rows of 1024 -> 2048:
            // 16.5 us against 25.7 with 128 x 128; 8192: 84.8 against 89.2)
            return tile_blocks(a, DIR, 64, 64) <= 2 * kCus ? launch_staged<T, DIR, 64, 64, 2, 2, 4, true>(a, da, db, s)
                                                           : launch_staged<T, DIR, 64, 64, 2, 2, 2, true>(a, da, db, s);
        }
    if constexpr (DIR == kGroupedForward)
        if (a.epilogue.on && few_fits(a, T::kBytes, da && db))
            return launch_few(a, values_of<T>(), s);
    const long long each = a.rows / a.groups;
    if constexpr (T::kBytes == 4) {
        if constexpr (DIR != kGroupedWeightGradient)
            if (each <= 32) return launch_staged<T, DIR, 32, 128, 1, 4, 4>(a, da, db, s);
        return launch_staged<T, DIR, 64, 64, 2, 2, 2>(a, da, db, s);
    } else {
        if (da && db && large_fits(a, DIR, T::kBytes) && (DIR != kGroupedForward || whole_epilogue(a)))
            return launch_large(a, DIR, values_of<T>(), s);
        if constexpr (DIR == kGroupedWeightGradient) {
            if (tile_blocks(a, DIR, 128, 128) < 256) return launch_staged<T, DIR, 64, 64, 2, 2, 2>(a, da, db, s);
            return launch_staged<T, DIR, 64, 128, 2, 2, 2>(a, da, db, s);
        } else {
            const int width = DIR == kGroupedForward ? a.outputs : a.inputs;
            const long long likely = (a.rows / 128 + a.groups / 2) * ((width + 127) / 128);
            if (each <= 48 || likely < 128)
                return tile_blocks(a, DIR, 64, 64) <= 2 * kCus ? launch_staged<T, DIR, 64, 64, 2, 2, 4>(a, da, db, s)
                                                               : launch_staged<T, DIR, 64, 64, 2, 2, 2>(a, da, db, s);
            if (each <= 192) return launch_staged<T, DIR, 64, 128, 2, 2, 2>(a, da, db, s);
            return launch_staged<T, DIR, 128, 128, 2, 2, 2>(a, da, db, s);
        }
    }
}

template <class T>
hipError_t launch_values(const GroupedArgs &a, int direction, hipStream_t s)
{
    switch (direction) {
    case kGroupedForward: return launch_direction<T, kGroupedForward>(a, s);
    case kGroupedInputGradient: return launch_direction<T, kGroupedInputGradient>(a, s);
    default: return launch_direction<T, kGroupedWeightGradient>(a, s);
    }
}

}  // namespace

bool grouped_fits(const GroupedArgs &a, int direction, int values)
{
    return tile_blocks(a, direction, 32, 64) <= kMaxBlocks;  // no tile is smaller
}

hipError_t launch_grouped(const GroupedArgs &a, int direction, int values, hipStream_t s)
{
    if (direction != kGroupedWeightGradient && a.rows == 0) return hipSuccess;
    switch (values) {
    case kValuesBf16: return launch_values<Bf16>(a, direction, s);
    case kValuesF16: return launch_values<F16>(a, direction, s);
    default: return launch_values<F32>(a, direction, s);
    }
}

}  // namespace gtmoe
