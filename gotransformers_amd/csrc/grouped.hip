// Ragged matrix products grouped by expert over plain rows (bf16, fp16 or
// fp32), in the three directions of a projection's training step:
//   forward          y[r]  = W_g x[r]               rows [off_g, off_{g+1})
//   input gradient   dx[r] = W_g^T dy[r]
//   weight gradient  dW_g (+)= sum_r dy[r] x[r]^T
// and, for one group of all rows, the shared projection beside many requests'
// adapters, whose second half (B_a u) the epilogue adds.
//
// One workgroup computes a BM x BN tile of one group's product on the matrix
// cores, fp32 accumulation: v_mfma_f32_32x32x16 for 16-bit values,
// v_mfma_f32_32x32x2_f32 for fp32.  A step takes 128 bytes of reduction (64
// 16-bit values, 32 fp32) of both operands into LDS; two stages, the next
// step's loads in flight while this one multiplies.
//
// An operand lies in memory either with the reduction contiguous (x and W in
// the forward, dy in the input gradient: [m][k], "KC") or with the tile's own
// axis contiguous (W in the input gradient, dy and x in the weight gradient:
// [k][m], "MC").  Both are staged as they lie, in 16-byte units:
//   KC  [m] rows of 128 bytes; a lane's MFMA operand (8 values of k for 16
//       bits, 4 for fp32) is one 16-byte LDS read.  Unit c of row m sits in slot
//       c ^ (m / 2) % 8: the 16 rows a read covers at a time fall on all 64
//       banks once.
//   MC  [k] rows of the tile's width; 16-bit operands are read with the LDS
//       transpose loads (four k of 16 columns per 16 lanes), fp32 ones value by
//       value.  Unit c of row k sits in slot c ^ f(k), f spreading the rows
//       that one read covers over the banks.
// Staging is by LDS-DMA loads where addresses, strides and widths are
// multiples of 16 bytes, else through registers with loads of any alignment.
//
// Row groups are found on the device: the grid holds the most tiles the rows
// can need, every wave scans the offsets for its tile, surplus workgroups end.
#include <type_traits>

#include "grouped.h"

namespace gtmoe {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kRawBufferWord3 = 0x00020000;  // raw (untyped) buffer access on CDNA
constexpr uint32_t kOutside = 0x80000000u;   // a buffer offset past every buffer: reads zeros
constexpr long long kMaxBlocks = (1ll << 32) / 1024 - 1;  // a grid holds 2^32 - 1 threads
constexpr int kStepBytes = 128;              // reduction per step and row

struct Bf16 {
    typedef uint16_t Store;
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ float load(Store v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ Store round(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi)
    {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, bf16x2));
    }
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};

struct F16 {
    typedef uint16_t Store;
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ float load(Store v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ Store round(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi)
    {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, f16x2));
    }
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

struct F32 {
    typedef float Store;
    static constexpr int kBytes = 4;
    static __device__ __forceinline__ float load(Store v) { return v; }
    static __device__ __forceinline__ Store round(float v) { return v; }
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c)
    {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
};

// The rows of group g, held inside the row buffers whatever the offsets say.
__device__ __forceinline__ void group_rows(const GroupedArgs &a, int g, int &lo, int &hi)
{
    lo = 0;
    hi = a.rows;
    if (a.offsets) {
        lo = min(max(a.offsets[g], 0), a.rows);
        hi = min(max(a.offsets[g + 1], lo), a.rows);
    }
}

__device__ __forceinline__ int wave_sum_before(int v, int &total)
{
    const int lane = threadIdx.x & 63;
    int s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    total = __builtin_amdgcn_readlane(s, 63);
    return s - v;
}

// Tile of rows of block b (the hardware hands block b to XCD b % 8): XCD x
// takes the x-th eighth of the row tiles in order, each with its `columns`
// column tiles back to back, so that a group's matrix and a tile's rows are
// fetched once per XCD.  False for the blocks past the last tile.
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

// Slot rotation of unit c of LDS row r (see the head of the file).
template <class T, bool KC, int ROWS>
__device__ __forceinline__ int swizzle(int r)
{
    if constexpr (KC) return (r >> 1) & 7;
    else if constexpr (T::kBytes == 2) return ROWS >= 128 ? (r & 3) << 2 : ROWS == 64 ? ((r >> 1) & 1) << 2 : 0;
    else return ((r >> 2) & 1) << 3;
}

// One operand's way into LDS: ROWS of the tile's axis, kStepBytes of the
// reduction per step, THREADS threads.
template <class T, bool KC, int ROWS, int THREADS>
struct Operand {
    static constexpr int kUnit = 16 / T::kBytes;               // values per 16-byte unit
    static constexpr int kStep = kStepBytes / T::kBytes;       // reduction values per step
    static constexpr int kRowUnits = KC ? 8 : ROWS / kUnit;    // units per LDS row
    static constexpr int kLoads = ROWS * kStepBytes / 16 / THREADS;
    static constexpr int kLoadRows = THREADS / kRowUnits;      // LDS rows between a thread's units
    const char *base;   // the tile's first value at reduction 0
    long long row;      // bytes between rows
    int valid;          // values of the tile's axis that exist
    int length;         // reduction values that exist
    int r0, c;          // the thread's first LDS row, and its unit there (the same for all its rows)
    uint32_t off;       // byte offset of that unit from the step's base

    __device__ __forceinline__ Operand(const void *p, long long stride, int valid_, int length_)
        : base(reinterpret_cast<const char *>(p)), row(stride * T::kBytes), valid(valid_), length(length_)
    {
        static_assert(kLoads * THREADS * 16 == ROWS * kStepBytes && kLoadRows * kRowUnits == THREADS, "");
        r0 = threadIdx.x / kRowUnits;
        c = (threadIdx.x % kRowUnits) ^ swizzle<T, KC, ROWS>(r0);
        off = (uint32_t)r0 * (uint32_t)row + c * 16u;
    }

    // LDS-DMA: every unit lies wholly inside its row or wholly outside
    __device__ __forceinline__ void dma(char *lds, int step) const
    {
        const int k0 = step * kStep, left = max(length - k0, 0);
        const char *p = base + (KC ? (long long)k0 * T::kBytes : k0 * row);
        const int bytes = left == 0 || valid <= 0 ? 0
                          : KC ? (int)((valid - 1) * row) + left * T::kBytes
                               : (int)((min(left, kStep) - 1) * row) + valid * T::kBytes;
        const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), 0, bytes, kRawBufferWord3);
        const bool in = c * kUnit < (KC ? left : valid);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t o = in ? off + (uint32_t)(i * kLoadRows) * (uint32_t)row : kOutside;
            char *to = lds + (i * THREADS + __builtin_amdgcn_readfirstlane(threadIdx.x & ~63)) * 16;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void *)to, 16, o, 0, 0, 0);
        }
    }

    // through registers: units that end inside are read value by value
    __device__ __forceinline__ void fetch(u32x4 (&q)[kLoads], int step) const
    {
        const int k0 = step * kStep, left = length - k0;
        const char *p = base + (KC ? (long long)k0 * T::kBytes : k0 * row);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = r0 + i * kLoadRows;
            const int n = r < (KC ? valid : left) ? (KC ? left : valid) - c * kUnit : 0;
            const char *at = p + r * row + c * 16;
            u32x4 v = {0u, 0u, 0u, 0u};
            if (n >= kUnit) {
                __builtin_memcpy(&v, at, 16);
            } else if (n > 0) {
                if constexpr (T::kBytes == 2) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < n) {
                            uint16_t w;
                            __builtin_memcpy(&w, at + 2 * e, 2);
                            v[e >> 1] |= (uint32_t)w << (16 * (e & 1));
                        }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < n) {
                            uint32_t w;
                            __builtin_memcpy(&w, at + 4 * e, 4);
                            v[e] = w;
                        }
                }
            }
            q[i] = v;
        }
    }
    __device__ __forceinline__ void put(char *lds, const u32x4 (&q)[kLoads]) const
    {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) *reinterpret_cast<u32x4 *>(lds + (i * THREADS + threadIdx.x) * 16) = q[i];
    }

    // The MFMA operand of the 32 rows from m0 on at reduction group kk (32
    // bytes of it: lane l holds row m0 + l % 32, half l / 32 of the group).
    static __device__ __forceinline__ u32x4 read(const char *lds, int m0, int kk)
    {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        if constexpr (KC) {
            const int r = m0 + (lane & 31);
            return *reinterpret_cast<const u32x4 *>(lds + r * kStepBytes + ((2 * kk + h) ^ swizzle<T, KC, ROWS>(r)) * 16);
        } else if constexpr (T::kBytes == 2) {
            // lanes 16 g .. 16 g + 15 read four k of 16 columns, four columns
            // of one k each; lane i of them gets column i's four k
            const int m = m0 + (lane & 16) + 4 * (lane & 3);
            u32x4 v;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int r = 16 * kk + 8 * h + 4 * p + ((lane >> 2) & 3);
                const char *at = lds + r * (ROWS * 2) + ((m >> 3) ^ swizzle<T, KC, ROWS>(r)) * 16 + (m & 4) * 2;
                const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *)const_cast<char *>(at));
                const uint2 w = __builtin_bit_cast(uint2, t);
                v[2 * p] = w.x;
                v[2 * p + 1] = w.y;
            }
            return v;
        } else {
            const int m = m0 + (lane & 31);
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 8 * kk + 4 * h + e;
                v[e] = *reinterpret_cast<const uint32_t *>(lds + r * (ROWS * 4) + ((m >> 2) ^ swizzle<T, KC, ROWS>(r)) * 16 +
                                                           (m & 3) * 4);
            }
            return v;
        }
    }
};

// Four consecutive values of a row of out from column n on, `left` of them
// inside the matrix.
template <class T>
__device__ __forceinline__ void store4(typename T::Store *p, const float (&v)[4], int left, bool aligned)
{
    if (left >= 4 && aligned) {
        if constexpr (T::kBytes == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(T::pack(v[0], v[1]), T::pack(v[2], v[3]));
        else *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) p[e] = T::round(v[e]);
    }
}

template <class T>
__device__ __forceinline__ void load4(const typename T::Store *p, float (&v)[4], int left, bool aligned)
{
    if (left >= 4 && aligned) {
        if constexpr (T::kBytes == 2) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
            v[0] = T::load((uint16_t)w.x);
            v[1] = T::load((uint16_t)(w.x >> 16));
            v[2] = T::load((uint16_t)w.y);
            v[3] = T::load((uint16_t)(w.y >> 16));
        } else {
            const float4 w = *reinterpret_cast<const float4 *>(p);
            v[0] = w.x;
            v[1] = w.y;
            v[2] = w.z;
            v[3] = w.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < left ? T::load(p[e]) : 0.f;
    }
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

// acc += u B_a^T for the rows that have an adapter: per 32-row block, every
// adapter that occurs in it in turn, as fp32 MFMAs over the rank (u stays fp32
// and a 16-bit B converts exactly), its products kept by the rows that are
// its own only, so that no adapter's values reach another's rows.  Returns the
// rows without an adapter (bit i: the lane's row of block i).
template <class T, int MI, int NJ>
__device__ __forceinline__ uint32_t add_adapters(f32x16 (&acc)[MI][NJ], const GroupedArgs &a, int m0, int n0, int m)
{
    uint32_t without = 0;
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const AdapterTerm &t = a.term;
    const typename T::Store *up = reinterpret_cast<const typename T::Store *>(t.up);
    const bool aligned = t.rank % 4 == 0 && (reinterpret_cast<uintptr_t>(t.up) & (4 * T::kBytes - 1)) == 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = m0 + 32 * i + (lane & 31);
        int mine = -1;
        if (row < m) {
            mine = t.adapter[row];
            if (mine >= t.adapters) mine = -1;
        }
        if (mine < 0) without |= 1u << i;
        uint64_t todo = __ballot(mine >= 0);
        while (todo) {
            const int cur = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
            const bool here = mine == cur;
            todo &= ~__ballot(here);
            f32x16 d[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) d[j][r] = 0.f;
            for (int c = 0; c < t.rank; c += 8) {
                const int k = c + 4 * h;
                f32x4 uv = {0.f, 0.f, 0.f, 0.f};
                if (here) uv = *reinterpret_cast<const f32x4 *>(t.u + (long long)row * t.ldu + k);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int col = n0 + 32 * j + (lane & 31);
                    float b[4] = {0.f, 0.f, 0.f, 0.f};
                    if (col < a.outputs && k < t.rank)
                        load4<T>(up + ((long long)cur * a.outputs + col) * t.rank + k, b, t.rank - k, aligned);
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(b[e], uv[e], d[j], 0, 0, 0);
                }
            }
            if (here) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] += d[j][r];
            }
        }
    }
    return without;
}

template <class T, int MI, int NJ>
__device__ __forceinline__ void add_bias(f32x16 (&acc)[MI][NJ], const void *bias, int n0, int n)
{
    const int h = (threadIdx.x >> 5) & 1;
    const typename T::Store *b = reinterpret_cast<const typename T::Store *>(bias);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int col = n0 + 32 * j + 8 * (r >> 2) + 4 * h + (r & 3);
            const float v = col < n ? T::load(b[col]) : 0.f;
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[i][j][r] += v;
        }
}

// BM x BN tile by WM x WN waves.
template <class T, int DIR, int BM, int BN, int WM, int WN, bool DMA, bool ADAPTED>
__global__ __launch_bounds__(64 * WM * WN) void grouped_kernel(GroupedArgs a)
{
    constexpr int THREADS = 64 * WM * WN;
    constexpr int MI = BM / WM / 32, NJ = BN / WN / 32;
    typedef Operand<T, DIR != kGroupedWeightGradient, BM, THREADS> A;
    typedef Operand<T, DIR == kGroupedForward, BN, THREADS> B;
    __shared__ __attribute__((aligned(1024))) char s0[(BM + BN) * kStepBytes];
    __shared__ __attribute__((aligned(1024))) char s1[(BM + BN) * kStepBytes];

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
    auto multiply = [&](const char *s) {
#pragma unroll
        for (int kk = 0; kk < kStepBytes / 32; ++kk) {
            u32x4 fa[MI], fb[NJ];
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[i] = A::read(s, wm + 32 * i, kk);
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[j] = B::read(s + BM * kStepBytes, wn + 32 * j, kk);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = T::mfma(fb[j], fa[i], acc[i][j]);
        }
    };
    if constexpr (DMA) {
        // step k's loads have landed and every wave is done with step k - 1:
        // its buffer takes step k + 1 while step k multiplies
        auto body = [&](char *cur, char *next, int k) {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            if (k + 1 < steps) {
                oa.dma(next, k + 1);
                ob.dma(next + BM * kStepBytes, k + 1);
            }
            multiply(cur);
        };
        if (steps > 0) {
            oa.dma(s0, 0);
            ob.dma(s0 + BM * kStepBytes, 0);
        }
        for (int k = 0; k < steps; k += 2) {
            body(s0, s1, k);
            if (k + 1 < steps) body(s1, s0, k + 1);
        }
    } else {
        u32x4 qa[A::kLoads], qb[B::kLoads];
        auto fetch = [&](int k) {
            oa.fetch(qa, k);
            ob.fetch(qb, k);
        };
        if (steps > 0) fetch(0);
        for (int k = 0; k < steps; ++k) {
            char *s = k & 1 ? s1 : s0;
            oa.put(s, qa);
            ob.put(s + BM * kStepBytes, qb);
            __syncthreads();
            if (k + 1 < steps) fetch(k + 1);
            multiply(s);
        }
    }

    uint32_t skip = 0;
    if constexpr (ADAPTED) {
        if (a.bias) add_bias<T>(acc, a.bias, tile_n + wn, a.outputs);
        const uint32_t without = add_adapters<T>(acc, a, tile_m + wm, tile_n + wn, tile_m + m);
        if (!a.b && !a.bias) skip = without;
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

template <class T, int DIR, int BM, int BN, int WM, int WN, bool DMA, bool ADAPTED = false>
hipError_t launch_tiles(const GroupedArgs &a, hipStream_t s)
{
    const long long blocks = tile_blocks(a, DIR, BM, BN);
    hipLaunchKernelGGL((grouped_kernel<T, DIR, BM, BN, WM, WN, DMA, ADAPTED>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0,
                       s, a);
    return hipGetLastError();
}

template <class T, int DIR>
hipError_t launch_direction(const GroupedArgs &a, hipStream_t s)
{
    // LDS-DMA: 16-byte aligned rows, and no unit partly outside a row
    constexpr int unit = 16 / T::kBytes;
    const bool dma = aligned16(a.a, a.lda * T::kBytes) && aligned16(a.b, a.ldb * T::kBytes) &&
                     (DIR == kGroupedWeightGradient || a.group_stride * T::kBytes % 16 == 0 || a.groups == 1) &&
                     a.inputs % unit == 0 && a.outputs % unit == 0;
    if constexpr (DIR == kGroupedForward)
        if (a.term.adapter)
            return dma ? launch_tiles<T, DIR, 128, 128, 2, 2, true, true>(a, s)
                       : launch_tiles<T, DIR, 128, 128, 2, 2, false, true>(a, s);
    return dma ? launch_tiles<T, DIR, 128, 128, 2, 2, true>(a, s) : launch_tiles<T, DIR, 128, 128, 2, 2, false>(a, s);
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
    return tile_blocks(a, direction, 128, 128) <= kMaxBlocks;
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

// ---------------------------------------------------------------------------
// The adapters' first half: u[t] = s_a A_a x[t].
// ---------------------------------------------------------------------------

namespace {

// 16 bytes of a row's reduction from value k on (zero at and past `length`),
// any alignment.
template <class T>
__device__ __forceinline__ u32x4 load_unit(const typename T::Store *row, int k, int length)
{
    constexpr int unit = 16 / T::kBytes;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (k + unit <= length) {
        __builtin_memcpy(&v, row + k, 16);
    } else if (k < length) {
        if constexpr (T::kBytes == 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < length) v[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (k + e < length) v[e] = __float_as_uint(row[k + e]);
        }
    }
    return v;
}

// c += a b^T over 64 bytes of reduction, 16 x 16: lane l holds 16 bytes
// (quarter l / 16) of row l % 16 of both operands.
template <class T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (std::is_same<T, Bf16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (std::is_same<T, F16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
}

constexpr int kDownWaves = 8;

// A workgroup takes `tile` (at most 16) rows and 16 ranks (blockIdx.y): every
// adapter among the rows in turn, its ranks times all the rows on 16 x 16
// MFMAs, the waves splitting the reduction; a row keeps its own adapter's
// products only.
template <class T>
__global__ __launch_bounds__(64 * kDownWaves) void adapter_down_kernel(AdapterDownArgs a, int tile)
{
    __shared__ float part[kDownWaves][16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, i = lane & 15;
    const int t0 = blockIdx.x * tile, j0 = blockIdx.y * 16;
    const int rows = min(tile, a.rows - t0);
    constexpr int unit = 16 / T::kBytes, step = 4 * unit;
    typedef typename T::Store Store;
    int mine = -1;
    if (i < rows) {
        mine = a.adapter[t0 + i];
        if (mine >= a.adapters) mine = -1;
    }
    const Store *x = reinterpret_cast<const Store *>(a.x) + (long long)(t0 + min(i, rows - 1)) * a.ldx;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    uint64_t todo = __ballot(mine >= 0);
    while (todo) {
        const int cur = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
        const bool here = mine == cur;
        todo &= ~__ballot(here);
        // ranks past the last repeat it: their results are not kept
        const Store *d = reinterpret_cast<const Store *>(a.down) +
                         ((long long)cur * a.rank + min(j0 + i, a.rank - 1)) * a.inputs;
        f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = wave * step; k < a.inputs; k += kDownWaves * step)
            p = mfma16<T>(load_unit<T>(d, k + q * unit, a.inputs), load_unit<T>(x, k + q * unit, a.inputs), p);
        if (here) acc = p;
    }
    // lane l: row l % 16, ranks 4 (l / 16) ..
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][i][4 * q + e] = acc[e];
    __syncthreads();
    const int r = threadIdx.x >> 4, c = threadIdx.x & 15;
    if (r < rows && j0 + c < a.ldu) {
        const int ad = a.adapter[t0 + r];
        float v = 0.f;
        if (ad >= 0 && ad < a.adapters && j0 + c < a.rank) {
#pragma unroll
            for (int w = 0; w < kDownWaves; ++w) v += part[w][r][c];
            v *= a.scales[ad];
        }
        a.u[(long long)(t0 + r) * a.ldu + j0 + c] = v;
    }
}

}  // namespace

hipError_t launch_adapter_down(const AdapterDownArgs &a, int values, hipStream_t s)
{
    if (a.rows == 0) return hipSuccess;
    const int tile = a.rows <= 512 ? 1 : a.rows >= 8192 ? 16 : (a.rows + 511) / 512;
    const dim3 grid((a.rows + tile - 1) / tile, (a.ldu + 15) / 16), block(64 * kDownWaves);
    switch (values) {
    case kValuesBf16: hipLaunchKernelGGL(adapter_down_kernel<Bf16>, grid, block, 0, s, a, tile); break;
    case kValuesF16: hipLaunchKernelGGL(adapter_down_kernel<F16>, grid, block, 0, s, a, tile); break;
    default: hipLaunchKernelGGL(adapter_down_kernel<F32>, grid, block, 0, s, a, tile); break;
    }
    return hipGetLastError();
}

}  // namespace gtmoe
