// Parts the ragged products' kernels share: the values' types, an operand's way
// from memory through LDS into MFMA operands, and the epilogues.
//
// An operand lies in memory either with the reduction contiguous (x and W in
// the forward, dy in the input gradient: [m][k], "KC") or with the tile's own
// axis contiguous (W in the input gradient, dy and x in the weight gradient:
// [k][m], "MC").  Both are staged as they lie, SB bytes of reduction per step
// (KC) or as many rows of it (MC), in 16-byte units:
//   KC  [m] rows of SB bytes; a lane's MFMA operand (8 values of k for 16
//       bits, 4 for fp32) is one 16-byte LDS read.  With 128-byte rows unit c of row
//       m sits in slot c ^ (m / 2) % 8: the 16 rows a read covers at a time fall on
//       all 64 banks once.
//   MC  [k] rows of the tile's width; 16-bit operands are read with the LDS
//       transpose loads (four k of 16 columns per 16 lanes), fp32 ones value by
//       value.  Unit c of row k sits in slot c ^ f(k), f spreading the rows
//       that one read covers over the banks.
// (Counters: no LDS bank conflicts in grouped_kernel, in any direction; in
// grouped_large_kernel the epilogue's, 3 to 22 % of its LDS cycles.)  Staging is by LDS-DMA
// loads where an operand's addresses, strides and contiguous width are
// multiples of 16 bytes, else through registers with loads of any alignment.
#pragma once

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

// The matrix cores take an fp16 factor below 2^-14 exactly, but with the exponent of
// 2^-14: a sum with it is rounded at 2^-38 of the other factor.
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
// The same of a group that is one for the whole wave, by scalar loads: they do
// not wait behind the wave's own loads and stores.
__device__ __forceinline__ void wave_group_rows(const GroupedArgs &a, int g, int &lo, int &hi)
{
    const __attribute__((address_space(4))) int32_t *p =
        (const __attribute__((address_space(4))) int32_t *)(a.offsets) + __builtin_amdgcn_readfirstlane(g);
    lo = min(max(p[0], 0), a.rows);
    hi = min(max(p[1], lo), a.rows);
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

// Slot rotation of unit c of LDS row r (see the head of the file).
template <class T, bool KC, int ROWS, int SB>
__device__ __forceinline__ int swizzle(int r)
{
    if constexpr (KC) return SB == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
    else if constexpr (T::kBytes == 2) return ROWS >= 128 ? (r & 3) << 2 : ROWS == 64 ? ((r >> 1) & 1) << 2 : 0;
    else return ((r >> 2) & 1) << 3;
}

// One operand's way into LDS: ROWS of the tile's axis, SB of the
// reduction per step, THREADS threads.
// GATHER (KC only): the tile's rows lie at the places an index gives.
template <class T, bool KC, int ROWS, int THREADS, int SB, bool GATHER = false>
struct Operand {
    static constexpr int kUnit = 16 / T::kBytes;               // values per 16-byte unit
    static constexpr int kStep = SB / T::kBytes;       // reduction values per step
    static constexpr int kRowUnits = KC ? SB / 16 : ROWS / kUnit;    // units per LDS row
    static constexpr int kLoads = ROWS * SB / 16 / THREADS;
    static constexpr int kReads = KC ? 1 : T::kBytes;            // LDS reads per MFMA operand
    static constexpr int kLoadRows = THREADS / kRowUnits;      // LDS rows between a thread's units
    const char *base;   // the tile's first value at reduction 0
    long long row;      // bytes between rows
    int valid;          // values of the tile's axis that exist
    int length;         // reduction values that exist
    int r0, c;          // the thread's first LDS row, and its unit there (the same for all its rows)
    uint32_t off;       // byte offset of that unit from the step's base
    int rows;           // GATHER: rows of the whole matrix
    uint32_t offs[GATHER ? kLoads : 1];  // GATHER: the offsets of all the thread's units

    __device__ __forceinline__ Operand(const void *p, long long stride, int valid_, int length_)
        : base(reinterpret_cast<const char *>(p)), row(stride * T::kBytes), valid(valid_), length(length_)
    {
        static_assert(kLoads * THREADS * 16 == ROWS * SB && kLoadRows * kRowUnits == THREADS, "");
        r0 = threadIdx.x / kRowUnits;
        c = (threadIdx.x % kRowUnits) ^ swizzle<T, KC, ROWS, SB>(r0);
        off = (uint32_t)r0 * (uint32_t)row + c * 16u;
    }
    // rows index[0 .. valid_) of a matrix of rows_ rows (less than 2^31 bytes)
    __device__ __forceinline__ Operand(const void *p, long long stride, int rows_, const int32_t *index, int valid_, int length_)
        : Operand(p, stride, valid_, length_)
    {
        static_assert(GATHER && KC, "");
        rows = rows_;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = r0 + i * kLoadRows;
            offs[i] = r < valid ? (uint32_t)index[r] * (uint32_t)row + c * 16u : kOutside;
        }
    }

    // LDS-DMA of one step: the buffer its offsets are checked against (every
    // unit lies wholly inside its row or wholly outside) and the thread's
    // first offset in it.
    struct Request {
        const char *p;
        int bytes;
        uint32_t row;
        uint32_t off[GATHER ? kLoads : 1];
    };
    __device__ __forceinline__ Request request(int step) const
    {
        const int k0 = step * kStep, left = max(length - k0, 0);
        const char *p = base + (KC ? (long long)k0 * T::kBytes : k0 * row);
        const int bytes = left == 0 || valid <= 0 ? 0
                          : KC ? (int)((valid - 1) * row) + left * T::kBytes
                               : (int)((min(left, kStep) - 1) * row) + valid * T::kBytes;
        const bool in = c * kUnit < (KC ? left : valid);
        if constexpr (GATHER) {
            Request q{p, left ? (int)((rows - 1) * row) + left * T::kBytes : 0, 0, {}};
#pragma unroll
            for (int i = 0; i < kLoads; ++i) q.off[i] = in ? offs[i] : kOutside;
            return q;
        } else {
            // (kOutside plus the rows' offsets stays outside: they are below 2^30)
            return {p, bytes, (uint32_t)row, {in ? off : kOutside}};
        }
    }
    static __device__ __forceinline__ void issue(char *lds, const Request &q)
    {
        const __amdgpu_buffer_rsrc_t src =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(q.p), 0, q.bytes, kRawBufferWord3);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t o = GATHER ? q.off[GATHER ? i : 0] : q.off[0] + (uint32_t)(i * kLoadRows) * q.row;
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

    // The lane's byte offset in a stage of its MFMA operand of the 32 rows from
    // m0 on (lane l holds row m0 + l % 32, half l / 32 of a reduction group of 32
    // bytes) at group 0; m0 a multiple of 32.
    static __device__ __forceinline__ uint32_t lane_offset(int m0)
    {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        if constexpr (KC) {
            const int r = m0 + (lane & 31);
            return r * SB + (h ^ swizzle<T, KC, ROWS, SB>(r)) * 16;
        } else if constexpr (T::kBytes == 2) {
            // lanes 16 g .. 16 g + 15 read four k of 16 columns, four columns
            // of one k each; lane i of them gets column i's four k
            const int r = 8 * h + ((lane >> 2) & 3), m = m0 + (lane & 16) + 4 * (lane & 3);
            return r * (ROWS * 2) + ((m >> 3) ^ swizzle<T, KC, ROWS, SB>(r)) * 16 + (m & 4) * 2;
        } else {
            const int r = 4 * h, m = m0 + (lane & 31);
            return r * (ROWS * 4) + ((m >> 2) ^ swizzle<T, KC, ROWS, SB>(r)) * 16 + (m & 3) * 4;
        }
    }
    // The operand at reduction group kk of the 32-row block i * EACH blocks behind
    // the one `at` is the lane offset of (the slot rotations repeat every 16
    // rows of a KC stage and leave the low bits of a group number alone; the
    // rotations of an MC stage stay inside 128 or 256 bytes and repeat with
    // k, so the block's column offset is exchanged in the slot's own bits).
    template <int EACH = 1>
    static __device__ __forceinline__ u32x4 read(const char *lds, uint32_t at, int i, int kk)
    {
        if constexpr (KC) {
            return *reinterpret_cast<const u32x4 *>(lds + ((at ^ (kk * 32)) + i * (EACH * 32 * SB)));
        } else if constexpr (T::kBytes == 2) {
            u32x4 v;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const char *from = lds + ((at ^ (i * (EACH * 64))) + (16 * kk + 4 * p) * (ROWS * 2));
                const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4 *)const_cast<char *>(from));
                const uint2 w = __builtin_bit_cast(uint2, t);
                v[2 * p] = w.x;
                v[2 * p + 1] = w.y;
            }
            return v;
        } else {
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = *reinterpret_cast<const uint32_t *>(lds + ((at ^ (i * (EACH * 128))) + (8 * kk + e) * (ROWS * 4)));
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

// Eight values of an adapter's up row from rank k on, zero at and past `rank`,
// any alignment.
template <class T>
__device__ __forceinline__ void load_ranks(const typename T::Store *row, int k, int rank, float (&v)[8])
{
    typename T::Store w[8];
    if (k + 8 <= rank) {
        __builtin_memcpy(w, row + k, sizeof w);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = k + e < rank ? row[k + e] : (typename T::Store)0;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = T::load(w[e]);
}

// The adapters' product on the 16-bit matrix cores, sixteen ranks at a time: a
// lane of half h = l / 32 holds ranks k .. k + 7, k = c + 8 h, of one row of u and
// of one row of the adapter's up matrix.  u, which is fp32, enters as three bf16
// numbers whose sum it is (each cut off after eight bits, the rest exact, 24 bits in
// all), Up's values as they are or, fp16, as two (eight and three bits).  Products
// of bf16 numbers are exact in fp32, so the term is as if made there, whatever a
// row's ranks' sizes beside each other, for three or five MFMAs; fp32 ones would
// take as long as sixteen.  (Of fp16 the smallest parts' product, below 2^-24 of the
// whole, is left out.)  What is not finite stays so.
struct RankRow {
    u32x4 part[3];
    __device__ __forceinline__ void split(const f32x4 (&v)[2])
    {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            uint32_t w[2][3];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float x = v[p >> 1][2 * (p & 1) + e];
                const float r = fabsf(x) < __builtin_inff() ? x - upper(x) : 0.f;
                w[e][0] = __float_as_uint(x);
                w[e][1] = __float_as_uint(r);
                w[e][2] = __float_as_uint(r - upper(r));
            }
#pragma unroll
            for (int q = 0; q < 3; ++q) part[q][p] = upper_halves(w[0][q], w[1][q]);
        }
    }
    __device__ __forceinline__ void load(const float *u, bool have)
    {
        f32x4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        if (have) {
            v[0] = *reinterpret_cast<const f32x4 *>(u);
            v[1] = *reinterpret_cast<const f32x4 *>(u + 4);
        }
        split(v);
    }
    // the bf16 number that x's upper half is
    static __device__ __forceinline__ float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t upper_halves(uint32_t lo, uint32_t hi)
    {
        return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
    }
};

// Eight ranks of a row of Up for the same product.
template <class T>
struct UpRow {
    u32x4 part[std::is_same<T, F16>::value ? 2 : 1];
    __device__ __forceinline__ void split(u32x4 v)
    {
        if constexpr (std::is_same<T, F16>::value) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float x = T::load((uint16_t)v[p]), y = T::load((uint16_t)(v[p] >> 16));
                part[0][p] = RankRow::upper_halves(__float_as_uint(x), __float_as_uint(y));
                part[1][p] = RankRow::upper_halves(__float_as_uint(x - RankRow::upper(x)), __float_as_uint(y - RankRow::upper(y)));
            }
        } else {
            part[0] = v;
        }
    }
};

// c += b u^T over sixteen ranks of 32 rows each.
template <class T>
__device__ __forceinline__ f32x16 multiply_ranks(const UpRow<T> &b, const RankRow &u, f32x16 c)
{
#pragma unroll
    for (int q = 0; q < 3; ++q) c = Bf16::mfma(b.part[0], u.part[q], c);
    if constexpr (std::is_same<T, F16>::value) {
#pragma unroll
        for (int q = 0; q < 2; ++q) c = Bf16::mfma(b.part[1], u.part[q], c);
    }
    return c;
}

// Eight ranks of B from rank k on, 16-bit values, for NJ 32-column blocks (`up`:
// the lane's row of each, or null past the matrix); zero at and past `rank`.
template <class T, int NJ>
__device__ __forceinline__ void load_columns(const typename T::Store *const (&up)[NJ], int k, int rank, UpRow<T> (&b)[NJ])
{
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (up[j] && k + 8 <= rank) {
            __builtin_memcpy(&v, up[j] + k, 16);
        } else if (up[j] && k < rank) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < rank) v[e >> 1] |= (uint32_t)up[j][k + e] << (16 * (e & 1));
        }
        b[j].split(v);
    }
}

// acc += u B_a^T for the wave's blocks (block i's first row m0 + 32 i, rows
// from m on do not exist) and the rows that have an adapter.  Returns the rows
// without one (bit i: the lane's row of block i).  A row sees its own adapter's
// values only, so that infinities in another's do not reach it:
//   all the wave's rows with one adapter (prompts): B_a is loaded once for
//     them and the products are added to acc directly;
//   a 32-row block with at most kAdapterPasses adapters: each in turn, its rows
//     keeping their own products;
//   more (decode batches): every lane gathers its own row's adapter, eight ranks of a
//     column at a time.
constexpr int kAdapterPasses = 3;

template <class T, int MI, int NJ>
__device__ __forceinline__ uint32_t add_adapters(f32x16 (&acc)[MI][NJ], const GroupedArgs &a, int m0, int n0, int m)
{
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const AdapterTerm &t = a.term;
    const typename T::Store *const up = reinterpret_cast<const typename T::Store *>(t.up);
    int mine[MI];
    uint32_t without = 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = m0 + 32 * i + (lane & 31);
        mine[i] = -2;  // past the rows
        if (row < m) {
            mine[i] = t.adapter[row];
            if (mine[i] < 0 || mine[i] >= t.adapters) {
                mine[i] = -1;
                without |= 1u << i;
            }
        }
    }
    const int one = __builtin_amdgcn_readfirstlane(mine[0]);
    bool same = true;
#pragma unroll
    for (int i = 0; i < MI; ++i) same = same && (mine[i] == one || mine[i] == -2);
    if (__ballot(!same) == 0) {
        if (one < 0) return without;
        if constexpr (T::kBytes == 2) {
            const typename T::Store *rows[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int col = n0 + 32 * j + (lane & 31);
                rows[j] = col < a.outputs ? up + ((long long)one * a.outputs + col) * t.rank : nullptr;
            }
            const typename T::Store *const(&cols)[NJ] = rows;
            for (int c = 0; c < t.rank; c += 16) {
                const int k = c + 8 * h;
                UpRow<T> b[NJ];
                load_columns<T, NJ>(cols, k, t.rank, b);
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    RankRow u;
                    u.load(t.u + (long long)(m0 + 32 * i + (lane & 31)) * t.ldu + k, mine[i] >= 0 && k < t.ldu);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = multiply_ranks<T>(b[j], u, acc[i][j]);
                }
            }
            return without;
        }
    }
    const bool aligned = t.rank % 4 == 0 && (reinterpret_cast<uintptr_t>(t.up) & (4 * T::kBytes - 1)) == 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int row = m0 + 32 * i + (lane & 31);
        const uint64_t rows = __ballot(mine[i] >= 0);
        uint64_t todo = rows;
        int passes = 0;
        while (todo && passes <= kAdapterPasses) {
            todo &= ~__ballot(mine[i] == __builtin_amdgcn_readlane(mine[i], __builtin_ctzll(todo)));
            ++passes;
        }
        if (passes > kAdapterPasses) {
            if (mine[i] >= 0) {
                const float *u = t.u + (long long)row * t.ldu;
                const typename T::Store *mat = up + (long long)mine[i] * a.outputs * t.rank;
                for (int c = 0; c < t.rank; c += 8) {
                    const f32x4 u0 = *reinterpret_cast<const f32x4 *>(u + c), u1 = *reinterpret_cast<const f32x4 *>(u + c + 4);
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int col = n0 + 32 * j + 8 * (r >> 2) + 4 * h + (r & 3);
                            if (col < a.outputs) {
                                float b[8];
                                load_ranks<T>(mat + (long long)col * t.rank, c, t.rank, b);
                                float d = u0[0] * b[0];
#pragma unroll
                                for (int e = 1; e < 4; ++e) d = fmaf(u0[e], b[e], d);
#pragma unroll
                                for (int e = 0; e < 4; ++e) d = fmaf(u1[e], b[4 + e], d);
                                acc[i][j][r] += d;
                            }
                        }
                }
            }
            continue;
        }
        todo = rows;
        while (todo) {
            const int cur = __builtin_amdgcn_readlane(mine[i], __builtin_ctzll(todo));
            const bool here = mine[i] == cur;
            todo &= ~__ballot(here);
            f32x16 d[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) d[j][r] = 0.f;
            if constexpr (T::kBytes == 2) {
                const typename T::Store *crows[NJ];
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int col = n0 + 32 * j + (lane & 31);
                    crows[j] = col < a.outputs ? up + ((long long)cur * a.outputs + col) * t.rank : nullptr;
                }
                const typename T::Store *const(&cols)[NJ] = crows;
                for (int c = 0; c < t.rank; c += 16) {
                    const int k = c + 8 * h;
                    UpRow<T> b[NJ];
                    load_columns<T, NJ>(cols, k, t.rank, b);
                    RankRow u;
                    u.load(t.u + (long long)row * t.ldu + k, here && k < t.ldu);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) d[j] = multiply_ranks<T>(b[j], u, d[j]);
                }
            } else {
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
    const bool aligned = (reinterpret_cast<uintptr_t>(bias) & (4 * T::kBytes - 1)) == 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = n0 + 32 * j + 8 * q + 4 * h;
            float v[4];
            load4<T>(b + col, v, n - col, aligned);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += v[e];
        }
}

}  // namespace

}  // namespace gtmoe
