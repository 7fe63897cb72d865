// Products of few rows that stream a matrix from memory into MFMA operands
// without LDS, and what an epilogue does with a product's values.
#pragma once

#include "grouped_tile.h"
#include "rows.h"

namespace gtmoe {

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

template <class T>
__device__ __forceinline__ u32x4 load_whole_unit(const typename T::Store *p)
{
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// c += a b^T over 64 bytes of reduction, 16 x 16: lane l holds 16 bytes
// (quarter l / 16) of row l % 16 of both operands, and of the result column
// l % 16 (b's row) and rows 4 (l / 16) .. + 3 (a's).
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

// acc[p][q] += a_p b_q^T over the reduction [0, length) that falls to this
// wave (every WAVES-th 64 bytes), a_p and b_q the lane's rows of NP and NQ
// 16-row operands.  Loads go straight to MFMA operands, those of `ahead` steps from
// one loop, in which the compiler keeps up to seven loads in flight (one and two operands of
// 16 bits: 18 loads, the first wait behind seven).  Steps that are fewer, and the last
// ones, go one by one, each behind its loads.
template <class T, int WAVES, int NP, int NQ>
__device__ __forceinline__ void multiply_rows(const typename T::Store *const (&pa)[NP], const typename T::Store *const (&pb)[NQ],
                                              int length, int wave, f32x4 (&acc)[NP][NQ])
{
    constexpr int unit = 16 / T::kBytes, step = 4 * unit;
    constexpr int ahead = NP + NQ <= 2 ? 8 : NP + NQ <= 3 ? 6 : 4;
    const int q0 = ((threadIdx.x & 63) >> 4) * unit;
    const int whole = length / step;  // steps that lie wholly inside
    int k = wave;
    for (; k + (ahead - 1) * WAVES < whole; k += ahead * WAVES) {
        u32x4 a[ahead][NP], b[ahead][NQ];
#pragma unroll
        for (int i = 0; i < ahead; ++i) {
            const int at = (k + i * WAVES) * step + q0;
#pragma unroll
            for (int p = 0; p < NP; ++p) a[i][p] = load_whole_unit<T>(pa[p] + at);
#pragma unroll
            for (int q = 0; q < NQ; ++q) b[i][q] = load_whole_unit<T>(pb[q] + at);
        }
#pragma unroll
        for (int i = 0; i < ahead; ++i)
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int q = 0; q < NQ; ++q) acc[p][q] = mfma16<T>(a[i][p], b[i][q], acc[p][q]);
    }
    for (; k * step < length; k += WAVES) {
        const int at = k * step + q0;
        u32x4 a[NP], b[NQ];
#pragma unroll
        for (int p = 0; p < NP; ++p) a[p] = load_unit<T>(pa[p], at, length);
#pragma unroll
        for (int q = 0; q < NQ; ++q) b[q] = load_unit<T>(pb[q], at, length);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int q = 0; q < NQ; ++q) acc[p][q] = mfma16<T>(a[p], b[q], acc[p][q]);
    }
}

template <class T>
constexpr int values_of()
{
    return T::kBytes == 4 ? kValuesF32 : std::is_same<T, Bf16>::value ? kValuesBf16 : kValuesF16;
}

// y = act(z + b) factor + residual of four columns of a row, z kept first where it
// is asked for; `left` of the columns exist, the first a multiple of four.
template <int VALUES>
__device__ __forceinline__ float epilogue_activated(float z, int activation)
{
    switch (activation) {
    case kActivationRelu: return activated<VALUES, kActivationRelu>(z);
    case kActivationSilu: return activated<VALUES, kActivationSilu>(z);
    case kActivationGelu: return activated<VALUES, kActivationGelu>(z);
    case kActivationGeluTanh: return activated<VALUES, kActivationGeluTanh>(z);
    default: return z;
    }
}
template <class T>
__device__ __forceinline__ bool whole_fours(const void *p, long long stride)
{
    return stride % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & (4 * T::kBytes - 1)) == 0;
}
template <class T>
__device__ __forceinline__ void store_fused(const GroupedArgs &a, int g, long long row, int col, float (&v)[4], int left)
{
    typedef typename T::Store Store;
    const Epilogue &e = a.epilogue;
    if (e.bias) {
        float b[4];
        load4<T>(reinterpret_cast<const Store *>(e.bias) + g * e.ldbias + col, b, left, whole_fours<T>(e.bias, e.ldbias));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += b[i];
    }
    if (e.products)
        store4<T>(reinterpret_cast<Store *>(e.products) + row * e.ldproducts + col, v, left, whole_fours<T>(e.products, e.ldproducts));
    if (e.activation != kActivationNone) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = epilogue_activated<values_of<T>()>(v[i], e.activation);
    }
    if (e.factor) {
        float f[4];
        load4<T>(reinterpret_cast<const Store *>(e.factor) + row * e.ldfactor + col, f, left, whole_fours<T>(e.factor, e.ldfactor));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= f[i];
    }
    if (e.residual) {
        float r[4];
        load4<T>(reinterpret_cast<const Store *>(e.residual) + row * e.ldresidual + col, r, left,
                 whole_fours<T>(e.residual, e.ldresidual));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += r[i];
    }
    store4<T>(reinterpret_cast<Store *>(a.out) + row * a.ldo + col, v, left, whole_fours<T>(a.out, a.ldo));
}

// The same for the 32 x 32 blocks that a wave holds after MFMAs (lane l: row l % 32 and,
// in register r, column 8 (r / 4) + 4 (l / 32) + r % 4 of a block): block (i, j) is rows
// r0 + STEP i on of the tile's m from row0 on, columns c0 + 32 j on of its n from col0 on
// (m and n at least 1; a wave may have none of them).  The rows
// that are read and written cross between that layout and 16 bytes per lane, 128 (or 64)
// consecutive bytes of a row at a time, in 4 KiB of the wave's LDS, 16-byte unit u of
// row r in slot u ^ (r / 2) % 8 (r % 4 of four); what is read next is asked for before
// what is there is used.
// What an epilogue adds (MI355X, us): 16384 rows of 16 equal groups 1024 -> 2048 bf16 74 as the plain
// product, 77 with biases, 80 with SiLU, 88 with a factor, 100 with z kept: the 134 MB of
// factors and z take 27 at a copy's rate, and nothing else runs on a CU meanwhile.  1024
// rows of 1024 -> 2048 with bias, SiLU and factor 18.6 against 16.1 (29.4 where every value's
// four columns were loaded and stored by themselves).
// ACT: the activation, or -1 for a.epilogue's.  WHOLE: rows and row starts are whole 16
// bytes, and registers are scarce: addresses are held inside the rows instead of
// branched around, and made again for each use (kept, they were spilled).
template <class T, int MI, int NJ, int STEP, int ACT, bool WHOLE>
__device__ __forceinline__ void finish_blocks(f32x16 (&acc)[MI][NJ], const GroupedArgs &a, int g, long long row0, int r0, int m,
                                              long long col0, int c0, int n, char *stage, int el)
{
    typedef typename T::Store Store;
    constexpr int EACH = T::kBytes == 2 && NJ % 2 == 0 ? 2 : 1;  // blocks of columns at a time
    constexpr int WIDTH = 32 * EACH * T::kBytes, UNITS = WIDTH / 16, ROWS = 64 / UNITS, PASSES = 32 / ROWS, VALUES = 16 / T::kBytes;
    const Epilogue &e = a.epilogue;
    const int er = el & 31, h = el >> 5, ur = el / UNITS, unit = el % UNITS;
    auto swap = [](int r) { return (r >> 1) & (UNITS - 1); };
    // four consecutive values of the lane's row, and 16 bytes of row ROWS p + ur
    auto four = [&](int j, int q) {
        const int at = T::kBytes == 2 ? ((4 * j + q) ^ swap(er)) * 16 + h * 8 : ((2 * q + h) ^ swap(er)) * 16;
        return stage + er * WIDTH + at;
    };
    auto piece = [&](int p) { return reinterpret_cast<u32x4 *>(stage + (ROWS * p + ur) * WIDTH + (unit ^ swap(ROWS * p + ur)) * 16); };
    auto again = [&]() {
        int own = ur;
        if constexpr (WHOLE) asm volatile("" : "+v"(own));
        return own;
    };
    auto ask = [&](u32x4 (&v)[PASSES], const void *from, long long ld, int i, int j0) {
        const int own = again(), col = c0 + 32 * j0 + VALUES * unit, left = n - col;
        const Store *base = reinterpret_cast<const Store *>(from) + row0 * ld + col0;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int row = r0 + STEP * i + ROWS * p + own;
            if constexpr (WHOLE) {
                const uint32_t at = ((uint32_t)min(row, m - 1) * (uint32_t)ld + (left > 0 ? col : 0)) * T::kBytes;
                v[p] = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const char *>(base) + at);
            } else {
                v[p] = row < m ? load_unit<T>(base + row * ld + col, 0, left) : u32x4{0u, 0u, 0u, 0u};
            }
        }
    };
    auto put = [&](const u32x4 (&v)[PASSES]) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) *piece(p) = v[p];
        __builtin_amdgcn_wave_barrier();
    };
    // the blocks' values, rounded, to rows of a matrix
    auto take = [&](void *to, long long ld, int i, int j0) {
#pragma unroll
        for (int j = 0; j < EACH; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x16 &v = acc[i][j0 + j];
                if constexpr (T::kBytes == 2)
                    *reinterpret_cast<uint2 *>(four(j, q)) = make_uint2(T::pack(v[4 * q], v[4 * q + 1]), T::pack(v[4 * q + 2], v[4 * q + 3]));
                else
                    *reinterpret_cast<float4 *>(four(j, q)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            }
        __builtin_amdgcn_wave_barrier();
        const int own = again(), col = c0 + 32 * j0 + VALUES * unit, left = n - col;
        Store *base = reinterpret_cast<Store *>(to) + row0 * ld + col0;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int row = r0 + STEP * i + ROWS * p + own;
            const u32x4 v = *piece(p);
            if (row < m && left > 0) {
                if constexpr (WHOLE) {
                    const uint32_t at = ((uint32_t)row * (uint32_t)ld + col) * T::kBytes;
                    *reinterpret_cast<u32x4 *>(reinterpret_cast<char *>(base) + at) = v;
                } else if (left >= VALUES) {
                    __builtin_memcpy(base + row * ld + col, &v, 16);
                } else {
#pragma unroll
                    for (int x = 0; x < VALUES; ++x)
                        if (x < left) {
                            if constexpr (T::kBytes == 2) base[row * ld + col + x] = (uint16_t)(v[x >> 1] >> (16 * (x & 1)));
                            else base[row * ld + col + x] = __uint_as_float(v[x]);
                        }
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    };
    auto each = [&](int i, int j0, auto &&f) {
#pragma unroll
        for (int j = 0; j < EACH; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float w[4];
                if constexpr (T::kBytes == 2) {
                    const uint2 t = *reinterpret_cast<const uint2 *>(four(j, q));
#pragma unroll
                    for (int c = 0; c < 4; ++c) w[c] = T::load((uint16_t)((c < 2 ? t.x : t.y) >> (16 * (c & 1))));
                } else {
                    __builtin_memcpy(w, four(j, q), 16);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][j0 + j][4 * q + c] = f(acc[i][j0 + j][4 * q + c], w[c]);
            }
        __builtin_amdgcn_wave_barrier();
    };
    auto act = [&](int i, int j0, auto kind) {
#pragma unroll
        for (int j = j0; j < j0 + EACH; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = activated<values_of<T>(), decltype(kind)::value>(acc[i][j][r]);
    };
    u32x4 rows[PASSES];  // what was asked for last: a block's factors, then its residual
    auto ask_first = [&](int i, int j0) {
        if (e.factor) ask(rows, e.factor, e.ldfactor, i, j0);
        else if (e.residual) ask(rows, e.residual, e.ldresidual, i, j0);
    };
    ask_first(0, 0);
    if (e.bias) add_bias<T>(acc, reinterpret_cast<const Store *>(e.bias) + g * e.ldbias, (int)col0 + c0, a.outputs);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j0 = 0; j0 < NJ; j0 += EACH) {
            const bool last = i + 1 == MI && j0 + EACH == NJ;
            const int ni = j0 + EACH == NJ ? i + 1 : i, nj = j0 + EACH == NJ ? 0 : j0 + EACH;
            if (e.products) take(e.products, e.ldproducts, i, j0);
            if constexpr (ACT > 0) {
                act(i, j0, std::integral_constant<int, ACT>());
            } else if constexpr (ACT < 0) {
                switch (e.activation) {
                case kActivationRelu: act(i, j0, std::integral_constant<int, kActivationRelu>()); break;
                case kActivationSilu: act(i, j0, std::integral_constant<int, kActivationSilu>()); break;
                case kActivationGelu: act(i, j0, std::integral_constant<int, kActivationGelu>()); break;
                case kActivationGeluTanh: act(i, j0, std::integral_constant<int, kActivationGeluTanh>()); break;
                default: break;
                }
            }
            if (e.factor) {
                put(rows);
                if (e.residual) ask(rows, e.residual, e.ldresidual, i, j0);
                else if (!last) ask(rows, e.factor, e.ldfactor, ni, nj);
                each(i, j0, [](float v, float w) { return v * w; });
            }
            if (e.residual) {
                put(rows);
                if (!last) ask_first(ni, nj);
                each(i, j0, [](float v, float w) { return v + w; });
            }
            take(a.out, a.ldo, i, j0);
        }
}

}  // namespace

}  // namespace gtmoe
