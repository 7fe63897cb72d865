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
// 16-row operands.  Loads go straight to MFMA operands; `ahead` steps of them
// are requested together.
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

// y = act(z + b) factor + residual of four columns of a row, z kept first where it
// is asked for; `left` of the columns exist, the first a multiple of four.
__device__ __forceinline__ float epilogue_activated(float z, int activation)
{
    switch (activation) {
    case kActivationRelu: return activated<kActivationRelu>(z);
    case kActivationSilu: return activated<kActivationSilu>(z);
    case kActivationGelu: return activated<kActivationGelu>(z);
    case kActivationGeluTanh: return activated<kActivationGeluTanh>(z);
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
        for (int i = 0; i < 4; ++i) v[i] = epilogue_activated(v[i], e.activation);
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

}  // namespace

}  // namespace gtmoe
