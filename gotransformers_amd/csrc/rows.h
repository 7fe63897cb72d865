// Parts the operators over plain rows share: the values' types, eight values of
// a row at a time, sums and maxima over neighbouring lanes, 8-bit codes with
// scales, and activations.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "grouped.h"

namespace gtmoe {

namespace {

typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));

// Eight consecutive values of a row as they lie in memory.
template <int VALUES>
struct Eight;
template <>
struct Eight<kValuesF32> {
    typedef float Store;
    float raw[8];
    __device__ __forceinline__ float get(int e) const { return raw[e]; }
    __device__ __forceinline__ void set(const float (&v)[8])
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[e] = v[e];
    }
};
template <>
struct Eight<kValuesBf16> {
    typedef uint16_t Store;
    uint32_t raw[4];
    __device__ __forceinline__ float get(int e) const
    {
        return __uint_as_float(e & 1 ? raw[e >> 1] & 0xffff0000u : raw[e >> 1] << 16);
    }
    __device__ __forceinline__ void set(const float (&v)[8])
    {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){v[2 * e], v[2 * e + 1]}, b2));
    }
};
template <>
struct Eight<kValuesF16> {
    typedef uint16_t Store;
    uint32_t raw[4];
    __device__ __forceinline__ float get(int e) const
    {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(raw[e >> 1] >> (16 * (e & 1))));
    }
    __device__ __forceinline__ void set(const float (&v)[8])
    {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){v[2 * e], v[2 * e + 1]}, h2));
    }
};

// The columns of a thread's eight values, `column` being eight times its place in the row:
// 16-bit values are eight consecutive ones, 16 bytes.  Of fp32, 16 threads share 128 columns,
// four consecutive ones each in the first 64 and four in the second, so that one
// instruction of theirs moves 256 consecutive bytes (eight consecutive ones, two
// instructions of 16 bytes every 32: SiLU's gradient of 4096 x 2048 from codes 42.6 us against
// 35.9, the norm's forward 34.5 against 28.9).
template <int VALUES>
__device__ __forceinline__ int column_of(int column, int j)
{
    if constexpr (VALUES == kValuesF32) return (column & ~127) + ((column & 127) >> 1) + (j & 3) + ((j & 4) << 4);
    return column + j;
}
// Whether some of them exist.
template <int VALUES>
__device__ __forceinline__ bool any_column(int column, int columns) { return column_of<VALUES>(column, 0) < columns; }

// `many` values from p on, any alignment; n of them exist, the others are zero.
template <int MANY, class Store>
__device__ __forceinline__ void load_some(void *v, const Store *p, int n)
{
    if (n >= MANY) {
        __builtin_memcpy(v, p, MANY * sizeof(Store));
    } else {
        Store w[MANY];
#pragma unroll
        for (int e = 0; e < MANY; ++e) w[e] = e < n ? p[e] : (Store)0;
        __builtin_memcpy(v, w, sizeof w);
    }
}
template <int MANY, class Store>
__device__ __forceinline__ void store_some(const void *v, Store *p, int n)
{
    if (n >= MANY) {
        __builtin_memcpy(p, v, MANY * sizeof(Store));
    } else {
        Store w[MANY];
        __builtin_memcpy(w, v, sizeof w);
#pragma unroll
        for (int e = 0; e < MANY; ++e)
            if (e < n) p[e] = w[e];
    }
}

// A thread's eight values of the row that begins at base[row].
template <int VALUES>
__device__ __forceinline__ void load_eight(Eight<VALUES> &v, const void *base, long long row, int column, int columns)
{
    typedef typename Eight<VALUES>::Store Store;
    const int c = column_of<VALUES>(column, 0), n = columns - c;
    const Store *p = reinterpret_cast<const Store *>(base) + row + c;
    if constexpr (VALUES == kValuesF32) {
        load_some<4>(v.raw, p, n);
        load_some<4>(v.raw + 4, p + 64, n - 64);
    } else {
        load_some<8>(v.raw, p, n);
    }
}
// The same where all of them exist: no branch between loads.
template <int VALUES>
__device__ __forceinline__ void load_whole_eight(Eight<VALUES> &v, const void *base, long long row, int column)
{
    typedef typename Eight<VALUES>::Store Store;
    const Store *p = reinterpret_cast<const Store *>(base) + row + column_of<VALUES>(column, 0);
    if constexpr (VALUES == kValuesF32) {
        __builtin_memcpy(v.raw, p, 16);
        __builtin_memcpy(v.raw + 4, p + 64, 16);
    } else {
        __builtin_memcpy(v.raw, p, 16);
    }
}
template <int VALUES>
__device__ __forceinline__ void store_eight(const Eight<VALUES> &v, void *base, long long row, int column, int columns)
{
    typedef typename Eight<VALUES>::Store Store;
    const int c = column_of<VALUES>(column, 0), n = columns - c;
    Store *p = reinterpret_cast<Store *>(base) + row + c;
    if constexpr (VALUES == kValuesF32) {
        store_some<4>(v.raw, p, n);
        store_some<4>(v.raw + 4, p + 64, n - 64);
    } else {
        store_some<8>(v.raw, p, n);
    }
}

// ---------------------------------------------------------------------------
// Neighbouring lanes, by DPP: after the exchanges with the lane beside, two and
// four (half mirrored) and eight (mirrored) away the 16 lanes of a row agree.
// ---------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kDppPairs = 0xB1, kDppFours = 0x4E, kDppEights = 0x141, kDppSixteens = 0x140;

// The largest of the `lanes` (a power of two up to 16) lanes' values.
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes)
{
    if (lanes > 1) v = max(v, moved<kDppPairs>(v));
    if (lanes > 2) v = max(v, moved<kDppFours>(v));
    if (lanes > 4) v = max(v, moved<kDppEights>(v));
    if (lanes > 8) v = max(v, moved<kDppSixteens>(v));
    return v;
}
__device__ __forceinline__ float sixteen_sum(float v)
{
    v += __uint_as_float(moved<kDppPairs>(__float_as_uint(v)));
    v += __uint_as_float(moved<kDppFours>(__float_as_uint(v)));
    v += __uint_as_float(moved<kDppEights>(__float_as_uint(v)));
    v += __uint_as_float(moved<kDppSixteens>(__float_as_uint(v)));
    return v;
}
__device__ __forceinline__ float lane_value(float v, int lane)
{
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}
__device__ __forceinline__ float wave_sum(float v)
{
    v = sixteen_sum(v);
    return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    v = lanes_max(v, 16);
    const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
    const uint32_t b = max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
    return max(a, b);
}

// ---------------------------------------------------------------------------
// 8-bit codes: the values of a block share scale = max|v| / 127 (int8) or / 448
// (e4m3), rounded to fp32.
//   int8  v / scale to the nearest whole number, halves away from zero, at most 127
//         in size (lowprecision.encodeInt8, lowprecision.go:66-78, for the same scale)
//   e4m3  v / scale rounded to fp32, then to the nearest e4m3, halves to even, at most
//         448 in size
// A block of zeros has scale 0 and codes 0; one with a value that is not finite
// has scale NaN and codes 0, so that all of it reads back as NaN.
// ---------------------------------------------------------------------------
enum Codes { kCodesNone = 0, kCodesInt8 = 1, kCodesE4m3 = 2 };

// max |v| as bits: the order of finite, infinite and NaN values in one comparison.
__device__ __forceinline__ uint32_t size_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Scale {
    float value;    // as it is stored
    float inverse;  // 1 / value, rounded; 0 for a block of zeros
    bool plain;     // value is 0 or well inside the normal numbers, and so is its inverse
    __device__ __forceinline__ Scale(uint32_t most_bits, int codes)
    {
        const float most = __uint_as_float(most_bits);
        value = codes == kCodesInt8 ? most / 127.f : most / 448.f;
        plain = value == 0.f || (value >= 0x1p-60f && most_bits < 0x7f800000u);
        if (most_bits >= 0x7f800000u) value = __uint_as_float(0x7fc00000u);
        inverse = value >= 0x1p-60f ? 1.f / value : 0.f;
    }
};

// The size of an int8 code.  inverse is made 2^-22 too small, which is more than all the
// roundings up to the sum with a half are, so that the whole number below it is the code or
// one less: which, the remainder a - q scale tells, exact in an fma.
__device__ __forceinline__ float int8_size(float a, float scale, float inverse, float half)
{
    const float q = floorf(fmaf(a, inverse, 0.5f));
    return fminf(q + (fmaf(-q, scale, a) >= half ? 1.f : 0.f), 127.f);
}
// The quotient v / scale, rounded: by the inverse, put right by its remainder.
__device__ __forceinline__ float e4m3_quotient(float v, float scale, float inverse)
{
    const float q = v * inverse;
    return fminf(fmaxf(fmaf(fmaf(-q, scale, v), inverse, q), -448.f), 448.f);
}

__device__ __forceinline__ uint32_t int8_bytes(float a, float b, float c, float d)
{
    const uint32_t lo = __builtin_amdgcn_perm((uint32_t)(int)b, (uint32_t)(int)a, 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm((uint32_t)(int)d, (uint32_t)(int)c, 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
__device__ __forceinline__ uint32_t e4m3_bytes(float a, float b, float c, float d)
{
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
}

// What coding a block's values takes.  odd, the same for a wave: a scale next to the
// subnormal numbers, where everything is taken times a power of two, or one that is not
// finite, whose codes are 0.
struct Coder {
    float scale, inverse, below, half, times = 1.f;
    bool odd, finite;
    __device__ __forceinline__ Coder(const Scale &s) : scale(s.value), inverse(s.inverse)
    {
        odd = __ballot(!s.plain) != 0;
        finite = true;
        if (odd) {
            const bool tiny = scale < 0x1p-60f && scale > 0.f;
            finite = scale == scale;
            times = tiny ? 0x1p90f : 1.f;
            scale = finite ? scale * times : 0.f;
            inverse = tiny ? 1.f / scale : inverse;
        }
        half = inverse > 0.f ? 0.5f * scale : __builtin_inff();
        below = inverse - inverse * 0x1p-22f;
    }
    template <int CODES>
    __device__ __forceinline__ uint32_t four_of(const float *v) const
    {
        float c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = v[e];
            if (odd) x = finite ? x * times : 0.f;
            c[e] = CODES == kCodesInt8 ? copysignf(int8_size(fabsf(x), scale, below, half), x) : e4m3_quotient(x, scale, inverse);
        }
        return CODES == kCodesInt8 ? int8_bytes(c[0], c[1], c[2], c[3]) : e4m3_bytes(c[0], c[1], c[2], c[3]);
    }
    __device__ __forceinline__ uint32_t four(const float *v, int codes) const
    {
        return codes == kCodesInt8 ? four_of<kCodesInt8>(v) : four_of<kCodesE4m3>(v);
    }
};
__device__ __forceinline__ void decode_four(uint32_t w, float scale, int codes, float *v)
{
    if (codes == kCodesInt8) {
        // a byte plus 128 is an unsigned number, which the hardware converts where it is
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ((float)((w ^ 0x80808080u) >> (8 * e) & 0xffu) - 128.f) * scale;
    } else {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        v[0] = lo[0] * scale;
        v[1] = lo[1] * scale;
        v[2] = hi[0] * scale;
        v[3] = hi[1] * scale;
    }
}

__device__ __forceinline__ uint32_t largest_of_four(const float *v)
{
    return max(max(size_bits(v[0]), size_bits(v[1])), max(size_bits(v[2]), size_bits(v[3])));
}

// Codes of a thread's eight values, which are zero past the last column, and, by the first
// thread of a block of columns, its scale.  Every thread of the block calls it.  most: the largest
// of the row where a row has one scale (scale_columns 0).
template <int VALUES>
__device__ __forceinline__ void keep_eight(const float (&v)[8], long long row, int column, int columns, const PackedRows &k,
                                           uint32_t most = 0)
{
    const uint32_t lo = largest_of_four(v), hi = largest_of_four(v + 4);
    const int bits = k.scale_columns ? __builtin_ctz(k.scale_columns) : 31;
    const int c = column_of<VALUES>(column, 0), n = columns - c;
    uint8_t *codes = k.codes + row * k.ldcodes + c;
    float *scales = k.scales + row * k.ldscales;
    auto first = [&](int at) { return (at & (int)((1u << bits) - 1)) == 0; };
    if constexpr (VALUES == kValuesF32) {
        // two blocks, or 128 columns or the row as one
        const bool one = k.scale_columns == 0 || k.scale_columns == 128;
        uint32_t m0 = one ? max(lo, hi) : lo, m1 = one ? m0 : hi;
        if (k.scale_columns == 0) {
            m0 = m1 = most;
        } else {
            m0 = lanes_max(m0, one ? 16 : k.scale_columns / 4);
            m1 = one ? m0 : lanes_max(m1, k.scale_columns / 4);
        }
        const Scale s0(m0, k.code_type);
        Scale s1 = s0;
        Coder c0(s0), c1 = c0;
        if (!one) {
            s1 = Scale(m1, k.code_type);
            c1 = Coder(s1);
        }
        const uint32_t w0 = c0.four(v, k.code_type), w1 = c1.four(v + 4, k.code_type);
        if (n > 0) {
            store_some<4>(&w0, codes, n);
            if (first(c)) scales[c >> bits] = s0.value;
        }
        if (n > 64) {
            store_some<4>(&w1, codes + 64, n - 64);
            if (!one && first(c + 64)) scales[(c + 64) >> bits] = s1.value;
        }
    } else {
        const Scale s(k.scale_columns ? lanes_max(max(lo, hi), k.scale_columns / 8) : most, k.code_type);
        const Coder coder(s);
        const uint32_t w[2] = {coder.four(v, k.code_type), coder.four(v + 4, k.code_type)};
        if (n <= 0) return;
        store_some<8>(w, codes, n);
        if (first(c)) scales[c >> bits] = s.value;
    }
}

// The values that a thread's eight codes stand for; one of them exists at least.
template <int VALUES>
__device__ __forceinline__ void kept_eight(float (&v)[8], long long row, int column, int columns, const PackedRows &k)
{
    const int bits = k.scale_columns ? __builtin_ctz(k.scale_columns) : 31;
    const int c = column_of<VALUES>(column, 0), n = columns - c;
    const uint8_t *codes = k.codes + row * k.ldcodes + c;
    const float *scales = k.scales + row * k.ldscales;
    uint32_t w[2];
    if constexpr (VALUES == kValuesF32) {
        load_some<4>(w, codes, n);
        load_some<4>(w + 1, codes + 64, n - 64);
    } else {
        load_some<8>(w, codes, n);
    }
    const float s0 = scales[c >> bits];
    decode_four(w[0], s0, k.code_type, v);
    decode_four(w[1], VALUES == kValuesF32 && n > 64 ? scales[(c + 64) >> bits] : s0, k.code_type, v + 4);
}

// ---------------------------------------------------------------------------
// Activations and their derivatives in fp32.
// ---------------------------------------------------------------------------
enum Activation { kActivationNone = 0, kActivationRelu = 1, kActivationSilu = 2, kActivationGelu = 3, kActivationGeluTanh = 4 };

__device__ __forceinline__ float inverse_of(float d)  // d at least 1, far from the largest numbers
{
    const float x = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, x, 1.f), x, x);
}

// Activations z times a factor.  The hardware's functions know no subnormal numbers, and
// z e^z may still be one, or a normal number of bf16 and fp32, where e^z is none (z = -88): there
// e^z is taken times a power of two, and that put right behind the product with z.

// 1 / (1 + e^-z) = value * times for 16-bit rows: a power of two and a reciprocal of the
// hardware's, good to a unit each, of an argument good to |z| 2^-24.  fp16 has no numbers as small.
template <int VALUES>
struct Logistic {
    float value, times;
    __device__ __forceinline__ Logistic(float z)
    {
        constexpr float by = (float)-1.44269504088896340736;
        const bool far = VALUES == kValuesBf16 && z < 0.f;
        times = far ? 0x1p-32f : 1.f;
        value = __builtin_amdgcn_rcpf(times + __builtin_amdgcn_exp2f(VALUES == kValuesBf16 ? fmaf(by, z, far ? -32.f : 0.f) : by * z));
    }
};

// 2^(whole + fraction) = e * times for fp32 rows: an exponent t rounded to fp32 would cost |t|
// units, the fraction holds what is left of it beside its whole part.
struct Power {
    float e, times;
    __device__ __forceinline__ Power(float whole, float fraction)
    {
        const bool far = whole < -64.f;
        times = far ? 0x1p-64f : 1.f;
        e = ldexpf(__builtin_amdgcn_exp2f(fraction), (int)whole + (far ? 64 : 0));
    }
};
constexpr double kLog2e = 1.44269504088896340736;
// what fp32 leaves of a constant
constexpr float rest_of(double c) { return (float)(c - (double)(float)c); }
// s = value * times = 1 / (1 + e^-y) and rest = 1 - s, of y's sign and p = e^-|y|.
struct WideLogistic {
    float value, times, rest;
    __device__ __forceinline__ WideLogistic(bool below, const Power &p)
    {
        const float e = p.e * p.times, r = inverse_of(1.f + e);
        value = below ? p.e * r : r;
        times = below ? p.times : 1.f;
        rest = below ? r : e * r;
    }
};

__device__ constexpr float kTail[10] = {0.25388533f, 0.25388303f,  0.22827554f, 0.17520681f,  0.12021917f,
                                        -0.023251647f, 0.14413364f, -0.30252245f, 0.1918485f, -0.041677944f};

// act(z) and, where asked for, act'(z).  A NaN stays one.  16-bit rows keep 8 or 11 bits of them
// and take short forms, whose arithmetic bounds kernels beside their bytes; fp32 rows have both
// the time and the use for exponents of more bits than fp32: rms errors of SiLU 5.1e-8 of the value,
// GELU 7.3e-8, its tanh form 4.8e-8 (an exponent rounded to fp32: 8e-8 for SiLU below 4, 4e-7 from 10 on).  What
// both cost (us, against factors that end at 2^-126 and fp32 by the short forms): SiLU 4096 x 2048
// bf16 forward with codes 15.8 -> 16.3, gradient from them 18.7 -> 19.0, fp32 26.4 -> 27.8 and 34.4 -> 35.3;
// without codes fp32 20.5 -> 20.7 and 42.7 -> 42.8.
template <int VALUES, int ACT, bool SLOPE>
__device__ __forceinline__ void activation_of(float z, float &a, float &slope)
{
    constexpr bool WIDE = VALUES == kValuesF32;
    if constexpr (ACT == kActivationNone) {
        a = z;
        slope = 1.f;
    } else if constexpr (ACT == kActivationRelu) {
        a = z <= 0.f ? 0.f : z;
        slope = z <= 0.f ? 0.f : z != z ? z : 1.f;
    } else if constexpr (ACT == kActivationSilu) {
        if constexpr (WIDE) {
            constexpr float by = (float)-kLog2e, by_rest = rest_of(-kLog2e);
            const float size = fminf(fabsf(z), 200.f), whole = rintf(size * by);
            const Power e(whole, fmaf(size, by_rest, fmaf(size, by, -whole)));
            const WideLogistic l(z < 0.f, e);
            a = z * l.value * l.times;
            if constexpr (SLOPE) slope = fmaf(z, l.rest, 1.f) * l.value * l.times;
        } else {
            const Logistic<VALUES> l(z);
            a = z * l.value * l.times;
            const float s = l.value * l.times;
            if constexpr (SLOPE) slope = fmaf(a, 1.f - s, s);
        }
    } else if constexpr (ACT == kActivationGelu) {
        // z times the normal distribution, from its smaller tail so that nothing
        // cancels: with x = |z| / sqrt 2 the tail is e^(-x^2) / 2 times e^(x^2) erfc(x), which
        // over r in (0, 1], r = 1 / (1 + 0.45 x), is r times a polynomial (a Chebyshev fit, as
        // rounded good to 6.2e-8 over x up to 2000)
        constexpr float density = 0.39894228040143267794f, by = (float)(-0.5 * kLog2e);
        // e and the tail are taken 2^32 times as large but for fp16, which has no numbers there
        constexpr float shift = VALUES == kValuesF16 ? 0.f : 32.f, half = VALUES == kValuesF16 ? 0.5f : 0x1p-33f;
        const float size = WIDE ? fminf(fabsf(z), 32.f) : fabsf(z), r = __builtin_amdgcn_rcpf(fmaf(0.31819805153394638598f, size, 1.f));
        const float square = size * size;
        float e, p = kTail[9];
        if constexpr (WIDE) {
            const float whole = rintf(square * by), rest = fmaf(square, rest_of(-0.5 * kLog2e), fmaf(size, size, -square) * by);
            e = ldexpf(__builtin_amdgcn_exp2f(fmaf(square, by, -whole) + rest), (int)whole + 32);
        } else {
            e = __builtin_amdgcn_exp2f(fmaf(square, by, shift));
        }
#pragma unroll
        for (int i = 8; i >= 0; --i) p = fmaf(p, r, kTail[i]);
        const float w = e * (r * p);
        const float c = z > 0.f ? fmaf(w, -half, 1.f) : w, times = z > 0.f ? 1.f : half;
        a = z * c * times;
        if constexpr (SLOPE) slope = fmaf(z * (2.f * half * density), e, c * times);
    } else {
        // 0.5 z (1 + tanh(u)) = z logistic(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3)
        constexpr double k64 = 1.59576912160573071176, c64 = 0.044715;
        constexpr float k = (float)k64, c3 = (float)c64;
        // (beyond 16 in size the slope is 0 or 1; of infinite squares it would be no number)
        const float held = __builtin_amdgcn_fmed3f(z, -64.f, 64.f), dy = k * fmaf(3.f * c3 * held, held, 1.f);
        if constexpr (WIDE) {
            // -|y| log2 e = u v, u = -k log2 e |z| and v = 1 + c3 z^2, each with what its rounding left
            constexpr float by = (float)(-k64 * kLog2e), by_rest = rest_of(-k64 * kLog2e);
            const float size = fminf(fabsf(z), 16.f), square = size * size;
            const float u = size * by, u_rest = fmaf(size, by_rest, fmaf(size, by, -u));
            const float v = fmaf(c3, square, 1.f);
            const float v_rest = fmaf(c3, square, 1.f - v) + fmaf(rest_of(c64), square, c3 * fmaf(size, size, -square));
            const float whole = rintf(u * v);
            const Power e(whole, fmaf(u, v, -whole) + fmaf(u, v_rest, v * u_rest));
            const WideLogistic l(z < 0.f, e);
            a = z * l.value * l.times;
            if constexpr (SLOPE) slope = z != z ? z : fmaf(held * l.rest, dy, 1.f) * l.value * l.times;
        } else {
            const Logistic<VALUES> l(k * z * fmaf(c3 * z, z, 1.f));
            a = z * l.value * l.times;
            const float s = l.value * l.times;
            if constexpr (SLOPE) slope = fmaf(a * (1.f - s), dy, s);
        }
    }
}
template <int VALUES, int ACT>
__device__ __forceinline__ float activated(float z)
{
    float a, slope;
    activation_of<VALUES, ACT, false>(z, a, slope);
    return a;
}
}  // namespace

}  // namespace gtmoe
