// Dropout whose mask is a function of a counter and never stored:
//   out[r][c] = base[r][c] + (keep(r, c) ? x[row(r)][c] * scale : 0)
// keep takes 16 bits of Philox4x32 with ten rounds (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): the eight
// columns 8 b .. 8 b + 7 of row r are the low and high halves of the four words
// of counter (b, r, offset low, offset high) under the key (seed low, seed
// high), and a value is kept where its 16 bits are at least `threshold`.
// The gradient of x is the same function of the output's gradient.
//
// Sixteen bits per value instead of 32 halve the random numbers: a counter's
// ten rounds (twenty 32 x 32 -> 64 products) serve eight values.  scale is
// 65536 / (65536 - threshold), the inverse of the share that is kept exactly.
// A dropped value is selected away, not multiplied by zero: infinities and
// NaN in dropped places do not reach the output.
//
// What bounds it (MI355X): memory, with the ten rounds' quarter-rate products
// close behind.  8192 x 2048 in bf16, with and without a base, 39 us for both calls:
// 168 MB at 4.3 TB/s, where a large copy reaches 5.1.  A thread that steps
// through rows and columns without the 64-bit division per item, on as many
// workgroups as the chip holds, took 40 us.
#include "grouped.h"

namespace gtmoe {

namespace {

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1)
{
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int VALUES>
struct Kind;
template <>
struct Kind<kValuesF32> {
    typedef float Store;
    static __device__ __forceinline__ float load(float v) { return v; }
    static __device__ __forceinline__ float round(float v) { return v; }
};
template <>
struct Kind<kValuesBf16> {
    typedef uint16_t Store;
    static __device__ __forceinline__ float load(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t round(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <>
struct Kind<kValuesF16> {
    typedef uint16_t Store;
    static __device__ __forceinline__ float load(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ uint16_t round(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// Eight values of a row, any alignment; n of them exist.
template <class S>
__device__ __forceinline__ void load8(const S *p, S (&v)[8], int n)
{
    if (n >= 8) {
        __builtin_memcpy(v, p, sizeof v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (S)0;
    }
}

template <int VALUES>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a, int blocks)
{
    typedef Kind<VALUES> K;
    typedef typename K::Store Store;
    const long long total = (long long)a.rows * blocks;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int r = (int)(i / blocks), b = (int)(i - (long long)r * blocks);
        const int n = a.columns - 8 * b;
        const int src = a.index ? a.index[r] : r;
        Store x[8], y[8];
        load8(reinterpret_cast<const Store *>(a.x) + src * a.ldx + 8 * b, x, n);
        const Words w = philox(b, r, (uint32_t)a.offset, (uint32_t)(a.offset >> 32), (uint32_t)a.seed,
                               (uint32_t)(a.seed >> 32));
        if (a.base) load8(reinterpret_cast<const Store *>(a.base) + r * a.ldbase + 8 * b, y, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t bits = (w.w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
            const float v = bits >= a.threshold ? K::load(x[e]) * a.scale : 0.f;
            y[e] = K::round(a.base ? K::load(y[e]) + v : v);
        }
        Store *out = reinterpret_cast<Store *>(a.out) + r * a.ldo + 8 * b;
        if (n >= 8) {
            __builtin_memcpy(out, y, sizeof y);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) out[e] = y[e];
        }
    }
}

}  // namespace

hipError_t launch_dropout(const DropoutArgs &a, int values, hipStream_t s)
{
    if (a.rows == 0 || a.columns == 0) return hipSuccess;
    const int blocks = (a.columns + 7) / 8;
    const long long total = (long long)a.rows * blocks;
    const unsigned grid = (unsigned)((total + 255) / 256 < 65536 ? (total + 255) / 256 : 65536);
    switch (values) {
    case kValuesBf16: hipLaunchKernelGGL(dropout_kernel<kValuesBf16>, dim3(grid), dim3(256), 0, s, a, blocks); break;
    case kValuesF16: hipLaunchKernelGGL(dropout_kernel<kValuesF16>, dim3(grid), dim3(256), 0, s, a, blocks); break;
    default: hipLaunchKernelGGL(dropout_kernel<kValuesF32>, dim3(grid), dim3(256), 0, s, a, blocks); break;
    }
    return hipGetLastError();
}

}  // namespace gtmoe
