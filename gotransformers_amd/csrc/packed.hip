// Rows kept in 8 bits, and what a gated activation's backward takes from them:
//   y = act(min(gate, L)) clamp(up, -L, L)          (feedforward/gatedfeedforward.go:49-57,
//                                                    clamped: moreactivationfunctions.go:207-244)
//   dgate = dy clamp(up) act'(gate) [gate <= L],  dup = dy act(min(gate, L)) [|up| <= L]
// The forward writes y and, in the same pass, gate and up as codes with a scale per
// scale_columns columns; the gradient reads those instead of the 16-bit rows and
// makes y again, which the next product's weight gradient wants.
//
// A thread takes eight columns of a row; a scale's columns are two to sixteen
// neighbouring lanes, whose maximum they find by DPP.
//
// What bounds it (MI355X): memory, with arithmetic close behind in the forward with codes.
// 16384 x 2048 bf16, SiLU, int8 with a scale per 128 columns: forward 61 us (273 MB, 4.5 TB/s),
// gradient with y again 64 (340 MB, 5.3 TB/s); per 16 columns 59 and 66; without codes 39 and 75
// (201 and 403 MB).  2331 x 1201 fp32, GELU, E4M3 per 32: 13.6 and 15.0.  Packing 8192 x 2048
// fp16 rows per 16 columns 13.5 to 15, back 10.2.
#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace gtmoe {

namespace {

constexpr int kThreads = 256;

// Eight columns of a row per thread: rows are padded to whole scales, `per`
// threads each.
struct Place {
    long long row;
    int column;
};
__device__ __forceinline__ Place place_of(long long i, int per, bool narrow)
{
    if (narrow) {
        const uint32_t r = (uint32_t)i / (uint32_t)per;
        return {(long long)r, (int)((uint32_t)i - r * (uint32_t)per) * 8};
    }
    const long long r = i / per;
    return {r, (int)(i - r * per) * 8};
}

template <int VALUES>
__global__ __launch_bounds__(kThreads) void pack_kernel(PackArgs a, int per, long long total, bool narrow)
{
    for (long long i0 = (long long)blockIdx.x * kThreads; i0 < total; i0 += (long long)gridDim.x * kThreads) {
        const Place p = place_of(i0 + threadIdx.x, per, narrow);
        const int columns = p.row < a.rows ? a.columns : 0;
        Eight<VALUES> e;
        load_eight(e, a.x, p.row * a.ldx, p.column, columns);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = e.get(j);
        keep_eight<VALUES>(v, p.row, p.column, columns, a.kept);
    }
}

template <int VALUES>
__global__ __launch_bounds__(kThreads) void unpack_kernel(PackArgs a, int per, long long total, bool narrow)
{
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
        const Place p = place_of(i, per, narrow);
        if (!any_column<VALUES>(p.column, a.columns)) continue;
        float v[8];
        kept_eight<VALUES>(v, p.row, p.column, a.columns, a.kept);
        Eight<VALUES> e;
        e.set(v);
        store_eight(e, a.out, p.row * a.ldx, p.column, a.columns);
    }
}

// gate and up held within the limit (a NaN stays one); bit j: value j was beyond it.
struct Beyond {
    uint32_t gate = 0, up = 0;
};
__device__ __forceinline__ Beyond hold(float (&g)[8], float (&u)[8], float limit)
{
    Beyond b;
    if (limit == __builtin_inff()) return b;  // the same for all
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (g[j] > limit) {
            g[j] = limit;
            b.gate |= 1u << j;
        }
        if (fabsf(u[j]) > limit) {
            u[j] = copysignf(limit, u[j]);
            b.up |= 1u << j;
        }
    }
    return b;
}

template <int VALUES, int ACT>
__global__ __launch_bounds__(kThreads) void activation_forward_kernel(ActivationArgs a, int per, long long total, bool narrow)
{
    for (long long i0 = (long long)blockIdx.x * kThreads; i0 < total; i0 += (long long)gridDim.x * kThreads) {
        const Place p = place_of(i0 + threadIdx.x, per, narrow);
        const int columns = p.row < a.rows ? a.columns : 0;
        Eight<VALUES> ge, ue;
        load_eight(ge, a.gate, p.row * a.ldgate, p.column, columns);
        if (a.up) load_eight(ue, a.up, p.row * a.ldup, p.column, columns);
        float g[8], u[8], y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[j] = ge.get(j);
            u[j] = a.up ? ue.get(j) : 0.f;
        }
        if (a.kept_gate.codes) {
            keep_eight<VALUES>(g, p.row, p.column, columns, a.kept_gate);
            if (a.up) keep_eight<VALUES>(u, p.row, p.column, columns, a.kept_up);
        }
        if (!any_column<VALUES>(p.column, columns)) continue;
        hold(g, u, a.limit);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = activated<VALUES, ACT>(g[j]);
        if (a.up) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= u[j];
        }
        Eight<VALUES> e;
        e.set(y);
        store_eight(e, a.out, p.row * a.ldo, p.column, columns);
    }
}

template <int VALUES, int ACT>
__global__ __launch_bounds__(kThreads) void activation_gradient_kernel(ActivationArgs a, int per, long long total, bool narrow)
{
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (long long)gridDim.x * kThreads) {
        const Place p = place_of(i, per, narrow);
        if (!any_column<VALUES>(p.column, a.columns)) continue;
        const bool gated = a.up || a.kept_up.codes;
        Eight<VALUES> de;
        load_eight(de, a.dy, p.row * a.lddy, p.column, a.columns);
        float g[8], u[8];
        if (a.kept_gate.codes) {
            kept_eight<VALUES>(g, p.row, p.column, a.columns, a.kept_gate);
            if (gated) kept_eight<VALUES>(u, p.row, p.column, a.columns, a.kept_up);
        } else {
            Eight<VALUES> ge, ue;
            load_eight(ge, a.gate, p.row * a.ldgate, p.column, a.columns);
            if (gated) load_eight(ue, a.up, p.row * a.ldup, p.column, a.columns);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                g[j] = ge.get(j);
                if (gated) u[j] = ue.get(j);
            }
        }
        if (!gated) {
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = 0.f;
        }
        const Beyond beyond = hold(g, u, a.limit);
        float y[8], dg[8], du[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float act, slope;
            activation_of<VALUES, ACT, true>(g[j], act, slope);
            const float d = de.get(j), c = gated ? u[j] : 1.f;
            y[j] = act * c;
            dg[j] = d * c * slope;
            du[j] = d * act;
            // (eight at once would take registers, and so waves: GELU in bf16 79 instead of 66)
            if (j % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
        if (a.limit < __builtin_inff()) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (beyond.gate >> j & 1) dg[j] = 0.f;
                if (beyond.up >> j & 1) du[j] = 0.f;
            }
        }
        Eight<VALUES> e;
        if (a.dgate) {
            e.set(dg);
            store_eight(e, a.dgate, p.row * a.lddgate, p.column, a.columns);
        }
        if (a.dup) {
            e.set(du);
            store_eight(e, a.dup, p.row * a.lddup, p.column, a.columns);
        }
        if (a.out) {
            e.set(y);
            store_eight(e, a.out, p.row * a.ldo, p.column, a.columns);
        }
    }
}

// Threads of a row: whole scales, or groups of eight where there are none; of fp32
// whole 128 columns (column_of).
struct Grid {
    int per;
    long long total;
    bool narrow;
    dim3 blocks;
    Grid(int rows, int columns, int scale_columns, int values)
    {
        const int unit = values == kValuesF32 ? 128 : std::max(scale_columns, 8);
        per = (columns + unit - 1) / unit * (unit / 8);
        total = (long long)rows * per;
        narrow = total < (1ll << 31);
        blocks = dim3((unsigned)std::min<long long>((total + kThreads - 1) / kThreads, 1 << 20));
    }
};

template <class F>
hipError_t with_values(int values, F &&f)
{
    switch (values) {
    case kValuesBf16: return f(std::integral_constant<int, kValuesBf16>());
    case kValuesF16: return f(std::integral_constant<int, kValuesF16>());
    default: return f(std::integral_constant<int, kValuesF32>());
    }
}
template <class F>
hipError_t with_activation(int act, F &&f)
{
    switch (act) {
    case kActivationRelu: return f(std::integral_constant<int, kActivationRelu>());
    case kActivationSilu: return f(std::integral_constant<int, kActivationSilu>());
    case kActivationGelu: return f(std::integral_constant<int, kActivationGelu>());
    case kActivationGeluTanh: return f(std::integral_constant<int, kActivationGeluTanh>());
    default: return f(std::integral_constant<int, kActivationNone>());
    }
}

}  // namespace

hipError_t launch_pack(const PackArgs &a, int values, hipStream_t s)
{
    if (!a.kept.scale_columns) {
        // a scale per row: the norm's rows without a norm
        NormArgs n;
        n.x = a.x;
        n.ldx = a.ldx;
        n.kept = a.kept;
        n.rows = a.rows;
        n.columns = a.columns;
        n.norm = 0;
        return launch_norm_forward(n, values, s);
    }
    const Grid g(a.rows, a.columns, a.kept.scale_columns, values);
    return with_values(values, [&](auto v) {
        hipLaunchKernelGGL(pack_kernel<decltype(v)::value>, g.blocks, dim3(kThreads), 0, s, a, g.per, g.total, g.narrow);
        return hipGetLastError();
    });
}

hipError_t launch_unpack(const PackArgs &a, int values, hipStream_t s)
{
    const Grid g(a.rows, a.columns, 0, values);
    return with_values(values, [&](auto v) {
        hipLaunchKernelGGL(unpack_kernel<decltype(v)::value>, g.blocks, dim3(kThreads), 0, s, a, g.per, g.total, g.narrow);
        return hipGetLastError();
    });
}

hipError_t launch_activation(const ActivationArgs &a, bool gradient, int values, hipStream_t s)
{
    const Grid g(a.rows, a.columns, gradient ? 0 : a.kept_gate.scale_columns, values);
    return with_values(values, [&](auto v) {
        return with_activation(a.activation, [&](auto act) {
            constexpr int V = decltype(v)::value, A = decltype(act)::value;
            if (gradient)
                hipLaunchKernelGGL((activation_gradient_kernel<V, A>), g.blocks, dim3(kThreads), 0, s, a, g.per, g.total, g.narrow);
            else
                hipLaunchKernelGGL((activation_forward_kernel<V, A>), g.blocks, dim3(kThreads), 0, s, a, g.per, g.total, g.narrow);
            return hipGetLastError();
        });
    });
}

}  // namespace gtmoe
