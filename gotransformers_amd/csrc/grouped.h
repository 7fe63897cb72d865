// Declarations of the operators over plain rows (bf16, fp16 or fp32): ragged
// products grouped by expert, a shared projection with the adapters of many
// requests, and dropout.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gtmoe {

enum Values { kValuesF32 = 0, kValuesBf16 = 1, kValuesF16 = 2 };

inline int value_bytes(int values) { return values == kValuesF32 ? 4 : 2; }

// Low-rank adapters added to a product's rows: u [rows][ldu] fp32 holds
// s_a A_a x of every row with an adapter (zero beyond the rank, ldu a multiple
// of 8), up [adapters][N][rank].
struct AdapterTerm {
    const float *u = nullptr;
    const int32_t *adapter = nullptr;  // [rows]; outside [0, adapters): none
    const void *up = nullptr;
    int adapters = 0, rank = 0, ldu = 0;
    // rows sorted by adapter (grouped_large.hip): the sorted rows' places, group
    // `adapters` those without an adapter
    const int32_t *index = nullptr;
};

enum GroupedDirection { kGroupedForward = 0, kGroupedInputGradient = 1, kGroupedWeightGradient = 2 };

// One ragged product.  Strides in values.
//   forward          out[r][n] = sum_k a[r][k] b[g][n][k]
//   input gradient   out[r][k] = sum_n a[r][n] b[g][n][k]
//   weight gradient  out[g][n][k] (+)= sum_r a[r][n] b[r][k]
struct GroupedArgs {
    const int32_t *offsets = nullptr;  // [groups + 1]; null: one group of all rows
    int groups = 1, rows = 0, inputs = 0, outputs = 0;
    const void *a = nullptr, *b = nullptr;
    void *out = nullptr;
    long long lda = 0, ldb = 0, ldo = 0;
    long long group_stride = 0;  // of b, or of out for the weight gradient
    int out_f32 = 0;             // weight gradient: out holds fp32 whatever the operands' type
    int accumulate = 0;          // add to what out holds
    const void *bias = nullptr;  // [outputs], forward only
    AdapterTerm term;            // forward only
};

// Whether the product's tiles fit one launch.
bool grouped_fits(const GroupedArgs &a, int direction, int values);
hipError_t launch_grouped(const GroupedArgs &a, int direction, int values, hipStream_t s);

// The same for many rows of 16-bit values with both operands staged by LDS-DMA
// (grouped_large.hip).
bool large_fits(const GroupedArgs &a, int direction, int value_bytes);
hipError_t launch_large(const GroupedArgs &a, int direction, int values, hipStream_t s);
constexpr int kMaxSortedRank = 64;  // ranks of u in two steps

// u[t][j] = scales[a] sum_k down[a][j][k] x[t][k] for the rows with an adapter a,
// zero for the others.
struct AdapterDownArgs {
    const void *x = nullptr, *down = nullptr;
    const float *scales = nullptr;
    const int32_t *adapter = nullptr;
    float *u = nullptr;
    long long ldx = 0;
    int rows = 0, inputs = 0, rank = 0, adapters = 0, ldu = 0;
    const int32_t *index = nullptr;  // with sorted rows: their places, and adapter in the sorted order
};
hipError_t launch_adapter_down(const AdapterDownArgs &a, int values, hipStream_t s);
// The forward of one group with its adapters' term.
hipError_t launch_adapted(const GroupedArgs &a, int values, hipStream_t s);
// Whether both kernels' workgroups fit one launch each.
bool adapted_fits(const GroupedArgs &a, int values);
// Whether a forward with adapters takes its rows sorted by adapter
// (a.term.index): launch_adapter_sort first.
bool adapted_sorts(const GroupedArgs &a, int values);
// index [rows]: the rows by adapter, those without one last; sorted [rows]: the
// adapters in that order (`adapters`: none); offsets [adapters + 2]: where each
// adapter's begin.
hipError_t launch_adapter_sort(const int32_t *adapter, int rows, int adapters, int32_t *index, int32_t *sorted,
                               int32_t *offsets, hipStream_t s);

// out[r][c] = base[r][c] + (keep(r, c) ? x[index ? index[r] : r][c] * scale : 0),
// base null: no first term.
struct DropoutArgs {
    const void *x = nullptr, *base = nullptr;
    void *out = nullptr;
    const int32_t *index = nullptr;
    long long ldx = 0, ldbase = 0, ldo = 0;
    int rows = 0, columns = 0;
    uint32_t threshold = 0;  // of 65536: values whose 16 bits are below it are dropped
    float scale = 1.f;
    uint64_t seed = 0, offset = 0;
};
hipError_t launch_dropout(const DropoutArgs &a, int values, hipStream_t s);

}  // namespace gtmoe
