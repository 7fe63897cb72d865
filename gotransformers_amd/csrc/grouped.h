// Declarations of the operators over plain rows (bf16, fp16 or fp32): ragged
// products grouped by expert, a shared projection with the adapters of many
// requests, dropout, norms, activations with 8-bit checkpoints, and the choice
// of experts.
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
    // rows sorted by adapter (grouped_large.h): the sorted rows' places, group
    // `adapters` those without an adapter
    const int32_t *index = nullptr;
};

// What a forward does with its products before they are rounded:
// out = act(W x + bias) factor + residual, W x + bias to `products` on the way.
struct Epilogue {
    int on = 0, activation = 0;
    const void *bias = nullptr, *factor = nullptr, *residual = nullptr;
    void *products = nullptr;
    long long ldbias = 0, ldfactor = 0, ldresidual = 0, ldproducts = 0;  // ldbias: between groups
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
    Epilogue epilogue;           // forward only, without a term
};

// Whether the product's tiles fit one launch.
bool grouped_fits(const GroupedArgs &a, int direction, int values);
hipError_t launch_grouped(const GroupedArgs &a, int direction, int values, hipStream_t s);
// The forward of few rows with an epilogue, W streamed (grouped_few.hip); staged: LDS-DMA
// could take both operands.
bool few_fits(const GroupedArgs &a, int value_bytes, bool staged);
hipError_t launch_few(const GroupedArgs &a, int values, hipStream_t s);

// The same for many rows of 16-bit values with both operands staged by LDS-DMA
// (grouped_large.h).
bool large_fits(const GroupedArgs &a, int direction, int value_bytes);
hipError_t launch_large(const GroupedArgs &a, int direction, int values, hipStream_t s);
hipError_t launch_large_fused(const GroupedArgs &a, int values, hipStream_t s);
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

// Rows in 8 bits: codes and, per scale_columns columns (0: per row), a scale.
struct PackedRows {
    uint8_t *codes = nullptr;
    float *scales = nullptr;
    long long ldcodes = 0, ldscales = 0;
    int code_type = 0, scale_columns = 0;
};
// Norm forward (norm.hip); norm 0: the rows as they are, into codes.
struct NormArgs {
    const void *x = nullptr, *residual = nullptr, *w = nullptr;
    void *sums = nullptr, *out = nullptr;
    PackedRows kept;  // without codes: none
    long long ldx = 0, ldresidual = 0, ldsums = 0, ldo = 0;
    int rows = 0, columns = 0, norm = 1;
    double epsilon = 0;
};
hipError_t launch_norm_forward(const NormArgs &a, int values, hipStream_t s);

// Sums of partial rows: of all `count`, or (each > 0) of those of group g's rows.
struct AddPartialsArgs {
    const void *partial = nullptr;  // fp32, or fp64 those of column sums
    void *out = nullptr;
    const int32_t *offsets = nullptr;
    long long ldo = 0;
    int columns = 0, count = 0, each = 0, rows = 0, groups = 1;
    int out_f32 = 0, accumulate = 0;
};
struct NormGradientArgs {
    const void *dy = nullptr, *s = nullptr, *w = nullptr, *ds = nullptr;
    void *dx = nullptr;
    float *partial = nullptr;  // a row of dw's sums per workgroup
    float *inverse = nullptr;  // of every row, as two factors, where dw is summed apart
    AddPartialsArgs into;      // set by the launcher: dw itself
    long long lddy = 0, lds = 0, ldds = 0, lddx = 0;
    int rows = 0, columns = 0;
    double epsilon = 0;
};
// Bytes of workspace with dw.
size_t norm_gradient_bytes(int rows, int columns);
// into.out null: no dw.
hipError_t launch_norm_gradient(NormGradientArgs a, float *workspace, const AddPartialsArgs &into, int values, hipStream_t s);

// Sums of rows by group in fp64, partial rows of `each` consecutive rows first.
struct ColumnSumsArgs {
    const void *x = nullptr, *v = nullptr;
    const float *inverse = nullptr;
    const int32_t *offsets = nullptr;
    double *partial = nullptr;
    long long ldx = 0, ldv = 0;
    int rows = 0, columns = 0, groups = 1, each = 0;
    AddPartialsArgs into;  // set by the launcher: the sums themselves
};
int sum_rows_each(int rows, int groups, int columns);
size_t sum_bytes(int rows, int groups, int columns);
hipError_t launch_column_sums(ColumnSumsArgs a, const AddPartialsArgs &add, int values, hipStream_t s);

struct PackArgs {
    const void *x = nullptr;  // packed from,
    void *out = nullptr;      // or unpacked into; rows ldx apart
    long long ldx = 0;
    int rows = 0, columns = 0;
    PackedRows kept;
};
hipError_t launch_pack(const PackArgs &a, int values, hipStream_t s);
hipError_t launch_unpack(const PackArgs &a, int values, hipStream_t s);

// A gated activation and its gradient (packed.hip).  Without up and its codes
// the activation alone.  kept_gate.codes: written by the forward, read by the
// gradient in place of gate and up.
struct ActivationArgs {
    const void *gate = nullptr, *up = nullptr, *dy = nullptr;
    void *out = nullptr, *dgate = nullptr, *dup = nullptr;
    PackedRows kept_gate, kept_up;
    long long ldgate = 0, ldup = 0, lddy = 0, ldo = 0, lddgate = 0, lddup = 0;
    int rows = 0, columns = 0, activation = 0;
    float limit = 0;  // infinite: none
};
hipError_t launch_activation(const ActivationArgs &a, bool gradient, int values, hipStream_t s);

// A token's experts and gates, and the rows in expert order (choose.hip).
struct ChooseArgs {
    const void *logits = nullptr;
    const float *biases = nullptr;
    int32_t *chosen = nullptr;
    float *gates = nullptr;
    int32_t *offsets = nullptr, *rows = nullptr, *places = nullptr;  // offsets null: no lists
    long long ldlogits = 0;
    int tokens = 0, experts = 0, k = 0, groups = 1, chosen_groups = 1, group_best = 1;
    int logistic = 0, renormalize = 0;
    double scale = 1.0;
    // set by the launcher: tokens per workgroup, what each counted, the sums before it
    int each = 0, ldcounts = 0;
    uint32_t group_inverse = 0;
    uint16_t *counts = nullptr;
    int *totals = nullptr, *before = nullptr;
};
// The workspace: counts, then (many workgroups) totals and sums.
struct ChooseLayout {
    int each = 0, blocks = 0, ldcounts = 0;
    size_t totals = 0, before = 0, bytes = 0;
};
ChooseLayout choose_layout(int tokens, int experts);
hipError_t launch_choose(ChooseArgs a, int values, void *workspace, hipStream_t s);

struct ChooseGradientArgs {
    const void *logits = nullptr;
    const int32_t *chosen = nullptr;
    const float *gate_gradients = nullptr;
    void *logit_gradients = nullptr;
    long long ldlogits = 0, ldgradients = 0;
    int tokens = 0, experts = 0, k = 0, logistic = 0, renormalize = 0;
    double scale = 1.0;
};
hipError_t launch_choose_gradient(const ChooseGradientArgs &a, int values, hipStream_t s);

}  // namespace gtmoe
