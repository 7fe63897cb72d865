// The plain forms of grouped_large.h's kernel, and when a product takes it.
#include "grouped_large.h"

namespace gtmoe {

namespace {

template <class T>
hipError_t launch_values(const GroupedArgs &a, int direction, hipStream_t s)
{
    const dim3 grid(kCus), block(kThreads);
    switch (direction) {
    case kGroupedForward:
        if (a.term.index) hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedForward, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedForward, false>), grid, block, 0, s, a);
        break;
    case kGroupedInputGradient: hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedInputGradient, false>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedWeightGradient, false>), grid, block, 0, s, a); break;
    }
    return hipGetLastError();
}

}  // namespace

// The weight gradient from 128 tiles on (16 experts of 2048 x 1024, 512 tiles: 64
// rows 32.1 -> 26.7 us, 4096 rows 43.4 -> 35.1; 8 of 512 x 256, 16 tiles: 5.9
// against 10.7), the others from 112 rows per group on average and, by the
// rows' average, more than 128 tiles (64 experts of 2048 -> 1024: 64 rows each
// 54.0 against 66.0, 128 rows 92.3 -> 78.3; 16 of 1024 -> 2048: 128 rows, 128 tiles,
// 21.4 against 23.4, 256 rows, 192 tiles, 37.5 -> 28.1; input gradient of the
// latter, 96 tiles, 28.7 against 33.8).  bf16, against 128 x 128 tiles.
// With an epilogue the same holds (bf16, against the tiles of grouped.hip with it): 8192 rows of 1024 ->
// 2048 with biases 38.7 against 46.6, a residual 40.0 against 45.5, biases, SiLU, factor and z kept 53.0
// against 61.8; 16 groups of 1024 -> 2048, 1024 rows each 101.9 against 121.2 with all of these and 119.5
// against 138.3 of uneven groups; 64 of 2048 -> 1024, 128 rows each 92.0 against 106.9.  Equal groups
// of one whole tile's rows go the other way (16 of 256 rows 41.2 against 36.6) where uneven ones of
// as many rows do not (44.1 against 54.6), and the host knows neither.
bool large_fits(const GroupedArgs &a, int direction, int value_bytes)
{
    if (value_bytes != 2) return false;
    const long long columns = ((direction == kGroupedForward ? a.outputs : a.inputs) + kBn - 1) / kBn;
    if (direction == kGroupedWeightGradient) {
        const long long tiles = (a.outputs + kBm - 1) / kBm * columns * a.groups;
        return tiles >= 128 && tiles < 1 << 30;
    }
    const long long most = (a.rows / 64 + a.groups) * columns, likely = (a.rows / 256 + a.groups / 2) * columns;
    return a.rows / 112 >= a.groups && likely > 128 && most < 1 << 30;
}

hipError_t launch_large(const GroupedArgs &a, int direction, int values, hipStream_t s)
{
    if (direction == kGroupedForward && a.epilogue.on) return launch_large_fused(a, values, s);
    return values == kValuesBf16 ? launch_values<Bf16>(a, direction, s) : launch_values<F16>(a, direction, s);
}

}  // namespace gtmoe
