// grouped_large.h's kernel with an epilogue, one per activation.
#include "grouped_large.h"

namespace gtmoe {

namespace {

template <class T, int ACT>
hipError_t launch_fused(const GroupedArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL((grouped_large_kernel<T, kGroupedForward, false, ACT>), dim3(kCus), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_values(const GroupedArgs &a, hipStream_t s)
{
    switch (a.epilogue.activation) {
    case kActivationRelu: return launch_fused<T, kActivationRelu>(a, s);
    case kActivationSilu: return launch_fused<T, kActivationSilu>(a, s);
    case kActivationGelu: return launch_fused<T, kActivationGelu>(a, s);
    case kActivationGeluTanh: return launch_fused<T, kActivationGeluTanh>(a, s);
    default: return launch_fused<T, kActivationNone>(a, s);
    }
}

}  // namespace

hipError_t launch_large_fused(const GroupedArgs &a, int values, hipStream_t s)
{
    return values == kValuesBf16 ? launch_values<Bf16>(a, s) : launch_values<F16>(a, s);
}

}  // namespace gtmoe
