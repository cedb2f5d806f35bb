// Float32 sums and products with one rounding each, for arithmetic that is held to a sequence of separately rounded operations.  __fmul_rn() and the like are plain
// operators that the compiler fuses; which of them it leaves alone hangs on the instructions it may choose from.
#pragma once
#include <hip/hip_runtime.h>

namespace ss {

__device__ __forceinline__ float mul_rn(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}
__device__ __forceinline__ float add_rn(float a, float b) {
#pragma clang fp contract(off)
    return a + b;
}
__device__ __forceinline__ float sub_rn(float a, float b) {
#pragma clang fp contract(off)
    return a - b;
}

}  // namespace ss
