// pairs.cuh — two fp32 operations an instruction (mul.rn.f32x2, fma.rn.f32x2):
// each half is rounded as the scalar operation would.
#pragma once

#include <cuda_runtime.h>

namespace drift {

using f2 = unsigned long long;
__device__ __forceinline__ f2 f2_pack(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ f2 f2_both(float a) { return f2_pack(a, a); }
__device__ __forceinline__ void f2_split(f2 x, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ f2 f2_mul(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// a + b, rounded: `one` is 1 in both halves, as a value that the compiler does not
// know. The assembler contracts a product and an add.rn.f32x2 into one fused
// operation, against -fmad=false; this sum it cannot.
__device__ __forceinline__ f2 f2_add(f2 a, f2 b, f2 one) { return f2_fma(a, one, b); }

}  // namespace drift
