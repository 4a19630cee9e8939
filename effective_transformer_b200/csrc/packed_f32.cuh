// Packed fp32 arithmetic (sm_100a): add, multiply and fused multiply-add on pairs, one issue slot for two elements, each
// rounded as the scalar instruction rounds.
#pragma once

#include <cuda_runtime.h>

namespace etb {

typedef float2 Pair;

__device__ __forceinline__ Pair pack2(float a, float b) { return make_float2(a, b); }
__device__ __forceinline__ void unpack2(const Pair& v, float& a, float& b) {
  a = v.x;
  b = v.y;
}
__device__ __forceinline__ Pair add2(const Pair& a, const Pair& b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ Pair mul2(const Pair& a, const Pair& b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ Pair fma2(const Pair& a, const Pair& b, const Pair& c) { return __ffma2_rn(a, b, c); }

}  // namespace etb
