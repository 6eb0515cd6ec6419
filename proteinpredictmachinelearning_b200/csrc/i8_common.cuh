// i8_common.cuh -- what the 8-bit integer product's kernels share: element types, the token quantizer's arithmetic and the
// epilogue of the product.
//
//   scale[t] = max_k |x[t][k]| / 127            q[t][k] = clamp(rint(x[t][k] / scale[t]), -127, 127)
//   C[m][n]  = act(a_scale[m] * b_scale[n] * sum_k A[m][k] B[n][k] + bias[n]) * gate[m][n]
//
// The sum is exact in int32 for every K up to kI8MaxK (128 * 128 * 131071 < 2^31), so no result depends on how a kernel
// splits K.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.h"

namespace ppml_b200 {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Magnitudes are compared as integers: the order of |x| for finite values, with infinities and NaN above all of them.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale of a row whose largest magnitude is `bits`.  A row that holds an infinity or a NaN has no scale: its result is NaN.
__device__ __forceinline__ float i8_scale(uint32_t bits) {
    return bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __fdiv_rn(__uint_as_float(bits), 127.0f);
}
// A scale of 0 (a row of zeros, or of numbers so small that the quotient underflows) or NaN gives 0.  The clamp only acts
// where the scale is subnormal and lost its low bits.
__device__ __forceinline__ int i8_quantize(float x, float scale) {
    if (!(scale > 0.0f)) return 0;
    const float r = rintf(__fdiv_rn(x, scale));
    return static_cast<int>(fminf(fmaxf(r, -127.0f), 127.0f));
}

// The activations of act_scalar with sigmoid, SiLU and GELU through the hardware's exp2 and reciprocal (about 2 ulp each, the
// exponent's argument rounded once; expf and an IEEE division cost a dozen instructions more per output):
// 0.5 x (1 + tanh(u)) = x * sigmoid(2 u).  tanh itself stays exact: 2 sigmoid(2 x) - 1 would cancel near 0.
__device__ __forceinline__ float i8_sigmoid(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}
__device__ __forceinline__ float i8_act(int kind, float x) {
    switch (kind) {
        case 1: return i8_sigmoid(x);
        case 2: return x * i8_sigmoid(x);
        case 3: return x * i8_sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
        case 4: return tanhf(x);
        case 5: return x < 0.0f ? 0.0f : x;            // keeps NaN
        default: return x;
    }
}
__device__ __forceinline__ float i8_epilogue(int sum, float a_scale, float b_scale, float bias, int act) {
    return i8_act(act, fmaf(static_cast<float>(sum) * a_scale, b_scale, bias));
}

}  // namespace ppml_b200
