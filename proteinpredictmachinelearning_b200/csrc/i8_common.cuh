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

// two values rounded and packed, the first in the low half
__device__ __forceinline__ uint32_t narrow2(float a, float b, __nv_bfloat16) { const __nv_bfloat162 t = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&t); }
__device__ __forceinline__ uint32_t narrow2(float a, float b, __half) { const __half2 t = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&t); }

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
// 1 / scale for i8_quantize_all; 0 where its shortcut does not hold
__device__ __forceinline__ float i8_inverse(float scale) { return scale > 1e-30f && scale < 1e30f ? __frcp_rn(scale) : 0.0f; }
// N values (a multiple of 4) as packed bytes, the same as i8_quantize, two values an instruction and without a division: with
// inv = 1 / scale rounded to nearest, y = x * inv corrected once by its remainder is within one unit in the last place of the
// quotient, and corrected a second time it is the correctly rounded quotient (Markstein's theorem).  A shortcut that took the
// quotient only for products next to a half was slower: a third of the warps holds such a value when x is bf16.  Adding
// 1.5 * 2^23 rounds to an integer (half to even) whose low byte is the result.
template <int N> __device__ __forceinline__ void i8_quantize_all(const float (&x)[N], float scale, float inv, uint32_t (&q)[N / 4]) {
    if (inv == 0.0f) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) q[i] = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) q[i / 4] |= (static_cast<uint32_t>(i8_quantize(x[i], scale)) & 255u) << (8 * (i & 3));
        return;
    }
    const uint64_t inv2 = pack2(inv, inv), minus2 = pack2(-scale, -scale), round2 = pack2(12582912.0f, 12582912.0f);
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        uint32_t b[4];
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const uint64_t v = pack2(x[i + k], x[i + k + 1]);
            uint64_t y = fmul2(v, inv2);
            y = ffma2(ffma2(y, minus2, v), inv2, y);
            y = ffma2(ffma2(y, minus2, v), inv2, y);
            float t0, t1;
            unpack2(fadd2(y, round2), t0, t1);
            b[k] = __float_as_uint(t0); b[k + 1] = __float_as_uint(t1);
        }
        q[i / 4] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
}

// 16 bytes of a row of x
template <typename T> struct Vec16 { static constexpr int kN = 16 / sizeof(T); };
// the largest magnitude among them, as fp32 bits; 16-bit types are compared two at a time
template <typename T> __device__ __forceinline__ uint32_t top_of(const uint4& v) {
    if constexpr (sizeof(T) == 4) {
        return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
    } else {
        const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
        const uint16_t h = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
        return magnitude_bits(to_f32(*reinterpret_cast<const T*>(&h)));
    }
}
template <typename T> __device__ __forceinline__ void unpack_vec(const uint4& v, float (&x)[Vec16<T>::kN]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else {
            const uint16_t lo = static_cast<uint16_t>(w[i] & 0xffffu), hi = static_cast<uint16_t>(w[i] >> 16);
            x[2 * i] = to_f32(*reinterpret_cast<const T*>(&lo));
            x[2 * i + 1] = to_f32(*reinterpret_cast<const T*>(&hi));
        }
    }
}
// 16 bytes of x as 4 (fp32) or 8 integers
template <typename T> __device__ __forceinline__ void quantize_vec(const uint4& v, float scale, float inv, uint32_t (&q)[Vec16<T>::kN / 4]) {
    float x[Vec16<T>::kN];
    unpack_vec<T>(v, x);
    i8_quantize_all(x, scale, inv, q);
}

// The activations of act_scalar with sigmoid, SiLU and GELU through the hardware's exp2 and reciprocal (expf and an IEEE division
// cost a dozen instructions more per output): 0.5 x (1 + tanh(u)) = x * sigmoid(2 u).  tanh itself stays exact: 2 sigmoid(2 x) - 1
// would cancel near 0.  With u = 2^-24: exp2 is off by 4 u, the sum by u, the reciprocal by 2 u, the last product by u, and the
// exponent's argument by 1.22 u of itself, so that sigmoid(v) and SiLU are off by at most (8 + 2 |v|) u of their value, and GELU, whose
// v has five roundings and a constant more, by (8 + 8 |v|) u.  Below v = -87.3 the reciprocal is subnormal and flushed: 0.
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
// The same with CUDA's expf and IEEE divisions, which PATH_SIMT asks for: at most 8 u (GELU: (8 + 8 |v|) u) down to v = -88.7, where
// expf overflows.
__device__ __forceinline__ float i8_act_exact(int kind, float x) {
    switch (kind) {
        case 1: return 1.0f / (1.0f + expf(-x));
        case 2: return x / (1.0f + expf(-x));
        case 3: return x / (1.0f + expf(-1.5957691216057308f * (x + 0.044715f * x * x * x)));
        default: return i8_act(kind, x);
    }
}
// N values with one branch on the kind, or with none where it is a constant.  (Four values by a call that is not inlined took 80 cycles
// a value more, a branch per value filled the instruction cache.)
template <int N> __device__ __forceinline__ void i8_act_all(int kind, float (&y)[N]) {
#define PPML_ACT(K) case K: { _Pragma("unroll") for (int j = 0; j < N; ++j) y[j] = i8_act(K, y[j]); break; }
    switch (kind) { PPML_ACT(1) PPML_ACT(2) PPML_ACT(3) PPML_ACT(4) PPML_ACT(5) default: break; }
#undef PPML_ACT
}
__device__ __forceinline__ float i8_epilogue(int sum, float a_scale, float b_scale, float bias, const I8Product& p) {
    const float y = fmaf(static_cast<float>(sum) * a_scale, b_scale, bias);
    return p.exact ? i8_act_exact(p.act, y) : i8_act(p.act, y);
}

}  // namespace ppml_b200
