// Shared by the training operators' kernels (policy_loss.cu, block_norm.cu,
// act8.cu, wgrad8.cu): element types, row reductions, the 8-bit block code.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "train_ops.h"

namespace wctrain {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the CTA in a fixed order; every thread gets it. `s` holds one
// float per warp; the call ends with the array free for the next one.
__device__ __forceinline__ float cta_sum(float v, float* s) {
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (lane == 0) s[warp] = v;
    __syncthreads();
    float t = lane < nw ? s[lane] : 0.0f;
    t = warp_sum(t);
    __syncthreads();
    return t;
}

// The unit of an 8-bit block whose largest magnitude is `top`: the smallest
// power of two 2^e with top <= 127 2^e, as e + 127 (at least 1, so the unit
// and its reciprocal are normal numbers). top = 1.M 2^(E - 127); 64 (1.M)
// exceeds 127 just when M > 0x7e0000. 255 (an infinity or NaN in the block)
// reads back as NaN.
__device__ __forceinline__ uint32_t act8_code(float top) {
    const uint32_t b = __float_as_uint(top) & 0x7fffffffu, E = b >> 23;
    if (E == 255) return 255;
    const int c = (int)E - 6 + ((b & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return c < 1 ? 1u : (uint32_t)c;
}
__device__ __forceinline__ float act8_unit(uint32_t code) {
    return code == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(code << 23);
}
// 2^-e of a code; the product with a block's value is exact (or too small to round to anything but 0)
__device__ __forceinline__ float act8_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }

// At the largest unit a whole number stops at 63: 64 times it would be no number of 32 bits.
constexpr uint32_t ACT8_LARGEST = 249;
constexpr float ACT8_MOST = 0x1.f8p127f;
// one value of a block
__device__ __forceinline__ int8_t act8_whole(float v, uint32_t code) {
    if (code == 255) return 0;
    return (int8_t)__float2int_rn((code == ACT8_LARGEST ? fminf(fmaxf(v, -ACT8_MOST), ACT8_MOST) : v) * act8_inverse(code));
}

// A thread's 8 values of a block (4 threads next to each other hold one) as bytes, and the block's code.
// Magnitudes are compared as integers, where NaN is above infinity above the rest, so either shows in the code.
__device__ __forceinline__ uint2 quantise8(const float* in, uint32_t* code) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(in[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    *code = act8_code(__uint_as_float(top));
    if (*code == 255) return make_uint2(0, 0);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = in[i];
    if (*code == ACT8_LARGEST)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fminf(fmaxf(v[i], -ACT8_MOST), ACT8_MOST);
    const float inv = act8_inverse(*code);
    uint32_t b[8];
    // adding 1.5 2^23 rounds to a whole number, ties to even, and leaves its two's complement in the low bits
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(fmaf(v[i], inv, 12582912.0f));
    uint2 r;
    r.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    return r;
}

// 1 / (1 + exp(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3): GELU (tanh form) is x times it, with no cancellation for
// negative x. The hardware's power and reciprocal are good to a few 2^-23. Where the power overflows the reciprocal is 0.
__device__ __forceinline__ float gelu_gate(float x2, float x, float* e) {
    const float u = x * fmaf(0.044715f * 0.7978845608f, x2, 0.7978845608f);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(*e) : "f"(-2.8853900817779268f * u));
    float s;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + *e));
    return s;
}
// (x = -inf has u = -inf and a gate of 0: GELU there is its limit 0, not -inf 0)
__device__ __forceinline__ float gelu(float x) {
    float e;
    const float s = gelu_gate(x * x, x, &e);
    return s == 0.0f ? s * 0.0f : x * s;
}
// Its derivative s + 2 x s (1 - s) u'(x); 1 - s is e s, again without cancellation. Beyond |x| = 10 it is 0 or 1 in 32
// bits, and the products of what grows with what vanishes are left out.
__device__ __forceinline__ float gelu_slope(float x) {
    const float x2 = x * x;
    float e;
    const float s = gelu_gate(x2, x, &e), du = fmaf(3.0f * 0.044715f * 0.7978845608f, x2, 0.7978845608f);
    return fabsf(x) > 10.0f ? s : fmaf(2.0f * x * du, (e * s) * s, s);
}

}  // namespace wctrain
