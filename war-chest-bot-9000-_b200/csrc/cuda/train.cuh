// Shared by the training operators' kernels (policy_loss.cu, block_norm.cu,
// act8.cu, wgrad8.cu): element types, row reductions, the 8-bit block code.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "train_ops.h"
#include "umma.cuh"

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

// Arithmetic on two 32-bit numbers in one instruction, each rounded as the scalar form
using Pair = unsigned long long;
__device__ __forceinline__ Pair twice(float v) { return umma::f2(v, v); }
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair add(Pair a, Pair b) { return umma::f2_add(a, b); }
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) { return umma::f2_fma(a, b, c); }
__device__ __forceinline__ float both(Pair a) { return umma::f2_lo(a) + umma::f2_hi(a); }
// ... of single numbers that hand NaN on
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Waits of at most `limit_ns`. A limit below a microsecond is one look, as the end of a sleep is not that exact.
constexpr uint64_t LOOK_NS = 1000;
__device__ __forceinline__ bool look_at(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(umma::smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ bool wait_within(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
    return look_at(bar, parity) || (limit_ns >= LOOK_NS && umma::mbar_wait(bar, parity, limit_ns));
}
// ... the first part of a wait, up to SLEEP_NS, asleep: a warp that polls takes issue slots and shared-memory cycles from
// the warps it waits for
constexpr uint64_t SLEEP_NS = 100000;
__device__ __forceinline__ bool sleep_on(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
    if (limit_ns < LOOK_NS) return look_at(bar, parity);
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(umma::smem_u32(bar)), "r"(parity), "r"((uint32_t)min(limit_ns, SLEEP_NS))
        : "memory");
    return done != 0;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The unit of an 8-bit block whose largest magnitude is `top`: the smallest
// power of two 2^e with top <= 127 2^e, as e + 127 (at least 1, so the unit
// and its reciprocal are normal numbers). top = 1.M 2^(E - 127); 64 (1.M)
// exceeds 127 just when M > 0x7e0000, where adding 0x1ffff carries into E. 255
// (an infinity or NaN in the block) reads back as NaN.
__device__ __forceinline__ uint32_t act8_code(float top) {
    const uint32_t b = __float_as_uint(top);
    return b >= 0x7f800000u ? 255u : (uint32_t)max((int)((b + 0x1ffffu) >> 23) - 6, 1);
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
__device__ __forceinline__ uint2 quantise8(const Pair* in, uint32_t* code) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max_nan(max_nan(top, fabsf(umma::f2_lo(in[i]))), fabsf(umma::f2_hi(in[i])));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    *code = act8_code(top);
    uint32_t b[8];
    if (*code < ACT8_LARGEST) {
        // adding 1.5 2^23 rounds to a whole number, ties to even, and leaves its two's complement in the low bits
        const Pair inv = twice(act8_inverse(*code)), round = twice(12582912.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Pair w = fma(in[i], inv, round);
            b[2 * i] = (uint32_t)w, b[2 * i + 1] = (uint32_t)(w >> 32);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            b[2 * i] = (uint8_t)act8_whole(umma::f2_lo(in[i]), *code), b[2 * i + 1] = (uint8_t)act8_whole(umma::f2_hi(in[i]), *code);
    }
    uint2 r;
    r.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    return r;
}
__device__ __forceinline__ uint2 quantise8(const float* v, uint32_t* code) {
    const Pair in[4] = {umma::f2(v[0], v[1]), umma::f2(v[2], v[3]), umma::f2(v[4], v[5]), umma::f2(v[6], v[7])};
    return quantise8(in, code);
}
// A byte as a number: 2^23 + 128 + q, as 32 bits hold it, less that (a conversion would wait for a slower unit)
__device__ __forceinline__ float act8_number(uint32_t q) { return __uint_as_float((q ^ 0x80u) | 0x4b000000u) - 8388736.0f; }
// 8 bytes back as values
__device__ __forceinline__ void dequantise8(uint2 q, uint32_t code, Pair* v) {
    const Pair unit = twice(act8_unit(code)), off = twice(-8388736.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = (i < 2 ? q.x : q.y) ^ 0x80808080u;
        v[i] = mul(add(umma::f2(__byte_perm(w, 0x4b000000u, i & 1 ? 0x7542 : 0x7540), __byte_perm(w, 0x4b000000u, i & 1 ? 0x7543 : 0x7541)), off),
                   unit);
    }
}

// GELU in its tanh form is x s with s = 1 / (1 + exp(-2u)), u = sqrt(2/pi) (x + 0.044715 x^3): no cancellation for
// negative x. The hardware's power and reciprocal are good to a few 2^-23; where the power overflows the reciprocal is 0.
constexpr float GELU_U1 = 0.7978845608028654f, GELU_U3 = 0.044715f * 0.7978845608028654f, GELU_P = -2.8853900817779268f;
__device__ __forceinline__ float gelu_power(float t) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    return e;
}
__device__ __forceinline__ float gelu_reciprocal(float d) {
    float s;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(d));
    return s;
}
// (Below -1e4 it is 0, as at -1e4: -inf times a gate of 0 would be none.)
__device__ __forceinline__ Pair gelu(Pair v) {
    const Pair x = umma::f2(max_nan(umma::f2_lo(v), -1e4f), max_nan(umma::f2_hi(v), -1e4f));
    const Pair t = mul(x, fma(mul(x, x), twice(GELU_U3 * GELU_P), twice(GELU_U1 * GELU_P)));
    const Pair d = add(umma::f2(gelu_power(umma::f2_lo(t)), gelu_power(umma::f2_hi(t))), twice(1.0f));
    return mul(x, umma::f2(gelu_reciprocal(umma::f2_lo(d)), gelu_reciprocal(umma::f2_hi(d))));
}
__device__ __forceinline__ float gelu(float v) { return umma::f2_lo(gelu(umma::f2(v, v))); }
// Its derivative s + 2 x s (1 - s) u'(x); 1 - s is e s (e the power), again without cancellation. With e held to 2^126
// nothing overflows up to |x| = 2^27, from where the second term is 0 in 32 bits.
__device__ __forceinline__ Pair gelu_slope(Pair x) {
    const Pair x2 = mul(x, x), t = mul(x, fma(x2, twice(GELU_U3 * GELU_P), twice(GELU_U1 * GELU_P)));
    const Pair e = umma::f2(gelu_power(min_nan(umma::f2_lo(t), 126.0f)), gelu_power(min_nan(umma::f2_hi(t), 126.0f)));
    const Pair d = add(e, twice(1.0f)), s = umma::f2(gelu_reciprocal(umma::f2_lo(d)), gelu_reciprocal(umma::f2_hi(d)));
    const Pair v = mul(x, fma(x2, twice(6.0f * GELU_U3), twice(2.0f * GELU_U1)));
    return fma(v, mul(mul(e, s), s), s);
}
// ... of values of a block; where its unit makes them larger than that they are cut to a size at which the slope is 0 or 1
__device__ __forceinline__ void gelu_cut(uint32_t code, Pair* v, int n) {
    if (code <= 147 || code == 255) return;
    for (int i = 0; i < n; ++i)
        v[i] = umma::f2(fminf(fmaxf(umma::f2_lo(v[i]), -1048576.0f), 1048576.0f), fminf(fmaxf(umma::f2_hi(v[i]), -1048576.0f), 1048576.0f));
}

}  // namespace wctrain
