// Activations of a FullConnect layer with their slopes, and the element types of its tensors.
#pragma once
#include "../../include/alpha_conv_b200.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace alpha {

// Sigmoid of z, and of -z, from one exponential of a value that cannot overflow: neither loses the digits that 1 - s would, nor is there a quotient by more than
// 2^126, for which __fdividef gives 0 (silu(-88) is -5e-37, no denormal).
struct Sigmoid { float pos, neg; };
template <bool FAST> __device__ __forceinline__ Sigmoid sigmoid_both(float z)
{
    const float e = FAST ? __expf(-fabsf(z)) : expf(-fabsf(z));
    const float big = __fdividef(1.f, 1.f + e), small = e * big;
    return z >= 0.f ? Sigmoid{big, small} : Sigmoid{small, big};
}

// The normal distribution function at z and exp(-z^2 / 2), to 9e-6 of its value for |z| < 9: with x = |z| / sqrt(2), erfc(x) = exp(-x^2) erfcx(x), and
// erfcx(x) as a polynomial in t = 1 / (1 + 0.44 x), fitted by weighted least squares for 0 <= x <= 12 (relative error 5.2e-6).  Enough for results
// of 11 bits; erfcf with an exponential beside it took twice the time of the whole gradient pass (117 us instead of 60, 4096 x 11008).
struct NormalCdf { float cdf, exp; };
__device__ __forceinline__ NormalCdf normal_cdf_16(float z)
{
    const float t = __fdividef(1.f, fmaf(0.44f * 0.70710678f, fabsf(z), 1.f)), e = __expf(-0.5f * z * z);
    float p = fmaf(t, -0.14610653f, 0.35065508f);
    p = fmaf(t, p, 0.0407281f);
    p = fmaf(t, p, 0.26358804f);
    p = fmaf(t, p, 0.24256907f);
    p = fmaf(t, p, 0.24856107f);
    const float tail = 0.5f * t * p * e;
    return NormalCdf{z >= 0.f ? 1.f - tail : tail, e};
}

// k z of a LeakyReLU.  With k = 0 it is a ReLU, whose value at -Inf is 0 and not the NaN of 0 * -Inf; a NaN stays one.
__device__ __forceinline__ float leaky(float z, float k)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(z), "f"(k == 0.f ? -0x1.fffffep127f : -__int_as_float(0x7f800000)));
    return k * y;
}

// Value and slope of activation ACT at z.  Quotients err by 2 units of 2^-23, exponentials by as much, or (FAST, for results that are rounded to
// 16 bits) by 2 + |argument| units.  z = -Inf gives NaN where the definition is -Inf * 0 (silu, gelu, gelu_tanh).
template <int ACT, bool FAST> __device__ __forceinline__ float act_value(float z, float k)
{
    if constexpr (ACT == ALPHA_ACT_NONE) return z;
    else if constexpr (ACT == ALPHA_ACT_LEAKY_RELU) return z > 0.f ? z : leaky(z, k);
    else if constexpr (ACT == ALPHA_ACT_SIGMOID) return sigmoid_both<FAST>(z).pos;
    else if constexpr (ACT == ALPHA_ACT_SILU) return z * sigmoid_both<FAST>(z).pos;
    else if constexpr (ACT == ALPHA_ACT_GELU) return FAST ? z * normal_cdf_16(z).cdf : 0.5f * z * erfcf(-0.70710678f * z);
    else {
        // z (1 + tanh(u)) / 2 = z sigmoid(2 u)
        return z * sigmoid_both<FAST>(1.59576912f * (z + 0.044715f * z * z * z)).pos;
    }
}
template <int ACT, bool FAST> __device__ __forceinline__ void act_both(float z, float k, float& value, float& slope)
{
    if constexpr (ACT == ALPHA_ACT_NONE) { value = z; slope = 1.f; }
    else if constexpr (ACT == ALPHA_ACT_LEAKY_RELU) { slope = z > 0.f ? 1.f : k; value = z > 0.f ? z : leaky(z, k); }
    else if constexpr (ACT == ALPHA_ACT_SIGMOID) {
        const Sigmoid s = sigmoid_both<FAST>(z);
        value = s.pos; slope = s.pos * s.neg;
    } else if constexpr (ACT == ALPHA_ACT_SILU) {
        const Sigmoid s = sigmoid_both<FAST>(z);
        value = z * s.pos; slope = s.pos * (1.f + z * s.neg);
    } else if constexpr (ACT == ALPHA_ACT_GELU) {
        const NormalCdf n = FAST ? normal_cdf_16(z) : NormalCdf{0.5f * erfcf(-0.70710678f * z), expf(-0.5f * z * z)};
        value = z * n.cdf; slope = n.cdf + z * 0.39894228f * n.exp;
    } else {
        const Sigmoid s = sigmoid_both<FAST>(1.59576912f * (z + 0.044715f * z * z * z));
        // (from |z| = 16 on the slope is 0 or 1, and the square of a larger z may overflow)
        const float c = fminf(fmaxf(z, -16.f), 16.f);
        value = z * s.pos; slope = s.pos * (1.f + c * s.neg * 1.59576912f * (1.f + 0.134145f * c * c));
    }
}

// f(std::integral_constant<int, ACT>) for the activation of a call: the choice is made once, outside the loops over elements.
template <class F> __host__ __device__ __forceinline__ void with_act(int act, F&& f)
{
    switch (act) {
    case ALPHA_ACT_NONE: f(std::integral_constant<int, ALPHA_ACT_NONE>{}); break;
    case ALPHA_ACT_LEAKY_RELU: f(std::integral_constant<int, ALPHA_ACT_LEAKY_RELU>{}); break;
    case ALPHA_ACT_SIGMOID: f(std::integral_constant<int, ALPHA_ACT_SIGMOID>{}); break;
    case ALPHA_ACT_SILU: f(std::integral_constant<int, ALPHA_ACT_SILU>{}); break;
    case ALPHA_ACT_GELU: f(std::integral_constant<int, ALPHA_ACT_GELU>{}); break;
    default: f(std::integral_constant<int, ALPHA_ACT_GELU_TANH>{}); break;
    }
}

// ---- element types ----------------------------------------------------------------------------------------------

// Two elements of a 32-bit word as floats and back, each rounded to nearest.
template <class T> __device__ __forceinline__ void unpack16(uint32_t w, float& a, float& b);
template <> __device__ __forceinline__ void unpack16<__nv_bfloat16>(uint32_t w, float& a, float& b)
{
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
}
template <> __device__ __forceinline__ void unpack16<__half>(uint32_t w, float& a, float& b)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x; b = f.y;
}
template <class T> __device__ __forceinline__ uint32_t pack16(float a, float b);
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack16<__half>(float a, float b)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// A 16-byte word of a tensor as floats and back: 4 elements of fp32, 8 of the 16-bit types.
template <class T> struct Word16 {
    static constexpr int N = 8;
    __device__ static void load(const uint4& w, float* f)
    {
        unpack16<T>(w.x, f[0], f[1]); unpack16<T>(w.y, f[2], f[3]); unpack16<T>(w.z, f[4], f[5]); unpack16<T>(w.w, f[6], f[7]);
    }
    __device__ static uint4 store(const float* f) { return make_uint4(pack16<T>(f[0], f[1]), pack16<T>(f[2], f[3]), pack16<T>(f[4], f[5]), pack16<T>(f[6], f[7])); }
    static constexpr bool kFast = true;
};
template <> struct Word16<float> {
    static constexpr int N = 4;
    __device__ static void load(const uint4& w, float* f)
    {
        f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
    }
    __device__ static uint4 store(const float* f) { return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])); }
    static constexpr bool kFast = false;
};

}  // namespace alpha
