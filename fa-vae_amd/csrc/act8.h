// Device helpers shared by the residual-block operators (groupnorm.hip, linear.hip, ckpt8.hip): vectors of 1 to 8 elements, the
// activations with their derivatives, and the 8-bit activation format.
#pragma once
#include <type_traits>
#include "common.h"
#include "favae_hip.h"

// ---- vectors -------------------------------------------------------------------------------------------------------------
// VEC elements of T in registers as they lie in memory; converted to fp32 where they are used (half the registers for bf16)
template <class T, int VEC> struct VecOf;
template <> struct VecOf<float, 4> { typedef float4 raw; };
template <> struct VecOf<float, 2> { typedef float2 raw; };
template <> struct VecOf<float, 1> { typedef float raw; };
template <> struct VecOf<bf16_t, 8> { typedef uint4 raw; };
template <> struct VecOf<bf16_t, 2> { typedef unsigned raw; };
template <> struct VecOf<bf16_t, 1> { typedef bf16_t raw; };

__device__ __forceinline__ void vec_get(float (&f)[4], const float4& r) { f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w; }
__device__ __forceinline__ void vec_get(float (&f)[2], const float2& r) { f[0] = r.x; f[1] = r.y; }
__device__ __forceinline__ void vec_get(float (&f)[1], const float& r) { f[0] = r; }
__device__ __forceinline__ void vec_get(float (&f)[8], const uint4& r) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
}
__device__ __forceinline__ void vec_get(float (&f)[2], const unsigned& r) {
    f[0] = __uint_as_float(r << 16);
    f[1] = __uint_as_float(r & 0xffff0000u);
}
__device__ __forceinline__ void vec_get(float (&f)[1], const bf16_t& r) { f[0] = bf16_to_f32(r); }

__device__ __forceinline__ void vec_put(float4& r, const float (&f)[4]) { r = make_float4(f[0], f[1], f[2], f[3]); }
__device__ __forceinline__ void vec_put(float2& r, const float (&f)[2]) { r = make_float2(f[0], f[1]); }
__device__ __forceinline__ void vec_put(float& r, const float (&f)[1]) { r = f[0]; }
__device__ __forceinline__ void vec_put(uint4& r, const float (&f)[8]) {
    r = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void vec_put(unsigned& r, const float (&f)[2]) { r = pack_bf16x2(f[0], f[1]); }
__device__ __forceinline__ void vec_put(bf16_t& r, const float (&f)[1]) { r = f32_to_bf16(f[0]); }

// ---- activations ---------------------------------------------------------------------------------------------------------
// sigmoid(t).  bf16 data: the hardware's exp2 and reciprocal (a few 2^-24 of relative error each, against a 2^-9 rounding of the
// result); fp32 data: expf and the division.  t -> -inf gives 1 / inf = 0.
template <class T> __device__ __forceinline__ float sigmoid_of(float t) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t * -1.44269504088896341f));
    else return 1.f / (1.f + expf(-t));
}
constexpr float GELU_C = 1.59576912160573081f;        // sqrt(8 / pi): gelu_tanh(z) = z sigmoid(GELU_C (z + 0.044715 z^3))

template <class T, int ACT, int N> __device__ __forceinline__ void act_apply(float (&z)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if constexpr (ACT == FAVAE_ACT_SILU) z[j] = z[j] * sigmoid_of<T>(z[j]);
        if constexpr (ACT == FAVAE_ACT_GELU_TANH) z[j] = z[j] * sigmoid_of<T>(GELU_C * z[j] * fmaf(0.044715f * z[j], z[j], 1.f));
        if constexpr (ACT == FAVAE_ACT_LRELU) z[j] = z[j] > 0.f ? z[j] : 0.01f * z[j];
    }
}
// d[j] *= act'(z[j])
template <class T, int ACT, int N> __device__ __forceinline__ void act_grad_mul(float (&d)[N], const float (&z)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if constexpr (ACT == FAVAE_ACT_SILU) {
            const float s = sigmoid_of<T>(z[j]);
            d[j] *= s * fmaf(z[j], 1.f - s, 1.f);
        }
        if constexpr (ACT == FAVAE_ACT_GELU_TANH) {
            const float s = sigmoid_of<T>(GELU_C * z[j] * fmaf(0.044715f * z[j], z[j], 1.f));
            // past |z| = 20 s is 0 or 1 to the last bit and the second term vanishes; the bound keeps z^3 from overflowing there
            const float c = fminf(fmaxf(z[j], -20.f), 20.f);
            d[j] *= s * fmaf(c * (1.f - s), GELU_C * fmaf(0.134145f * c, c, 1.f), 1.f);
        }
        if constexpr (ACT == FAVAE_ACT_LRELU) d[j] = z[j] > 0.f ? d[j] : 0.01f * d[j];
    }
}
// f(std::integral_constant<int, act>): the choice is made once, outside the loops
template <class F> __device__ __forceinline__ void with_act(int act, F&& f) {
    if (act == FAVAE_ACT_SILU) f(std::integral_constant<int, FAVAE_ACT_SILU>());
    else if (act == FAVAE_ACT_GELU_TANH) f(std::integral_constant<int, FAVAE_ACT_GELU_TANH>());
    else if (act == FAVAE_ACT_LRELU) f(std::integral_constant<int, FAVAE_ACT_LRELU>());
    else f(std::integral_constant<int, FAVAE_ACT_NONE>());
}

template <int ACT, class F> __device__ __forceinline__ void act_choice(int act, F&& f) {
    if constexpr (ACT >= 0) f(std::integral_constant<int, ACT>());
    else with_act(act, f);
}
template <class F> void with_act_host(int act, F&& f) {
    if (act == FAVAE_ACT_SILU) f(std::integral_constant<int, FAVAE_ACT_SILU>());
    else if (act == FAVAE_ACT_GELU_TANH) f(std::integral_constant<int, FAVAE_ACT_GELU_TANH>());
    else if (act == FAVAE_ACT_LRELU) f(std::integral_constant<int, FAVAE_ACT_LRELU>());
    else f(std::integral_constant<int, FAVAE_ACT_NONE>());
}

// ---- 8-bit activations ---------------------------------------------------------------------------------------------------
// 32 channels of a row share a step 2^(code - 127): value = q * 2^(code - 127), q in [-127, 127].  The step is a power of two, so
// x / step and q * step are exact, the only rounding is rint, and a decoded value is a bf16 number whatever type it came from
// (7 bits of q): the matrix products of the backward pass read it without a further rounding.
constexpr int CK_BLOCK = 32;
__device__ __forceinline__ float ck_scale(unsigned code) { return __uint_as_float(code << 23); }   // 255 (inf or NaN in the block, q = 0): 0 * inf = NaN

// code of a block from the largest |x| as bits: the least step on which no value passes 127 steps.  Infinities and NaN order above
// every finite value as bits and give 255.  The step exponent stays in [-126, 121]: above, 127 steps would leave fp32's range.
__device__ __forceinline__ unsigned ck_code(unsigned amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255u;
    const int E = (int)(amax_bits >> 23);                       // floor(log2 amax) + 127
    int e = E - 133 < -126 ? -126 : E - 133;                    // amax / 2^e in [64, 128)
    const float top = rintf(__uint_as_float(amax_bits) * __uint_as_float((unsigned)(127 - e) << 23));
    if (top > 127.f && e < 121) ++e;
    return (unsigned)(e + 127);
}
__device__ __forceinline__ int ck_round(float x, unsigned code) {
    if (code == 255u) return 0;
    const float q = rintf(x * __uint_as_float((254u - code) << 23));
    return (int)fminf(fmaxf(q, -127.f), 127.f);
}
// value of byte j of w at step s: a conversion that selects and sign-extends its byte, and a product
__device__ __forceinline__ float ck_value(unsigned w, int j, float s) { return (float)(signed char)(w >> (8 * j)) * s; }
