// Device helpers shared by the residual-block operators (groupnorm.hip, linear.hip, ckpt8.hip): vectors of 1 to 8 elements, the
// activations with their derivatives, and the 8-bit activation format.
#pragma once
#include <type_traits>
#include "common.h"
#include "favae_hip.h"

// ---- vectors -------------------------------------------------------------------------------------------------------------
// 16 bytes of T in registers as they lie in memory; converted to fp32 where they are used (half the registers for bf16)
template <class T> constexpr int VEC16 = 16 / (int)sizeof(T);
__device__ __forceinline__ void vec_get(float (&f)[4], const uint4& r) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void vec_get(float (&f)[8], const uint4& r) {
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[2 * j] = __uint_as_float(w[j] << 16);
        f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
}
__device__ __forceinline__ void vec_put(uint4& r, const float (&f)[4]) {
    r = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ void vec_put(uint4& r, const float (&f)[8]) {
    r = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
// Loads and stores of 16 bytes at any alignment of T (the memory system takes them, at a cost where they cross lines), or of the first
// nv elements of them: the end of a row
template <class T> __device__ __forceinline__ uint4 load16(const T* a, int nv) {
    uint4 t = make_uint4(0u, 0u, 0u, 0u);
    if (nv >= VEC16<T>) __builtin_memcpy(&t, a, 16);
    else {
        T tmp[VEC16<T>];
#pragma unroll
        for (int j = 0; j < VEC16<T>; ++j) tmp[j] = j < nv ? a[j] : (T)0;
        __builtin_memcpy(&t, tmp, 16);
    }
    return t;
}
template <class T> __device__ __forceinline__ void store16(T* a, const uint4& r, int nv) {
    if (nv >= VEC16<T>) __builtin_memcpy(a, &r, 16);
    else {
        T tmp[VEC16<T>];
        __builtin_memcpy(tmp, &r, 16);
#pragma unroll
        for (int j = 0; j < VEC16<T>; ++j) if (j < nv) a[j] = tmp[j];
    }
}

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
// N values into N / 4 words of bytes: x / step + 1.5 * 2^23 rounds x / step to the nearest even integer, which is then the low byte of the
// sum.  (The product is exact and |x / step| <= 128.)
template <int N> __device__ __forceinline__ void ck_bytes(unsigned (&w)[N / 4], float (&f)[N], unsigned code) {
    const float inv = __uint_as_float((254u - (code == 255u ? 127u : code)) << 23);
    if (code == 248u) {                                          // the largest step cannot grow: 127 steps at most
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = fminf(fmaxf(f[j], -0x1.fcp127f), 0x1.fcp127f);
    }
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
        unsigned b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(fmaf(f[4 * k + j], inv, 12582912.f));
        w[k] = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
        if (code == 255u) w[k] = 0u;
    }
}
// largest |x| of N values, as bits
template <int N> __device__ __forceinline__ unsigned ck_amax(const float (&f)[N]) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
    return m;
}
// host, ckpt8.hip: x [N][S][C] with any strides of a sample and of a position (N, S, C > 0, S < 2^31 for N > 1) -> q, e of N S rows
int ck_pack_samples(const void* x, long long xn, long long xs, long long N, long long S, int C, void* q, long long ldq, void* e, long long lde, int dtype,
                    hipStream_t st);
// value of byte j of w at step s: a conversion that selects and sign-extends its byte, and a product
__device__ __forceinline__ float ck_value(unsigned w, int j, float s) { return (float)(signed char)(w >> (8 * j)) * s; }
