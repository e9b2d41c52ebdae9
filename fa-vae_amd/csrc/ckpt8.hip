// Activation checkpoints in 8 bits: pack and unpack.
//
// q [R][C] int8 and one code byte per 32 channels of a row; the format is defined in act8.h.  Both directions are one pass over the
// data and bound by memory: pack reads 2 or 4 bytes a value and writes 33/32, unpack the reverse.
#include "act8.h"

namespace {

struct CkP {
    const void* x; long long ldx;
    unsigned char* q; long long ldq;
    unsigned char* e; long long lde;
    void* out; long long ldo;
    long long R; int C, nb;              // nb = blocks of 32 channels in a row
    long long items;
};

// Wide form: one lane takes 8 channels, 4 neighbouring lanes a block (C a multiple of 8, rows 16-byte aligned; lanes of a row's last
// block that lie past C are idle).  U items a thread, all loads issued before the first use.
template <class T, int U> __global__ __launch_bounds__(256) void ck_pack_wide(const CkP p) {
    const int per_row = p.nb * 4;
    const long long base = (long long)blockIdx.x * (256 * U);
    const long long row0 = base / per_row;
    const int off0 = (int)(base - row0 * per_row);
    float f[U][8];
    long long row[U]; int c[U]; bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned t = (unsigned)(off0 + u * 256) + threadIdx.x;
        const unsigned dr = t / (unsigned)per_row;
        row[u] = row0 + dr;
        c[u] = (int)(t - dr * (unsigned)per_row) * 8;
        ok[u] = row[u] < p.R && c[u] < p.C;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[u][j] = 0.f;
        if (ok[u]) {
            const T* s = (const T*)p.x + row[u] * p.ldx + c[u];
            if constexpr (sizeof(T) == 2) vec_get(f[u], *(const uint4*)s);
            else {
                float lo[4], hi[4];
                vec_get(lo, *(const float4*)s);
                vec_get(hi, *(const float4*)(s + 4));
#pragma unroll
                for (int j = 0; j < 4; ++j) { f[u][j] = lo[j]; f[u][4 + j] = hi[j]; }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[u][j]) & 0x7fffffffu);
        m = max(m, (unsigned)__shfl_xor((int)m, 1, 64));
        m = max(m, (unsigned)__shfl_xor((int)m, 2, 64));
        const unsigned code = ck_code(m);
        unsigned w[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2] |= ((unsigned)ck_round(f[u][j], code) & 0xffu) << (8 * (j & 3));
        if (ok[u]) {
            *(uint2*)(p.q + row[u] * p.ldq + c[u]) = make_uint2(w[0], w[1]);
            if ((c[u] & 31) == 0) p.e[row[u] * p.lde + (c[u] >> 5)] = (unsigned char)code;
        }
    }
}

// Any width, stride and alignment: half a wave takes a block, one channel a lane
template <class T, int U> __global__ __launch_bounds__(256) void ck_pack_any(const CkP p) {
    const int lane = threadIdx.x & 31;
    const long long b0 = (long long)blockIdx.x * (8 * U) + (threadIdx.x >> 5);
    float f[U];
    long long row[U]; int c[U]; bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long b = b0 + 8 * u;
        row[u] = b / p.nb;
        c[u] = (int)(b - row[u] * p.nb) * 32 + lane;
        ok[u] = row[u] < p.R && c[u] < p.C;
        f[u] = ok[u] ? to_f32<T>(((const T*)p.x)[row[u] * p.ldx + c[u]]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        unsigned m = __float_as_uint(f[u]) & 0x7fffffffu;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
        const unsigned code = ck_code(m);
        if (ok[u]) {
            p.q[row[u] * p.ldq + c[u]] = (unsigned char)ck_round(f[u], code);
            if (lane == 0) p.e[row[u] * p.lde + (c[u] >> 5)] = (unsigned char)code;
        }
    }
}

template <class T, int U> __global__ __launch_bounds__(256) void ck_unpack_wide(const CkP p) {
    const int per_row = p.nb * 4;
    const long long base = (long long)blockIdx.x * (256 * U);
    const long long row0 = base / per_row;
    const int off0 = (int)(base - row0 * per_row);
    uint2 w[U]; unsigned code[U];
    long long row[U]; int c[U]; bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned t = (unsigned)(off0 + u * 256) + threadIdx.x;
        const unsigned dr = t / (unsigned)per_row;
        row[u] = row0 + dr;
        c[u] = (int)(t - dr * (unsigned)per_row) * 8;
        ok[u] = row[u] < p.R && c[u] < p.C;
        w[u] = make_uint2(0u, 0u);
        code[u] = 0u;
        if (ok[u]) {
            w[u] = *(const uint2*)(p.q + row[u] * p.ldq + c[u]);
            code[u] = p.e[row[u] * p.lde + (c[u] >> 5)];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!ok[u]) continue;
        const float s = ck_scale(code[u]);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = ck_value(j < 4 ? w[u].x : w[u].y, j & 3, s);
        T* o = (T*)p.out + row[u] * p.ldo + c[u];
        if constexpr (sizeof(T) == 2) { uint4 r; vec_put(r, f); *(uint4*)o = r; }
        else { *(float4*)o = make_float4(f[0], f[1], f[2], f[3]); *(float4*)(o + 4) = make_float4(f[4], f[5], f[6], f[7]); }
    }
}

template <class T, int U> __global__ __launch_bounds__(256) void ck_unpack_any(const CkP p) {
    const int lane = threadIdx.x & 31;
    const long long b0 = (long long)blockIdx.x * (8 * U) + (threadIdx.x >> 5);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long b = b0 + 8 * u;
        const long long row = b / p.nb;
        const int c = (int)(b - row * p.nb) * 32 + lane;
        if (row < p.R && c < p.C)
            ((T*)p.out)[row * p.ldo + c] = from_f32<T>((float)(signed char)p.q[row * p.ldq + c] * ck_scale(p.e[row * p.lde + (c >> 5)]));
    }
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

constexpr int U_WIDE = 4, U_ANY = 4;
// a launch has at most 2^31 - 1 blocks
template <class F> int launch_ck(long long blocks, const char* who, F&& f) {
    FAVAE_CHECK_ARG(blocks <= 0x7fffffffLL, "%s: too many rows for one launch", who);
    if (blocks > 0) f((unsigned)blocks);
    FAVAE_LAUNCH_CHECK();
    return FAVAE_OK;
}

}  // namespace

extern "C" int favae_ckpt8_pack(const void* x, long long ldx, long long R, int C, void* q, long long ldq, void* e, long long lde, int dtype,
                                void* stream) {
    FAVAE_CHECK_ARG(R >= 0 && C >= 0 && (dtype == FAVAE_F32 || dtype == FAVAE_BF16), "favae_ckpt8_pack: bad sizes or dtype");
    if (R == 0 || C == 0) return FAVAE_OK;
    const int nb = cdiv(C, CK_BLOCK);
    FAVAE_CHECK_ARG(x && q && e && ldx >= C && ldq >= C && lde >= nb, "favae_ckpt8_pack: null pointer or a row stride below the row's length");
    FAVAE_CHECK_ARG(C <= (1 << 28), "favae_ckpt8_pack: more than 2^28 channels");
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    FAVAE_CHECK_ARG(aligned(x, es), "favae_ckpt8_pack: x is not aligned to its type");
    CkP p = {x, ldx, (unsigned char*)q, ldq, (unsigned char*)e, lde, nullptr, 0, R, C, nb, 0};
    const hipStream_t st = (hipStream_t)stream;
    const bool wide = C % 8 == 0 && aligned(x, 16) && (ldx * es) % 16 == 0 && aligned(q, 8) && ldq % 8 == 0;
    if (wide)
        return launch_ck(cdivll(R * nb * 4, 256 * U_WIDE), "favae_ckpt8_pack", [&](unsigned g) {
            if (dtype == FAVAE_F32) ck_pack_wide<float, U_WIDE><<<g, 256, 0, st>>>(p);
            else ck_pack_wide<bf16_t, U_WIDE><<<g, 256, 0, st>>>(p);
        });
    return launch_ck(cdivll(R * nb, 8 * U_ANY), "favae_ckpt8_pack", [&](unsigned g) {
        if (dtype == FAVAE_F32) ck_pack_any<float, U_ANY><<<g, 256, 0, st>>>(p);
        else ck_pack_any<bf16_t, U_ANY><<<g, 256, 0, st>>>(p);
    });
}

extern "C" int favae_ckpt8_unpack(const void* q, long long ldq, const void* e, long long lde, long long R, int C, void* out, long long ldo,
                                  int dtype, void* stream) {
    FAVAE_CHECK_ARG(R >= 0 && C >= 0 && (dtype == FAVAE_F32 || dtype == FAVAE_BF16), "favae_ckpt8_unpack: bad sizes or dtype");
    if (R == 0 || C == 0) return FAVAE_OK;
    const int nb = cdiv(C, CK_BLOCK);
    FAVAE_CHECK_ARG(out && q && e && ldo >= C && ldq >= C && lde >= nb, "favae_ckpt8_unpack: null pointer or a row stride below the row's length");
    FAVAE_CHECK_ARG(C <= (1 << 28), "favae_ckpt8_unpack: more than 2^28 channels");
    const int es = dtype == FAVAE_F32 ? 4 : 2;
    FAVAE_CHECK_ARG(aligned(out, es), "favae_ckpt8_unpack: out is not aligned to its type");
    CkP p = {nullptr, 0, (unsigned char*)q, ldq, (unsigned char*)e, lde, out, ldo, R, C, nb, 0};
    const hipStream_t st = (hipStream_t)stream;
    const bool wide = C % 8 == 0 && aligned(out, 16) && (ldo * es) % 16 == 0 && aligned(q, 8) && ldq % 8 == 0;
    if (wide)
        return launch_ck(cdivll(R * nb * 4, 256 * U_WIDE), "favae_ckpt8_unpack", [&](unsigned g) {
            if (dtype == FAVAE_F32) ck_unpack_wide<float, U_WIDE><<<g, 256, 0, st>>>(p);
            else ck_unpack_wide<bf16_t, U_WIDE><<<g, 256, 0, st>>>(p);
        });
    return launch_ck(cdivll(R * nb, 8 * U_ANY), "favae_ckpt8_unpack", [&](unsigned g) {
        if (dtype == FAVAE_F32) ck_unpack_any<float, U_ANY><<<g, 256, 0, st>>>(p);
        else ck_unpack_any<bf16_t, U_ANY><<<g, 256, 0, st>>>(p);
    });
}
