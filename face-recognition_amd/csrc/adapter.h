// Element types, raw vector access and activations shared by the adapter kernels (k_linear, k_norm, k_route).
#pragma once
#include "kernels.h"

typedef _Float16 f16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

static inline bool type_ok(int t) { return t == FR_TYPE_F32 || t == FR_TYPE_BF16 || t == FR_TYPE_F16; }
static inline int type_bytes(int t) { return t == FR_TYPE_F32 ? 4 : 2; }

// Vectors at an element's own alignment: gfx950 global loads and stores of 4..16 bytes take any address.
typedef u32x4 __attribute__((aligned(2), may_alias)) u32x4_any;
typedef u32x2 __attribute__((aligned(2), may_alias)) u32x2_any;

// Eight consecutive elements as they lie in memory (fp32: 32 bytes, 16-bit types: 16 bytes in `a`).
struct Raw8 { u32x4 a, b; };

template <bool ALIGNED>
FR_DEV Raw8 raw_load8(const void* base, long i, int type) {
    Raw8 r;
    if (type == FR_TYPE_F32) {
        const float* p = reinterpret_cast<const float*>(base) + i;
        if constexpr (ALIGNED) { r.a = reinterpret_cast<const u32x4*>(p)[0]; r.b = reinterpret_cast<const u32x4*>(p)[1]; }
        else { r.a = reinterpret_cast<const u32x4_any*>(p)[0]; r.b = reinterpret_cast<const u32x4_any*>(p + 4)[0]; }
    } else {
        const unsigned short* p = reinterpret_cast<const unsigned short*>(base) + i;
        if constexpr (ALIGNED) r.a = *reinterpret_cast<const u32x4*>(p);
        else r.a = *reinterpret_cast<const u32x4_any*>(p);
        r.b = u32x4{0, 0, 0, 0};
    }
    return r;
}
FR_DEV float f16bits_to_f(unsigned short v) { return (float)__builtin_bit_cast(f16, v); }
FR_DEV Vec8f raw_to_f(const Raw8& r, int type) {
    Vec8f o;
    if (type == FR_TYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { o.v[i] = __uint_as_float(r.a[i]); o.v[4 + i] = __uint_as_float(r.b[i]); }
    } else if (type == FR_TYPE_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { o.v[2 * i] = __uint_as_float(r.a[i] << 16); o.v[2 * i + 1] = __uint_as_float(r.a[i] & 0xFFFF0000u); }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { o.v[2 * i] = f16bits_to_f((unsigned short)r.a[i]); o.v[2 * i + 1] = f16bits_to_f((unsigned short)(r.a[i] >> 16)); }
    }
    return o;
}
FR_DEV float load1(const void* base, long i, int type) {
    if (type == FR_TYPE_F32) return reinterpret_cast<const float*>(base)[i];
    const unsigned short v = reinterpret_cast<const unsigned short*>(base)[i];
    return type == FR_TYPE_BF16 ? bfbits_to_f(v) : f16bits_to_f(v);
}
FR_DEV unsigned pack2(float lo, float hi, int type) {
    if (type == FR_TYPE_BF16) return pack2bf(lo, hi);
    return (unsigned)__builtin_bit_cast(unsigned short, (f16)lo) | ((unsigned)__builtin_bit_cast(unsigned short, (f16)hi) << 16);
}
FR_DEV void store1(void* base, long i, int type, float v) {
    if (type == FR_TYPE_F32) reinterpret_cast<float*>(base)[i] = v;
    else reinterpret_cast<unsigned short*>(base)[i] = (unsigned short)pack2(v, 0.f, type);
}
template <bool ALIGNED>
FR_DEV void store8t(void* base, long i, int type, const Vec8f& x) {
    if (type == FR_TYPE_F32) {
        float* p = reinterpret_cast<float*>(base) + i;
        u32x4 a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) { a[j] = __float_as_uint(x.v[j]); b[j] = __float_as_uint(x.v[4 + j]); }
        if constexpr (ALIGNED) { reinterpret_cast<u32x4*>(p)[0] = a; reinterpret_cast<u32x4*>(p)[1] = b; }
        else { reinterpret_cast<u32x4_any*>(p)[0] = a; reinterpret_cast<u32x4_any*>(p + 4)[0] = b; }
    } else {
        unsigned short* p = reinterpret_cast<unsigned short*>(base) + i;
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = pack2(x.v[2 * j], x.v[2 * j + 1], type);
        if constexpr (ALIGNED) *reinterpret_cast<u32x4*>(p) = a;
        else *reinterpret_cast<u32x4_any*>(p) = a;
    }
}

// LDS written by other lanes of this wave is read behind it (a wave's LDS accesses are carried out in order).
FR_DEV void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// Sums over the lanes up to each lane.
FR_DEV int scan_add(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);          // 1, 2, 4 and 8 lanes back in a row of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);          // the row before; the two rows before
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// act(v) of the adapter products.  GELU is the erf form v Phi(v), SiLU v sigmoid(v).
// exp2 and reciprocal are the hardware's (1 ulp).  Phi(-a) = erfc(a / sqrt 2) / 2 = t P(t) exp(-a^2 / 2) with
// t = 1 / (1 + 0.3 a / sqrt 2): P is a minimax fit of erfcx(z) / t over t in (0.23, 1], 2.0e-8 relative, so small values of
// either tail keep their digits.  SiLU is 0 below -88.7, where e^-v leaves fp32's range and |v sigmoid(v)| < 2.7e-37: the
// epilogue of a wide product is bound by its vector instructions, and a form that keeps those values costs five more.
FR_DEV float gelu(float v) {
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(v), 0.3f * 0.70710678118654752f, 1.f));
    float p = -0.12955585f;
    p = fmaf(p, t, 0.48573610f);
    p = fmaf(p, t, -0.51266706f);
    p = fmaf(p, t, 0.54820925f);
    p = fmaf(p, t, -0.095026374f);
    p = fmaf(p, t, 0.21510610f);
    p = fmaf(p, t, 0.14828666f);
    p = fmaf(p, t, 0.17072374f);
    p = fmaf(p, t, 0.16918743f);
    const float tail = 0.5f * (t * p) * __builtin_amdgcn_exp2f((v * v) * -0.72134752044448170f);
    return v * (v < 0.f ? tail : 1.f - tail);
}
FR_DEV float silu(float v) { return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f)); }
FR_DEV float adapter_act(float v, int act, float slope) {
    switch (act) {
        case FR_ACT_PRELU: return v >= 0.f ? v : v * slope;
        case FR_ACT_HSWISH: return v * __builtin_amdgcn_fmed3f(fmaf(v, 1.f / 6.f, 0.5f), 0.f, 1.f);
        case FR_ACT_RELU: return v < 0.f ? 0.f : v;
        case FR_ACT_HSIGMOID: return v != v ? v : __builtin_amdgcn_fmed3f(fmaf(v, 1.f / 6.f, 0.5f), 0.f, 1.f);
        case FR_ACT_GELU: return gelu(v);
        case FR_ACT_SILU: return silu(v);
        default: return v;
    }
}
