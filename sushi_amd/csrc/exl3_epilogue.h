// The epilogue of a linear, y = T(act(z) + residual) with z = project(x) + bias, and the activations' slopes for its
// backward pass.  Everything is f32 up to the one rounding to y's dtype (pre, the kept z, is rounded to it as well: the
// backward pass reads it at the width of the other activations).
#pragma once
#include "exl3_kernels.h"

namespace exl3 {

// The activations run on the hardware's exp2 and reciprocal (an ulp each).  A row block's epilogue holds no other work, so
// their instructions are its time: 200 rows of 2560 x 16384, finished in the tile, take 48.3 us without an activation, 49.4
// with silu, 50.4 with gelu_tanh, 52.7 with gelu (67 with the library's erfc and f32 divisions); 2048 rows of 4096 x 14336
// 230.4, 237.3, 240.0 and 245.9.
// gelu's normal CDF: its lower tail is Phi(-x) = t P(t) exp(-x^2 / 2) for x >= 0 with t = 1 / (1 + 0.21 x), P the polynomial of
// degree 8 with the least relative error (1.9e-8) up to x = 14.5, past which an f32 exp vanishes.  So the tail keeps its
// relative precision: within 5e-7 from -1 on, 1.5e-6 down to -5, 8e-6 at -12, there the exp's argument's rounding.  The exp
// is also the density of the slope.
__device__ __forceinline__ float rcp(float x) { return __builtin_amdgcn_rcpf(x); }
constexpr float GELU_A = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float GELU_B = 0.044715f;
constexpr float INV_SQRT_2PI = 0.3989422804014327f;

// Phi(z), and exp(-z^2 / 2) in `ex`.
__device__ __forceinline__ float normal_cdf(float z, float &ex) {
    const float t = rcp(1.f + 0.21f * fabsf(z));
    float poly = -0.0712944642f;
    poly = poly * t + 0.281802952f;
    poly = poly * t - 0.326489985f;
    poly = poly * t + 0.344983011f;
    poly = poly * t - 0.0907701403f;
    poly = poly * t + 0.123471074f;
    poly = poly * t + 0.0695700124f;
    poly = poly * t + 0.0850124061f;
    poly = poly * t + 0.0837151557f;
    ex = __builtin_amdgcn_exp2f(z * z * -0.72134752f);  // -log2(e) / 2
    const float q = poly * t * ex;
    return z >= 0.f ? 1.f - q : q;
}

__device__ __forceinline__ float act_value(int act, float z) {
    if (act == ACT_NONE) return z;
    if (act == ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
    if (act == ACT_GELU) {
        float ex;
        return z * normal_cdf(z, ex);
    }
    // silu and gelu_tanh are z times a logistic, which keeps the small values' relative precision
    const float u = act == ACT_SILU ? z : z * (2.f * GELU_A + (2.f * GELU_A * GELU_B) * z * z);
    return z * rcp(1.f + __expf(-u));
}

// act'(z).  Past |z| = 100 every slope is its limit to the last bit of an f32, and is taken as that: the formulas' products of
// an overflowed and a vanished factor (inf * 0) are formed there and dropped.  NaN fails the comparisons and stays NaN.
__device__ __forceinline__ float act_slope(int act, float z) {
    if (act == ACT_NONE) return 1.f;
    if (act == ACT_RELU) return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
    float s;
    if (act == ACT_GELU) {
        float ex;
        const float cdf = normal_cdf(z, ex);
        s = cdf + z * INV_SQRT_2PI * ex;
    } else {  // z g(u): g + z u' g (1 - g), with g and 1 - g from one exp of -|u|
        const float zz = z * z;
        const float u = act == ACT_SILU ? z : z * (2.f * GELU_A + (2.f * GELU_A * GELU_B) * zz);
        const float du = act == ACT_SILU ? 1.f : 2.f * GELU_A + (6.f * GELU_A * GELU_B) * zz;
        const float e = __expf(-fabsf(u)), r = rcp(1.f + e);
        s = (u >= 0.f ? r : e * r) + z * du * (e * r * r);
    }
    return z > 100.f ? 1.f : z < -100.f ? 0.f : s;
}

// The aligned 32-bit word that holds element i of an f16 / bf16 / f32 array (4-byte aligned, whole words), and the
// element from it, both without a branch on the dtype: words are fetched early and unpacked where they are used, so no
// wait sits between.
__device__ __forceinline__ uint32_t act_word(const void *p, int dt, size_t i) {
    const size_t byte = dt == DT_F32 ? i * 4 : i * 2;
    typedef __attribute__((address_space(1))) const uint32_t global_u32;
    return *(global_u32 *)(static_cast<const char *>(p) + (byte & ~(size_t)3));
}
__device__ __forceinline__ float act_from_word(uint32_t w, int dt, size_t i) {
    const uint32_t h = (w >> ((uint32_t)(i & 1) * 16u)) & 0xFFFFu;
    const float f16v = h2f((uint16_t)h), bf16v = __uint_as_float(h << 16);
    return dt == DT_F32 ? __uint_as_float(w) : dt == DT_F16 ? f16v : bf16v;
}

// Element i of an f16 / bf16 / f32 array.
__device__ __forceinline__ void store_any(void *p, int dt, size_t i, float v) {
    if (dt == DT_F16) store_act<DT_F16>(p, i, v);
    else if (dt == DT_BF16) store_act<DT_BF16>(p, i, v);
    else store_act<DT_F32>(p, i, v);
}

// One lane's bias and residual words of outputs (row-major element) i0 and i0 + 64, columns c0 and c0 + 64, fetched ahead
// of the sums they join; absent ones are not read.
struct EpilogueWords {
    uint32_t b0, b1, r0, r1;
};
__device__ __forceinline__ EpilogueWords epilogue_fetch(const EpilogueArgs &e, int y_dtype, size_t c0, size_t i0) {
    EpilogueWords w{};
    if (e.bias) {
        w.b0 = act_word(e.bias, e.bias_dtype, c0);
        w.b1 = act_word(e.bias, e.bias_dtype, c0 + 64);
    }
    if (e.residual) {
        w.r0 = act_word(e.residual, y_dtype, i0);
        w.r1 = act_word(e.residual, y_dtype, i0 + 64);
    }
    return w;
}
// act(z) + residual of one output from its words, with z stored to pre where it is kept.
__device__ __forceinline__ float epilogue_apply(const EpilogueArgs &e, int y_dtype, float v, uint32_t bw, size_t c,
                                                uint32_t rw, size_t i) {
    const float z = v + (e.bias ? act_from_word(bw, e.bias_dtype, c) : 0.f);
    if (e.pre) store_any(e.pre, y_dtype, i, z);
    return act_value(e.act, z) + (e.residual ? act_from_word(rw, y_dtype, i) : 0.f);
}

// y = act(z) of eight values, the activation chosen once for all of them (so their instructions interleave).
__device__ __forceinline__ void act_eight(int act, const float (&z)[8], float (&y)[8]) {
#define EXL3_ACT_EIGHT(A)                                                                                              \
    case A:                                                                                                            \
        _Pragma("unroll") for (int j = 0; j < 8; j++) y[j] = act_value(A, z[j]);                                       \
        break;
    switch (act) {
        EXL3_ACT_EIGHT(ACT_RELU)
        EXL3_ACT_EIGHT(ACT_SILU)
        EXL3_ACT_EIGHT(ACT_GELU)
        EXL3_ACT_EIGHT(ACT_GELU_TANH)
    default:
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = z[j];
    }
#undef EXL3_ACT_EIGHT
}

// d *= act'(z) of N values, likewise.
template <int N>
__device__ __forceinline__ void act_slopes(int act, const float (&z)[N], float (&d)[N]) {
#define EXL3_ACT_SLOPES(A)                                                                                             \
    case A:                                                                                                            \
        _Pragma("unroll") for (int j = 0; j < N; j++) d[j] *= act_slope(A, z[j]);                                      \
        break;
    switch (act) {
        EXL3_ACT_SLOPES(ACT_RELU)
        EXL3_ACT_SLOPES(ACT_SILU)
        EXL3_ACT_SLOPES(ACT_GELU)
        EXL3_ACT_SLOPES(ACT_GELU_TANH)
    default: break;
    }
#undef EXL3_ACT_SLOPES
}

// Two f32 values rounded to f16 or bf16 (gfx950 converts to both to nearest even).
__device__ __forceinline__ uint32_t pack2(bool bf16, float x, float y) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
    typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
    return bf16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{x, y}), bf2_t))
                : __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{x, y}), h2_t));
}

// Eight of them.
__device__ __forceinline__ uint4 pack8(bool bf16, const float (&v)[8]) {
    return uint4{pack2(bf16, v[0], v[1]), pack2(bf16, v[2], v[3]), pack2(bf16, v[4], v[5]), pack2(bf16, v[6], v[7])};
}

}  // namespace exl3
