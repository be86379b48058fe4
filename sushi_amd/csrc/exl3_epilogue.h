// The epilogue of a linear, y = T(act(z) + residual) with z = project(x) + bias, and the activations' slopes for its
// backward pass.  Everything is f32 up to the one rounding to y's dtype (pre, the kept z, is rounded to it as well: the
// backward pass reads it at the width of the other activations).
#pragma once
#include "exl3_kernels.h"

namespace exl3 {

// act(z).  silu and gelu_tanh are z times a logistic, and gelu's normal CDF is an erfc, so the small values left of zero
// keep their relative precision (1 + tanh and 1 + erf would cancel there).
__device__ __forceinline__ float logistic(float t) { return 1.f / (1.f + __expf(-t)); }
constexpr float GELU_A = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float GELU_B = 0.044715f;
constexpr float SQRT_HALF = 0.7071067811865476f;
constexpr float INV_SQRT_2PI = 0.3989422804014327f;

__device__ __forceinline__ float act_value(int act, float z) {
    switch (act) {
    case ACT_RELU: return z < 0.f ? 0.f : z;  // NaN stays NaN
    case ACT_SILU: return z * logistic(z);
    case ACT_GELU: return z * (0.5f * erfcf(-z * SQRT_HALF));
    case ACT_GELU_TANH: return z * logistic(2.f * GELU_A * (z + GELU_B * z * z * z));
    default: return z;
    }
}

// act'(z).  Past |z| = 100 every slope is its limit to the last bit of an f32, and the formulas' products of an overflowed
// and a vanished factor are never formed; NaN fails the comparison and stays NaN.
__device__ __forceinline__ float act_slope(int act, float z) {
    if (act == ACT_NONE) return 1.f;
    if (act == ACT_RELU) return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;
    if (fabsf(z) > 100.f) return z > 0.f ? 1.f : 0.f;
    if (act == ACT_SILU) {
        const float s = logistic(z);
        return s + z * s * logistic(-z);
    }
    if (act == ACT_GELU) return 0.5f * erfcf(-z * SQRT_HALF) + z * INV_SQRT_2PI * __expf(-0.5f * z * z);
    const float t = 2.f * GELU_A * (z + GELU_B * z * z * z);
    const float g = logistic(t);
    return g + z * g * logistic(-t) * (2.f * GELU_A) * (1.f + 3.f * GELU_B * z * z);
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
// of the sums they join.  An absent bias / residual is read from a stand-in the host supplies and dropped.
struct EpilogueWords {
    uint32_t b0, b1, r0, r1;
};
__device__ __forceinline__ EpilogueWords epilogue_fetch(const EpilogueArgs &e, int y_dtype, size_t c0, size_t i0) {
    return EpilogueWords{act_word(e.bias, e.bias_dtype, c0), act_word(e.bias, e.bias_dtype, c0 + 64),
                         act_word(e.residual, y_dtype, i0), act_word(e.residual, y_dtype, i0 + 64)};
}
// act(z) + residual of one output from its words, with z stored to pre where it is kept.
__device__ __forceinline__ float epilogue_apply(const EpilogueArgs &e, int y_dtype, float v, uint32_t bw, size_t c,
                                                uint32_t rw, size_t i) {
    const float z = v + (e.has_bias ? act_from_word(bw, e.bias_dtype, c) : 0.f);
    if (e.pre) store_any(e.pre, y_dtype, i, z);
    return act_value(e.act, z) + (e.has_residual ? act_from_word(rw, y_dtype, i) : 0.f);
}

}  // namespace exl3
