// What the router's kernels share: a row of logits over the lanes of a wave, its loads, stores, sums and softmax, and the
// instance that serves a number of experts.
#pragma once
#include "exl3_kernels.h"
#include "exl3_epilogue.h"

#include <type_traits>

namespace exl3 {

// Butterflies over the L lanes of a row: DPP within 16 lanes, a shuffle for the steps of 16 and 32.
template <int L, class F>
__device__ __forceinline__ float group_join(float v, F f) {
    if constexpr (L > 1) v = f(v, xor_lane_row<1>(v));
    if constexpr (L > 2) v = f(v, xor_lane_row<2>(v));
    if constexpr (L > 4) v = f(v, xor_lane_row<4>(v));
    if constexpr (L > 8) v = f(v, xor_lane_row<8>(v));
    if constexpr (L > 16) v = f(v, __shfl_xor(v, 16));
    if constexpr (L > 32) v = f(v, __shfl_xor(v, 32));
    return v;
}
template <int L>
__device__ __forceinline__ float group_max(float v) {
    return group_join<L>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    return group_join<L>(v, [](float a, float b) { return a + b; });
}

// The lane's PER logits of a row as loaded: whole, aligned vectors of the type (VEC; the host checks), or f32 values.
template <int PER, int DT, bool VEC>
struct Logits {
    static constexpr int SIZE = DT == DT_F32 ? 4 : 2;
    static constexpr int W = VEC ? (PER * SIZE + 3) / 4 : PER;
    uint32_t w[W];
    // at: the row's first logit.  A lane past the row's end loads what is there (unpack drops it).
    __device__ __forceinline__ void load(const void *logits, size_t at, int experts, int e0) {
        if constexpr (VEC) {
            constexpr int BYTES = PER * SIZE;
            const char *p = static_cast<const char *>(logits) + (at + (e0 < experts ? e0 : 0)) * SIZE;
            if constexpr (BYTES >= 16) {
#pragma unroll
                for (int q = 0; q < BYTES / 16; q++) {
                    const uint4 u = reinterpret_cast<const uint4 *>(p)[q];
                    w[4 * q] = u.x, w[4 * q + 1] = u.y, w[4 * q + 2] = u.z, w[4 * q + 3] = u.w;
                }
            } else if constexpr (BYTES == 8) {
                const uint2 u = *reinterpret_cast<const uint2 *>(p);
                w[0] = u.x, w[1] = u.y;
            } else if constexpr (BYTES == 4) {
                w[0] = *reinterpret_cast<const uint32_t *>(p);
            } else {
                w[0] = *reinterpret_cast<const uint16_t *>(p);
            }
        } else {
#pragma unroll
            for (int q = 0; q < PER; q++)
                w[q] = __float_as_uint(load_act<DT>(logits, at + (size_t)min(e0 + q, experts - 1)));
        }
    }
    // As f32: -inf past the row's end, and zeros in place of a row that is not live (whatever it holds).
    __device__ __forceinline__ void unpack(int experts, int e0, bool live, float (&v)[PER]) const {
        constexpr uint32_t LOW = !VEC || DT == DT_F32 ? 0xFF800000u : DT == DT_F16 ? 0xFC00FC00u : 0xFF80FF80u;
        uint32_t u[W];
#pragma unroll
        for (int q = 0; q < W; q++) u[q] = live ? (e0 + (VEC ? 0 : q) < experts ? w[q] : LOW) : 0u;
#pragma unroll
        for (int q = 0; q < PER; q++) {
            if constexpr (!VEC || DT == DT_F32) v[q] = __uint_as_float(u[q]);
            else {
                const uint32_t h = q & 1 ? u[q >> 1] >> 16 : u[q >> 1] & 0xFFFFu;
                v[q] = DT == DT_F16 ? h2f((uint16_t)h) : __uint_as_float(h << 16);
            }
        }
    }
};

// Their counterpart: PER values of a row (at: its first), rounded to the logits' type; zeros for a row that is not live.
template <int PER, int DT, bool VEC>
__device__ __forceinline__ void store_logits(void *p, size_t at, int experts, int e0, bool live, const float (&v)[PER]) {
    if constexpr (VEC && PER * (DT == DT_F32 ? 4 : 2) >= 4) {
        if (e0 >= experts) return;
        constexpr int W = PER * (DT == DT_F32 ? 4 : 2) / 4;
        uint32_t w[W];
#pragma unroll
        for (int q = 0; q < W; q++) {
            if constexpr (DT == DT_F32) w[q] = __float_as_uint(v[q]);
            else if constexpr (DT == DT_F16)
                w[q] = __half_as_ushort(__float2half_rn(v[2 * q])) | (uint32_t)__half_as_ushort(__float2half_rn(v[2 * q + 1])) << 16;
            else
                w[q] = __bfloat16_as_ushort(__float2bfloat16(v[2 * q])) |
                       (uint32_t)__bfloat16_as_ushort(__float2bfloat16(v[2 * q + 1])) << 16;
            w[q] = live ? w[q] : 0u;
        }
        char *o = static_cast<char *>(p) + (at + e0) * (DT == DT_F32 ? 4 : 2);
        if constexpr (W >= 4) {
#pragma unroll
            for (int q = 0; q < W / 4; q++)
                reinterpret_cast<uint4 *>(o)[q] = uint4{w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
        } else if constexpr (W == 2) {
            *reinterpret_cast<uint2 *>(o) = uint2{w[0], w[1]};
        } else {
            *reinterpret_cast<uint32_t *>(o) = w[0];
        }
    } else {
#pragma unroll
        for (int q = 0; q < PER; q++)
            if (e0 + q < experts) store_act<DT>(p, at + e0 + q, live ? v[q] : 0.f);
    }
}

// v becomes exp(v - the row's largest); returns the lane's share of their sum.  A row of -inf alone leaves zeros; NaN stays.
// (The difference comes before the product with log2 e: with a row at the type's lowest value an fma's terms overflow.)
template <int L, int PER>
__device__ __forceinline__ float row_exp(float (&v)[PER]) {
    float mx = v[0];
#pragma unroll
    for (int q = 1; q < PER; q++) mx = fmaxf(mx, v[q]);
    mx = group_max<L>(mx);
    const float base = mx == -INFINITY ? 0.f : mx;
    float den = 0.f;
#pragma unroll
    for (int q = 0; q < PER; q++) {
        v[q] = __expf(v[q] - base);
        den += v[q];
    }
    return den;
}

// Orders a wave's LDS accesses across lanes: the hardware runs them in order, the compiler must too.
__device__ __forceinline__ void wave_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// The lanes a row takes and the experts a lane holds: 8 experts a lane (16) once the row fills 8 (64) lanes.
template <class F>
static hipError_t with_shape(int experts, F f) {
    if (experts <= 8) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    if (experts <= 16) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
    if (experts <= 32) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
    if (experts <= 64) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
    if (experts <= 128) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 8>{});
    if (experts <= 256) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
    if (experts <= 512) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
    if (experts <= 1024) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
    return hipErrorInvalidValue;
}

template <int PER, int DT>
static bool whole_vectors(const void *logits, int experts) {
    const int bytes = PER * (DT == DT_F32 ? 4 : 2), align = bytes > 16 ? 16 : bytes;
    return experts % PER == 0 && reinterpret_cast<uintptr_t>(logits) % align == 0;
}

template <class F>
static hipError_t with_dtype(int dt, F f) {
    if (dt == DT_F16) return f(std::integral_constant<int, DT_F16>{});
    if (dt == DT_BF16) return f(std::integral_constant<int, DT_BF16>{});
    return f(std::integral_constant<int, DT_F32>{});
}

}  // namespace exl3
