// Eight neighbouring values of an array at any alignment of its elements, as a vector load or store: global memory takes
// 16 bytes at any address, so rows of odd widths and operands that begin anywhere need no path of their own.  What passes
// the array's end goes by elements.
#pragma once
#include "exl3_kernels.h"

namespace exl3 {

using Words4 = uint32_t __attribute__((ext_vector_type(4)));
using Words4At2 = Words4 __attribute__((aligned(2)));
using Words4At4 = Words4 __attribute__((aligned(4)));

// Element c of an array at the wave's address p: a byte offset of 32 bits, so that the address stays in scalar registers.
template <int DT>
__device__ __forceinline__ const char *elem(const void *p, uint32_t c) {
    return static_cast<const char *>(p) + c * (DT == DT_F32 ? 4u : 2u);
}
template <int DT>
__device__ __forceinline__ char *elem(void *p, uint32_t c) {
    return static_cast<char *>(p) + c * (DT == DT_F32 ? 4u : 2u);
}

// Eight values as they lie in memory.
template <int DT>
struct Raw8 {
    static constexpr int W = DT == DT_F32 ? 8 : 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const char *at) {
        if constexpr (DT == DT_F32) {
            const Words4At4 *s = reinterpret_cast<const Words4At4 *>(at);
            const Words4 lo = s[0], hi = s[1];
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = lo[q], w[4 + q] = hi[q];
        } else {
            const Words4 u = *reinterpret_cast<const Words4At2 *>(at);
#pragma unroll
            for (int q = 0; q < 4; q++) w[q] = u[q];
        }
    }
    // The first n of them (0 for the rest), an element at a time.
    __device__ __forceinline__ void load_some(const char *at, int n) {
#pragma unroll
        for (int q = 0; q < W; q++) w[q] = 0;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if (q >= n) continue;
            if constexpr (DT == DT_F32) w[q] = reinterpret_cast<const uint32_t *>(at)[q];
            else w[q / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(at)[q] << (16 * (q & 1));
        }
    }
    // -inf in place of all but the first n.
    __device__ __forceinline__ void keep(int n) {
        constexpr uint32_t LOW = DT == DT_F32 ? 0xFF800000u : DT == DT_F16 ? 0xFC00u : 0xFF80u;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if constexpr (DT == DT_F32) w[q] = q < n ? w[q] : LOW;
            else if (q & 1) w[q / 2] = q < n ? w[q / 2] : (w[q / 2] & 0xFFFFu) | LOW << 16;
            else w[q / 2] = q < n ? w[q / 2] : (w[q / 2] & 0xFFFF0000u) | LOW;
        }
    }
    __device__ __forceinline__ float get(int q) const {
        if constexpr (DT == DT_F32) return __uint_as_float(w[q]);
        else if constexpr (DT == DT_F16) return h2f((uint16_t)(q & 1 ? w[q / 2] >> 16 : w[q / 2]));
        else return __uint_as_float(q & 1 ? w[q / 2] & 0xFFFF0000u : w[q / 2] << 16);
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int q = 0; q < W; q++) {
            if constexpr (DT == DT_F32) w[q] = __float_as_uint(v[q]);
            else if constexpr (DT == DT_F16)
                w[q] = __half_as_ushort(__float2half_rn(v[2 * q])) | (uint32_t)__half_as_ushort(__float2half_rn(v[2 * q + 1])) << 16;
            else
                w[q] = __bfloat16_as_ushort(__float2bfloat16(v[2 * q])) |
                       (uint32_t)__bfloat16_as_ushort(__float2bfloat16(v[2 * q + 1])) << 16;
        }
    }
    __device__ __forceinline__ void store(char *at) const {
        Words4 lo;
#pragma unroll
        for (int q = 0; q < 4; q++) lo[q] = w[q];
        if constexpr (DT == DT_F32) {
            Words4 hi;
#pragma unroll
            for (int q = 0; q < 4; q++) hi[q] = w[4 + q];
            Words4At4 *s = reinterpret_cast<Words4At4 *>(at);
            s[0] = lo;
            s[1] = hi;
        } else {
            *reinterpret_cast<Words4At2 *>(at) = lo;
        }
    }
};

// How many of the eight values from c on lie before `width`, counted where it is asked for: in a loop over rows the masks of
// a row's last vector would otherwise be kept in scalar registers that the loop needs.
__device__ __forceinline__ int left_of(uint32_t c, uint32_t width) {
    int n = max(0, (int)(width - c));
    asm volatile("" : "+v"(n));
    return n;
}

// Values c .. c + 7 of an array from p on; zeros from `width` on.  WHOLE: the width is a multiple of eight, so a vector lies
// inside or outside.
template <int DT, bool WHOLE>
__device__ __forceinline__ void load_raw(const void *p, uint32_t c, uint32_t width, Raw8<DT> &r) {
    if (WHOLE ? c < width : c + 8 <= width) r.load(elem<DT>(p, c));
    else r.load_some(elem<DT>(p, c), WHOLE ? 0 : left_of(c, width));
}
template <int DT, bool WHOLE = false>
__device__ __forceinline__ void load8(const void *p, uint32_t c, uint32_t width, float (&v)[8]) {
    Raw8<DT> r;
    load_raw<DT, WHOLE>(p, c, width, r);
#pragma unroll
    for (int q = 0; q < 8; q++) v[q] = r.get(q);
}
template <bool WHOLE = false>
__device__ __forceinline__ void load8_any(const void *p, int dt, uint32_t c, uint32_t width, float (&v)[8]) {
    if (dt == DT_F16) load8<DT_F16, WHOLE>(p, c, width, v);
    else if (dt == DT_BF16) load8<DT_BF16, WHOLE>(p, c, width, v);
    else load8<DT_F32, WHOLE>(p, c, width, v);
}

// Eight values of a type known to the wave alone, as they lie in memory: the conversions, which wait for the loads, come when
// they are asked for, and the loads need no branch by the type.
struct RawAny {
    Words4 lo, hi;
    template <bool WHOLE>
    __device__ __forceinline__ void load(const void *p, int dt, uint32_t c, uint32_t width) {
        const bool f32 = dt == DT_F32;
        const char *at = static_cast<const char *>(p) + c * (f32 ? 4u : 2u);
        lo = hi = Words4{0, 0, 0, 0};
        if (WHOLE ? c < width : c + 8 <= width) {
            lo = *reinterpret_cast<const Words4At2 *>(at);
            if (f32) hi = reinterpret_cast<const Words4At2 *>(at)[1];
        } else if (!WHOLE) {
            const int n = left_of(c, width);
#pragma unroll
            for (int q = 0; q < 8; q++) {
                if (q >= n) continue;
                if (!f32) lo[q / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(at)[q] << (16 * (q & 1));
                else if (q < 4) lo[q & 3] = reinterpret_cast<const uint32_t *>(at)[q];
                else hi[q & 3] = reinterpret_cast<const uint32_t *>(at)[q];
            }
        }
    }
    // Plus `add`.
    __device__ __forceinline__ void get(int dt, float add, float (&v)[8]) const {
        if (dt == DT_F32) {
#pragma unroll
            for (int q = 0; q < 8; q++) v[q] = __uint_as_float(q < 4 ? lo[q & 3] : hi[q & 3]) + add;
        } else if (dt == DT_F16) {
#pragma unroll
            for (int q = 0; q < 8; q++) v[q] = h2f((uint16_t)(q & 1 ? lo[q / 2] >> 16 : lo[q / 2])) + add;
        } else {
#pragma unroll
            for (int q = 0; q < 8; q++) v[q] = __uint_as_float(q & 1 ? lo[q / 2] & 0xFFFF0000u : lo[q / 2] << 16) + add;
        }
    }
};

template <int DT, bool WHOLE = false>
__device__ __forceinline__ void store8(void *p, uint32_t c, uint32_t width, const float (&v)[8]) {
    if (WHOLE ? c < width : c + 8 <= width) {
        Raw8<DT> r;
        r.set(v);
        r.store(elem<DT>(p, c));
    } else if (!WHOLE) {
        const int n = left_of(c, width);
#pragma unroll
        for (int q = 0; q < 8; q++)
            if (q < n) store_act<DT>(elem<DT>(p, c), q, v[q]);
    }
}

}  // namespace exl3
