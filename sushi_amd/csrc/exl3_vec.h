// Eight neighbouring values of an array at any alignment of its elements, as a vector load or store: global memory takes
// 16 bytes at any address, so rows of odd widths and operands that begin anywhere need no path of their own.  What passes
// the array's end goes by elements, or as the last eight values before it.
#pragma once
#include "exl3_kernels.h"

namespace exl3 {

using Words4 = uint32_t __attribute__((ext_vector_type(4)));
using Words4At2 = Words4 __attribute__((aligned(2)));
using WordAt2 = uint32_t __attribute__((aligned(2)));
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
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int q = 0; q < W; q++) w[q] = 0;
    }
    // An array's n < 8 values as the last n.
    __device__ __forceinline__ void load_last(const void *p, int n) {
        clear();
#pragma unroll
        for (int q = 1; q < 8; q++) {
            if (q + n < 8) continue;
            if constexpr (DT == DT_F32) w[q] = static_cast<const uint32_t *>(p)[q + n - 8];
            else w[q / 2] |= (uint32_t)static_cast<const uint16_t *>(p)[q + n - 8] << (16 * (q & 1));
        }
    }
    // Zero in place of the first n.
    __device__ __forceinline__ void drop(int n) {
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if constexpr (DT == DT_F32) w[q] = q < n ? 0u : w[q];
            else w[q / 2] = q < n ? w[q / 2] & (q & 1 ? 0u : 0xFFFF0000u) : w[q / 2];
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

// A number counted where it is asked for: in a loop over rows the masks of a row's last vector would otherwise be kept in scalar
// registers that the loop needs.
__device__ __forceinline__ int opaque(int n) {
    asm volatile("" : "+v"(n));
    return n;
}

// A thread's eight values of a row, from column c on.  A row whose width is no multiple of eight ends inside a vector: that
// thread takes the row's last eight values instead and leaves out the first `skip`, which are another's: one vector load as
// everywhere, where elements one by one would each wait for the one before (gradient of 4096 rows of 3079 bf16 values with a
// channel gate: 83 us by elements, 58 so; 53 and, at 3080, 37 with the workgroups there are now).  Past the row's end all eight
// are left out.  WHOLE: the width is a multiple of eight, so a vector lies inside or outside.
struct Place {
    int c, skip;
};
template <bool WHOLE>
__device__ __forceinline__ Place place_of(uint32_t c, uint32_t width) {
    if (WHOLE) return {(int)c, c < width ? 0 : 8};
    const int at = opaque(min((int)c, (int)width - 8));
    return {at, min(8, (int)c - at)};
}

// The values as they lie in memory, those to be left out among them (a row of fewer than eight: its elements).
template <int DT, bool WHOLE>
__device__ __forceinline__ void load_raw(const void *p, uint32_t c, uint32_t width, Raw8<DT> &r) {
    if (WHOLE) {
        if (c < width) r.load(elem<DT>(p, c));
        else r.clear();
    } else if (width >= 8) {
        r.load(elem<DT>(p, (uint32_t)place_of<WHOLE>(c, width).c));
    } else {
        r.load_last(p, opaque((int)width));
    }
}
// Zeros in place of those to be left out.
template <int DT, bool WHOLE>
__device__ __forceinline__ void settle(uint32_t c, uint32_t width, Raw8<DT> &r) {
    if (WHOLE) return;
    const int skip = place_of<WHOLE>(c, width).skip;
    if (skip > 0) r.drop(opaque(skip));
}
template <int DT, bool WHOLE>
__device__ __forceinline__ void load8(const void *p, uint32_t c, uint32_t width, float (&v)[8]) {
    Raw8<DT> r;
    load_raw<DT, WHOLE>(p, c, width, r);
    settle<DT, WHOLE>(c, width, r);
#pragma unroll
    for (int q = 0; q < 8; q++) v[q] = r.get(q);
}
template <bool WHOLE>
__device__ __forceinline__ void load8_any(const void *p, int dt, uint32_t c, uint32_t width, float (&v)[8]) {
    if (dt == DT_F16) load8<DT_F16, WHOLE>(p, c, width, v);
    else if (dt == DT_BF16) load8<DT_BF16, WHOLE>(p, c, width, v);
    else load8<DT_F32, WHOLE>(p, c, width, v);
}

// Eight values of a type known to the wave alone, as they lie in memory: the conversions, which wait for the loads, come when
// they are asked for, and the loads need no branch by the type.
struct RawAny {
    Words4 lo, hi;
    // As load_raw and settle.
    template <bool WHOLE>
    __device__ __forceinline__ void load_row(const void *p, int dt, uint32_t c, uint32_t width) {
        lo = hi = Words4{0, 0, 0, 0};
        if (WHOLE && c >= width) return;
        if (!WHOLE && width < 8) {
            Raw8<DT_F32> wide;
            Raw8<DT_F16> half;
            wide.clear(), half.clear();
            if (dt == DT_F32) wide.load_last(p, opaque((int)width));
            else half.load_last(p, opaque((int)width));
#pragma unroll
            for (int q = 0; q < 4; q++) lo[q] = dt == DT_F32 ? wide.w[q] : half.w[q], hi[q] = wide.w[4 + q];
            return;
        }
        const char *at = static_cast<const char *>(p) + (uint32_t)place_of<WHOLE>(c, width).c * (dt == DT_F32 ? 4u : 2u);
        lo = *reinterpret_cast<const Words4At2 *>(at);
        if (dt == DT_F32) hi = reinterpret_cast<const Words4At2 *>(at)[1];
    }
    template <bool WHOLE>
    __device__ __forceinline__ void settle(int dt, uint32_t c, uint32_t width) {
        if (WHOLE || width < 8) return;  // (a row of fewer than eight came so)
        const int skip = opaque(place_of<WHOLE>(c, width).skip);
        if (skip <= 0) return;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if (q >= skip) continue;
            if (dt == DT_F32 && q < 4) lo[q & 3] = 0;
            else if (dt == DT_F32) hi[q & 3] = 0;
            else lo[q / 2] &= q & 1 ? 0u : 0xFFFF0000u;
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

template <int DT, bool WHOLE>
__device__ __forceinline__ void store8(void *p, uint32_t c, uint32_t width, const float (&v)[8]) {
    if (WHOLE ? c < width : c + 8 <= width) {
        Raw8<DT> r;
        r.set(v);
        r.store(elem<DT>(p, c));
    } else if (!WHOLE) {
        const Place l = place_of<WHOLE>(c, width);
        const int skip = opaque(l.skip);
        char *at = static_cast<char *>(p) + (ptrdiff_t)opaque(l.c) * (DT == DT_F32 ? 4 : 2);  // (before p in a row of fewer than eight)
        if constexpr (DT == DT_F32) {
#pragma unroll
            for (int q = 0; q < 8; q++)
                if (q >= skip) reinterpret_cast<float *>(at)[q] = v[q];
        } else {
            Raw8<DT> r;
            r.set(v);
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (2 * q >= skip) reinterpret_cast<WordAt2 *>(at)[q] = r.w[q];
                else if (2 * q + 1 == skip) reinterpret_cast<uint16_t *>(at)[2 * q + 1] = (uint16_t)(r.w[q] >> 16);
            }
        }
    }
}

}  // namespace exl3
