// The clip of many gradients by their global norm: norm = sqrt(sum of all g^2), scale = norm <= max_norm ? 1 : max_norm / norm,
// out = g scale.  Two passes over the gradients, as the scale needs every one of them; each is bound by its bytes.
//
// The tensors of a launch come as arguments.  They are cut into chunks of kClipChunk elements, numbered over the launch, and
// workgroup b takes chunks b, b + gridDim.x, ...  Squares are summed in 64 bits (an f32's square passes f32's range at 2e19),
// a workgroup's in a fixed order into its part, and the last workgroup to arrive in the last launch sums the parts in theirs.
#include "exl3_kernels.h"

namespace exl3 {

constexpr int CL_THREADS = 256;

// The tensor of chunk c: the last whose first chunk is not past it (tensors without elements have no chunks).
__device__ __forceinline__ int tensor_of(const ClipTensors &t, int c) {
    const int lane = threadIdx.x & 63;
    int before = 0;
#pragma unroll
    for (int i = 0; i < kClipTensors; i += 64) before += __popcll(__ballot(i + lane < t.count && t.first[min(i + lane, kClipTensors - 1)] <= c));
    return __builtin_amdgcn_readfirstlane(before - 1);
}

template <int DT>
struct Vec {
    static constexpr int N = DT == DT_F32 ? 4 : 8;  // elements of a 16-byte load
    static __device__ __forceinline__ void load(const void *p, int64_t i, float (&v)[N]) {
        if constexpr (DT == DT_F32) {
            const float4 u = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
            v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if constexpr (DT == DT_F16) v[2 * q] = h2f((uint16_t)w[q]), v[2 * q + 1] = h2f((uint16_t)(w[q] >> 16));
                else v[2 * q] = __uint_as_float(w[q] << 16), v[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
            }
        }
    }
};

template <int DT>
__device__ __forceinline__ double chunk_squares(const void *g, int64_t from, int64_t end) {
    constexpr int N = Vec<DT>::N;
    double s = 0.;
    if (reinterpret_cast<uintptr_t>(g) % 16 == 0) {
        int64_t i = from + (int64_t)threadIdx.x * N;
        for (; i + N <= end; i += CL_THREADS * N) {
            float v[N];
            Vec<DT>::load(g, i, v);
#pragma unroll
            for (int q = 0; q < N; q++) s += (double)v[q] * (double)v[q];
        }
        for (; i < end; i++) {  // one thread's, the last few
            const double v = load_act<DT>(g, i);
            s += v * v;
        }
    } else {
        for (int64_t i = from + threadIdx.x; i < end; i += CL_THREADS) {
            const double v = load_act<DT>(g, i);
            s += v * v;
        }
    }
    return s;
}

__device__ __forceinline__ double workgroup_sum(double s, double *red) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = red[0];
#pragma unroll
    for (int w = 1; w < CL_THREADS / 64; w++) s += red[w];
    __syncthreads();
    return s;
}

template <bool LAST>
__global__ __launch_bounds__(CL_THREADS) void clip_norm_kernel(ClipTensors t, ClipArgs a) {
    __shared__ double red[CL_THREADS / 64];
    __shared__ int flag;
    double s = 0.;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        const int64_t from = (int64_t)(c - t.first[k]) * kClipChunk, end = min(from + kClipChunk, t.n[k]);
        const int dt = t.dtype[k];
        if (dt == DT_F16) s += chunk_squares<DT_F16>(t.g[k], from, end);
        else if (dt == DT_BF16) s += chunk_squares<DT_BF16>(t.g[k], from, end);
        else s += chunk_squares<DT_F32>(t.g[k], from, end);
    }
    s = workgroup_sum(s, red);
    // A part is written through to memory and read past the caches, and counted once its store is acknowledged.
    if (threadIdx.x == 0) __hip_atomic_store(a.parts + a.first_part + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    if constexpr (LAST) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            const uint32_t old = __hip_atomic_fetch_add(a.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            flag = old == gridDim.x - 1;
            if (flag) __hip_atomic_store(a.counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!flag) return;
        s = 0.;
        for (int p = threadIdx.x; p < a.all_parts; p += CL_THREADS)
            s += __hip_atomic_load(a.parts + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        s = workgroup_sum(s, red);
        if (threadIdx.x == 0) {
            const double norm = sqrt(s);
            a.result[0] = (float)norm;
            const double scale = norm <= (double)a.max_norm ? 1. : (double)a.max_norm / norm;  // NaN stays NaN
            a.result[1] = (float)scale;
            // Below f32's normal range (a norm past 1e38) a factor has lost bits: it then comes in two.
            const bool tiny = scale > 0. && scale < 0x1p-100;
            a.factors[0] = tiny ? (float)(scale * 0x1p64) : (float)scale;
            a.factors[1] = tiny ? 0x1p-64f : 1.f;
        }
    }
}

template <int DT, int OT>
__device__ __forceinline__ void chunk_scale(const void *g, void *out, int64_t from, int64_t end, float scale, float rest) {
    for (int64_t i = from + threadIdx.x; i < end; i += CL_THREADS) store_act<OT>(out, i, load_act<DT>(g, i) * scale * rest);
}

template <int DT>
__device__ __forceinline__ void chunk_scale_to(const void *g, void *out, int ot, int64_t from, int64_t end, float scale, float rest) {
    if (ot == DT_F16) chunk_scale<DT, DT_F16>(g, out, from, end, scale, rest);
    else if (ot == DT_BF16) chunk_scale<DT, DT_BF16>(g, out, from, end, scale, rest);
    else chunk_scale<DT, DT_F32>(g, out, from, end, scale, rest);
}

__global__ __launch_bounds__(CL_THREADS) void clip_scale_kernel(ClipTensors t, const float *factors) {
    const float scale = factors[0], rest = factors[1];
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int k = tensor_of(t, c);
        if (scale == 1.f && t.g[k] == t.out[k]) continue;  // in place there is nothing to do
        const int64_t from = (int64_t)(c - t.first[k]) * kClipChunk, end = min(from + kClipChunk, t.n[k]);
        const int dt = t.dtype[k];
        if (dt == DT_F16) chunk_scale_to<DT_F16>(t.g[k], t.out[k], t.out_dtype[k], from, end, scale, rest);
        else if (dt == DT_BF16) chunk_scale_to<DT_BF16>(t.g[k], t.out[k], t.out_dtype[k], from, end, scale, rest);
        else chunk_scale_to<DT_F32>(t.g[k], t.out[k], t.out_dtype[k], from, end, scale, rest);
    }
}

hipError_t run_clip_norm(const ClipTensors &t, const ClipArgs &a, bool last, hipStream_t s) {
    const dim3 grid((unsigned)(t.chunks ? clip_parts(t.chunks) : 1));
    if (last) hipLaunchKernelGGL((clip_norm_kernel<true>), grid, dim3(CL_THREADS), 0, s, t, a);
    else hipLaunchKernelGGL((clip_norm_kernel<false>), grid, dim3(CL_THREADS), 0, s, t, a);
    return hipGetLastError();
}

hipError_t run_clip_scale(const ClipTensors &t, const float *factors, hipStream_t s) {
    hipLaunchKernelGGL(clip_scale_kernel, dim3((unsigned)(t.chunks < 4096 ? t.chunks : 4096)), dim3(CL_THREADS), 0, s, t, factors);
    return hipGetLastError();
}

}  // namespace exl3
