// The clip of many gradients by their global norm: norm = sqrt(sum of all g^2), scale = norm <= max_norm ? 1 : max_norm / norm,
// out = g scale.  Two passes over the gradients, as the scale needs every one of them; each is bound by its bytes: 193 tensors of
// 573 MB (bf16 and f32) in place take 347 us, 5.0 TB/s over two reads and a write.  Small ones are launches, one a pass for every
// 160 tensors (what a launch's arguments hold): 6 tensors of 0.5 MB take 7.1 us.
//
// The tensors of a launch come as arguments.  They are cut into chunks of kClipChunk elements, numbered over the launch, and a
// workgroup takes a run of them, so that it looks for its tensor once for each that it touches.  Squares are summed in 64 bits
// (an f32's square passes f32's range at 2e19), a workgroup's in a fixed order into its part, and the last workgroup to arrive
// in the last launch sums the parts in theirs.
#include "exl3_vec.h"

namespace exl3 {

constexpr int CL_THREADS = 256;
constexpr int CL_AHEAD = 4;  // vectors of eight that a thread has in flight
constexpr int CL_STEP = CL_THREADS * 8 * CL_AHEAD;

// The tensor of chunk c: the last whose first chunk is not past it (tensors without elements are left out).
__device__ __forceinline__ int tensor_of(const ClipTensors &t, int c) {
    const int lane = threadIdx.x & 63;
    int before = 0;
#pragma unroll
    for (int i = 0; i < kClipTensors; i += 64)
        before += __popcll(__ballot(i + lane < t.count && t.e[min(i + lane, kClipTensors - 1)].first <= c));
    return __builtin_amdgcn_readfirstlane(before - 1);
}

// Calls f(entry, from, end) for the elements of each tensor in this workgroup's run of chunks, the last tensor first if BACK.
template <bool BACK, class F>
__device__ __forceinline__ void for_run(const ClipTensors &t, F f) {
    const int per = (t.chunks + (int)gridDim.x - 1) / (int)gridDim.x;
    int first = min(t.chunks, (int)blockIdx.x * per), last = min(t.chunks, first + per);
    while (first < last) {
        const int k = tensor_of(t, BACK ? last - 1 : first), past = k + 1 < t.count ? t.e[min(k + 1, kClipTensors - 1)].first : t.chunks;
        const ClipEntry e = t.e[k];
        const int c = BACK ? max(first, e.first) : first;
        const int64_t from = (int64_t)(c - e.first) * kClipChunk, n = (int64_t)(past - 1 - e.first) * kClipChunk + e.last;
        const int64_t end = min(from + (int64_t)(last - c) * kClipChunk, n);
        f(e, from, end);
        if (BACK) last = c;
        else first += (int)((end - from + kClipChunk - 1) / kClipChunk);
    }
}

template <int DT>
__device__ __forceinline__ double squares(const char *g, int64_t count) {
    constexpr int SIZE = DT == DT_F32 ? 4 : 2;
    double s[2] = {0., 0.};
    int64_t i = (int64_t)threadIdx.x * 8;
    for (; i - (int64_t)threadIdx.x * 8 + CL_STEP <= count; i += CL_STEP) {
        Raw8<DT> r[CL_AHEAD];
#pragma unroll
        for (int k = 0; k < CL_AHEAD; k++) r[k].load(g + (i + k * CL_THREADS * 8) * SIZE);
#pragma unroll
        for (int k = 0; k < CL_AHEAD; k++)
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const double v = r[k].get(q);
                s[q & 1] = fma(v, v, s[q & 1]);
            }
    }
    for (; i < count; i += CL_THREADS * 8) {
        Raw8<DT> r;
        if (i + 8 <= count) r.load(g + i * SIZE);
        else r.load_some(g + i * SIZE, (int)(count - i));
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const double v = r.get(q);
            s[q & 1] = fma(v, v, s[q & 1]);
        }
    }
    return s[0] + s[1];
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
    for_run<false>(t, [&](const ClipEntry &e, int64_t from, int64_t end) {
        const char *g = static_cast<const char *>(e.g) + from * (e.dtype == DT_F32 ? 4 : 2);
        s += e.dtype == DT_F16    ? squares<DT_F16>(g, end - from)
             : e.dtype == DT_BF16 ? squares<DT_BF16>(g, end - from)
                                  : squares<DT_F32>(g, end - from);
    });
    s = workgroup_sum(s, red);
    // A part is written through to memory and read past the caches, and counted once its store is acknowledged.
    if (threadIdx.x == 0) __hip_atomic_store(a.parts + a.first_part + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    if constexpr (LAST) {
        if (threadIdx.x == 0) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const uint32_t old = __hip_atomic_fetch_add(a.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            flag = old == gridDim.x - 1;
            if (flag) __hip_atomic_store(a.counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!flag) return;
        s = 0.;
        for (int p0 = threadIdx.x; p0 < a.all_parts; p0 += 4 * CL_THREADS) {
            double v[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                v[i] = __hip_atomic_load(a.parts + min(p0 + i * CL_THREADS, a.all_parts - 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
#pragma unroll
            for (int i = 0; i < 4; i++) s += p0 + i * CL_THREADS < a.all_parts ? v[i] : 0.;
        }
        s = workgroup_sum(s, red);
        if (threadIdx.x == 0) {
            const double norm = sqrt(s);
            a.result[0] = (float)norm;
            const double scale = norm <= (double)a.max_norm ? 1. : (double)a.max_norm / norm;  // NaN stays NaN
            a.result[1] = (float)scale;
            // Towards the end of f32's range a factor loses bits, where its products with a far norm's gradients need not: it
            // then comes as a mantissa and a power of two (down to 2^-300, past any one factor).
            int power = 0;
            a.factors[0] = (float)(scale > 0. && scale < 0x1p-100 ? frexp(scale, &power) : scale);
            a.factors[1] = (float)power;
        }
    }
}

// Each vector is read by the thread that writes it, in place too.  From the end to the beginning, as the first pass read the end
// last: what of it the memory-side cache still holds is not read from memory again.
template <int DT, int OT>
__device__ __forceinline__ void scaled(const char *g, char *out, int64_t count, float scale, int power) {
    constexpr int SIZE = DT == DT_F32 ? 4 : 2, OSIZE = OT == DT_F32 ? 4 : 2;
    auto times = [&](const Raw8<DT> &r, Raw8<OT> &o) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; q++) v[q] = __builtin_amdgcn_ldexpf(r.get(q) * scale, power);
        o.set(v);
    };
    const int64_t whole = count / CL_STEP * CL_STEP;
    for (int64_t i = whole + (int64_t)threadIdx.x * 8; i < count; i += CL_THREADS * 8) {
        if (i + 8 <= count) {
            Raw8<DT> r;
            Raw8<OT> o;
            r.load(g + i * SIZE);
            times(r, o);
            o.store(out + i * OSIZE);
        } else {
            for (int64_t j = i; j < count; j++) store_act<OT>(out, j, __builtin_amdgcn_ldexpf(load_act<DT>(g, j) * scale, power));
        }
    }
    for (int64_t i = whole - CL_STEP + (int64_t)threadIdx.x * 8; i >= 0; i -= CL_STEP) {
        Raw8<DT> r[CL_AHEAD];
#pragma unroll
        for (int k = 0; k < CL_AHEAD; k++) r[k].load(g + (i + k * CL_THREADS * 8) * SIZE);
#pragma unroll
        for (int k = 0; k < CL_AHEAD; k++) {
            Raw8<OT> o;
            times(r[k], o);
            o.store(out + (i + k * CL_THREADS * 8) * OSIZE);
        }
    }
}

template <int DT>
__device__ __forceinline__ void scaled_to(const char *g, char *out, int ot, int64_t count, float scale, int power) {
    if (ot == DT_F16) scaled<DT, DT_F16>(g, out, count, scale, power);
    else if (ot == DT_BF16) scaled<DT, DT_BF16>(g, out, count, scale, power);
    else scaled<DT, DT_F32>(g, out, count, scale, power);
}

__global__ __launch_bounds__(CL_THREADS) void clip_scale_kernel(ClipTensors t, const float *factors) {
    const float scale = factors[0];
    const int power = (int)factors[1];
    for_run<true>(t, [&](const ClipEntry &e, int64_t from, int64_t end) {
        if (scale == 1.f && !power && e.g == e.out) return;  // in place there is nothing to do
        const char *g = static_cast<const char *>(e.g) + from * (e.dtype == DT_F32 ? 4 : 2);
        char *out = static_cast<char *>(e.out) + from * (e.out_dtype == DT_F32 ? 4 : 2);
        if (e.dtype == DT_F16) scaled_to<DT_F16>(g, out, e.out_dtype, end - from, scale, power);
        else if (e.dtype == DT_BF16) scaled_to<DT_BF16>(g, out, e.out_dtype, end - from, scale, power);
        else scaled_to<DT_F32>(g, out, e.out_dtype, end - from, scale, power);
    });
}

hipError_t run_clip_norm(const ClipTensors &t, const ClipArgs &a, bool last, hipStream_t s) {
    const dim3 grid((unsigned)(t.chunks ? clip_parts(t.chunks) : 1));
    if (last) hipLaunchKernelGGL((clip_norm_kernel<true>), grid, dim3(CL_THREADS), 0, s, t, a);
    else hipLaunchKernelGGL((clip_norm_kernel<false>), grid, dim3(CL_THREADS), 0, s, t, a);
    return hipGetLastError();
}

hipError_t run_clip_scale(const ClipTensors &t, const float *factors, hipStream_t s) {
    hipLaunchKernelGGL(clip_scale_kernel, dim3((unsigned)clip_parts(t.chunks)), dim3(CL_THREADS), 0, s, t, factors);
    return hipGetLastError();
}

}  // namespace exl3
