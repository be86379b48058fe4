// The router's balance loss with the experts' counts, and the gradient of the router's logits.
//
// Over T live rows (mask), E experts and k slots a row, p = softmax(logits) and c_e the live rows' slots on expert e:
//   w_e = coef E c_e / (T k) / T,   loss = sum_e w_e sum_r p_re
//   dlogit_re = dloss p_re (w_e - sum_j w_j p_rj)  +  sum over r's slots i on expert e of s_i (ds_i - sum_j s_j ds_j)
// with s the softmax of the logits that the row's slots picked (the routing chain's scores) and ds their gradient.  The
// counts are constants of the gradient.  Both passes read the logits once and are bound by that read.
//
// A row is held by L lanes, lane l of them holding experts PER l .. PER l + PER - 1 (one 16- or 32-byte load where the row's
// length allows it), so a wave holds 64 / L rows and a row's sums take log2(L) DPP or shuffle steps; the balance loss adds
// each row's p to sums that stay in the lane's registers over all its rows.  Every sum has a fixed order.
#include "exl3_kernels.h"
#include "exl3_epilogue.h"

#include <type_traits>

namespace exl3 {

template <int L>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int m = L / 2; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int m = L / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// The lane's PER logits of a row as f32; -inf past the row's end.  VEC: whole, aligned vectors (the host checks).
template <int PER, int DT, bool VEC>
__device__ __forceinline__ void load_logits(const void *logits, size_t row, int experts, int e0, float (&v)[PER]) {
    const size_t at = row * (size_t)experts;
    if constexpr (VEC) {
        constexpr int BYTES = PER * (DT == DT_F32 ? 4 : 2);
        const bool in = e0 < experts;  // experts is a multiple of PER: all of the lane's or none
        const char *p = static_cast<const char *>(logits) + (at + (in ? e0 : 0)) * (DT == DT_F32 ? 4 : 2);
        uint32_t w[(BYTES + 3) / 4];
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
#pragma unroll
        for (int q = 0; q < PER; q++) {
            float x;
            if constexpr (DT == DT_F32) x = __uint_as_float(w[q]);
            else {
                const uint32_t h = q & 1 ? w[q >> 1] >> 16 : w[q >> 1] & 0xFFFFu;
                x = DT == DT_F16 ? h2f((uint16_t)h) : __uint_as_float(h << 16);
            }
            v[q] = in ? x : -INFINITY;
        }
    } else {
#pragma unroll
        for (int q = 0; q < PER; q++) {
            const float x = load_act<DT>(logits, at + (size_t)min(e0 + q, experts - 1));
            v[q] = e0 + q < experts ? x : -INFINITY;
        }
    }
}

// v becomes the row's softmax.  A row of -inf alone has no probabilities (zeros); NaN stays.
template <int L, int PER>
__device__ __forceinline__ void row_softmax(float (&v)[PER]) {
    float mx = -INFINITY;
#pragma unroll
    for (int q = 0; q < PER; q++) mx = fmaxf(mx, v[q]);
    mx = group_max<L>(mx);
    const float base = mx == -INFINITY ? 0.f : mx;
    float den = 0.f;
#pragma unroll
    for (int q = 0; q < PER; q++) {
        v[q] = __expf(v[q] - base);
        den += v[q];
    }
    den = group_sum<L>(den);
    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
    for (int q = 0; q < PER; q++) v[q] *= inv;
}

constexpr int RB_THREADS = 256;

// The loss, counts and weights from E sums and counts in LDS (all threads of the workgroup).
__device__ __forceinline__ void balance_finish(const BalanceArgs &a, const float *psum, const int *count, int live,
                                               float *red) {
    const float T = (float)live;
    const float scale = live > 0 ? a.coef * (float)a.experts / (T * (float)a.topk) / T : 0.f;
    float part = 0.f;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        const float w = scale * (float)count[e];
        a.weight[e] = w;
        a.counts[e] = count[e];
        part += w * psum[e];
    }
    part = group_sum<64>(part);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = part;
    __syncthreads();
    if (threadIdx.x == 0) {
        float s = 0.f;
        for (int w = 0; w < (int)(blockDim.x >> 6); w++) s += red[w];
        *a.loss = s;
    }
}

// Workgroup b sums rows b, b + gridDim.x, ... (in strides of the rows it holds at once) into its part: E sums, E counts and
// its live rows.  A grid of one workgroup finishes by itself.
template <int L, int PER, int DT, bool VEC>
__global__ __launch_bounds__(RB_THREADS) void balance_kernel(BalanceArgs a) {
    constexpr int G = RB_THREADS / L;  // rows at once
    __shared__ float sums[L * PER];
    __shared__ int hist[L * PER];
    __shared__ int live_rows;
    __shared__ float red[RB_THREADS / 64];
    const int tid = threadIdx.x, l = tid & (L - 1), grp = tid / L, e0 = l * PER;
    for (int e = tid; e < L * PER; e += RB_THREADS) hist[e] = 0;
    if (tid == 0) live_rows = 0;
    __syncthreads();
    float acc[PER] = {};
    int mine = 0;
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < (size_t)a.rows; r0 += (size_t)gridDim.x * G) {
        const size_t r = r0 + grp;
        const size_t rr = r < (size_t)a.rows ? r : (size_t)a.rows - 1;
        const bool live = r < (size_t)a.rows && (!a.mask || a.mask[rr]);
        float v[PER];
        load_logits<PER, DT, VEC>(a.logits, rr, a.experts, e0, v);
        row_softmax<L, PER>(v);
#pragma unroll
        for (int q = 0; q < PER; q++) acc[q] += live ? v[q] : 0.f;
        if (live) {
            for (int j = l; j < a.topk; j += L) {
                const uint32_t e = a.inds[rr * a.topk + j];
                if (e < (uint32_t)a.experts) atomicAdd(&hist[e], 1);
            }
            mine += l == 0 ? 1 : 0;
        }
    }
    if (mine) atomicAdd(&live_rows, mine);
    // the workgroup's row groups one after another, so the order of the sum is fixed
    for (int g = 0; g < G; g++) {
        if (grp == g) {
#pragma unroll
            for (int q = 0; q < PER; q++) sums[e0 + q] = g == 0 ? acc[q] : sums[e0 + q] + acc[q];
        }
        __syncthreads();
    }
    if (gridDim.x == 1) {
        balance_finish(a, sums, hist, live_rows, red);
        return;
    }
    for (int e = tid; e < a.experts; e += RB_THREADS) {
        a.part_sum[(size_t)blockIdx.x * a.experts + e] = sums[e];
        a.part_count[(size_t)blockIdx.x * a.experts + e] = hist[e];
    }
    if (tid == 0) a.part_live[blockIdx.x] = live_rows;
}

// One workgroup: the parts of the `parts` workgroups, in their order.
constexpr int BF_THREADS = 1024;
__global__ __launch_bounds__(BF_THREADS) void balance_finish_kernel(BalanceArgs a, int parts) {
    __shared__ float sums[BF_THREADS];
    __shared__ int hist[BF_THREADS];
    __shared__ float red[BF_THREADS / 64];
    __shared__ int live_rows;
    const int tid = threadIdx.x;
    // S threads an expert, thread s of them summing parts s, s + S, ...; their sums then added in order
    int width = 1;
    while (width < a.experts) width <<= 1;
    const int S = BF_THREADS / width, e = tid & (width - 1), s = tid / width;
    if (tid == 0) live_rows = 0;
    float x = 0.f;
    int c = 0;
    if (e < a.experts)
        for (int b = s; b < parts; b += S) {
            x += a.part_sum[(size_t)b * a.experts + e];
            c += a.part_count[(size_t)b * a.experts + e];
        }
    sums[tid] = x;
    hist[tid] = c;
    int live = 0;
    __syncthreads();
    for (int b = tid; b < parts; b += BF_THREADS) live += a.part_live[b];
    if (live) atomicAdd(&live_rows, live);
    for (int half = S / 2; half >= 1; half >>= 1) {
        if (s < half) {
            sums[tid] += sums[tid + half * width];
            hist[tid] += hist[tid + half * width];
        }
        __syncthreads();
    }
    __syncthreads();
    balance_finish(a, sums, hist, live_rows, red);
}

// dlogits: each group of L lanes takes rows in strides of the grid.
template <int L, int PER, int DT, bool VEC>
__global__ __launch_bounds__(RB_THREADS) void router_backward_kernel(RouterGradArgs a) {
    constexpr int G = RB_THREADS / L;
    constexpr int SPL = L >= 32 ? 1 : 32 / L;  // slots a lane holds (up to 32 a row)
    const int l = threadIdx.x & (L - 1), grp = threadIdx.x / L, e0 = l * PER;
    float w[PER];
    const float dloss = a.weight ? *a.dloss : 0.f;
#pragma unroll
    for (int q = 0; q < PER; q++) w[q] = a.weight && e0 + q < a.experts ? a.weight[e0 + q] : 0.f;
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < (size_t)a.rows; r0 += (size_t)gridDim.x * G) {
        const size_t r = r0 + grp, rr = r < (size_t)a.rows ? r : (size_t)a.rows - 1;
        const bool live = !a.mask || a.mask[rr];
        float d[PER];
        load_logits<PER, DT, VEC>(a.logits, rr, a.experts, e0, d);
        if (a.weight) {
            row_softmax<L, PER>(d);
            float dot = 0.f;
#pragma unroll
            for (int q = 0; q < PER; q++) dot += w[q] * d[q];
            dot = group_sum<L>(dot);
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] = dloss * d[q] * (w[q] - dot);
        } else {
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] = 0.f;
        }
        if (a.dscores) {
            // the row's slots: lane l holds slots l, l + L, ...; a slot with no expert has no score
            int ind[SPL];
            float s[SPL], g[SPL], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                const int j = l + i * L;
                const bool has = j < a.topk;
                const uint32_t e = has ? a.inds[rr * a.topk + j] : 0xFFFFFFFFu;
                g[i] = has ? a.dscores[rr * a.topk + j] : 0.f;
                ind[i] = e < (uint32_t)a.experts ? (int)e : -1;
                s[i] = ind[i] >= 0 ? load_act<DT>(a.logits, rr * (size_t)a.experts + ind[i]) : -INFINITY;
                mx = fmaxf(mx, s[i]);
            }
            mx = group_max<L>(mx);
            const float base = mx == -INFINITY ? 0.f : mx;
            float den = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                s[i] = __expf(s[i] - base);
                den += s[i];
            }
            den = group_sum<L>(den);
            const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                s[i] *= inv;
                dot += ind[i] >= 0 ? s[i] * g[i] : 0.f;
            }
            dot = group_sum<L>(dot);
#pragma unroll
            for (int i = 0; i < SPL; i++) g[i] = s[i] * (g[i] - dot);
            // each slot's term to the lane that holds its expert, in slot order
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                const int n = min(L, a.topk - i * L);
                for (int j = 0; j < n; j++) {
                    const int e = __shfl(ind[i], j, L) - e0;
                    const float t = __shfl(g[i], j, L);
#pragma unroll
                    for (int q = 0; q < PER; q++) d[q] += e == q ? t : 0.f;
                }
            }
        }
        if (r < (size_t)a.rows) {
            const size_t o = r * (size_t)a.experts + e0;
#pragma unroll
            for (int q = 0; q < PER; q++)
                if (e0 + q < a.experts) store_act<DT>(a.dlogits, o + q, live ? d[q] : 0.f);
        }
    }
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

static int lanes_of(int experts) {
    return experts <= 64 ? 8 : experts <= 128 ? 16 : experts <= 256 ? 32 : 64;
}

int balance_parts(int rows, int experts) {
    const int at_once = RB_THREADS / lanes_of(experts);
    const long groups = ((long)rows + at_once - 1) / at_once;
    return (int)(groups <= 4 ? 1 : groups < kBalanceMaxParts ? groups : kBalanceMaxParts);
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

hipError_t run_balance_loss(const BalanceArgs &a, hipStream_t s) {
    const int parts = balance_parts(a.rows, a.experts);
    const hipError_t e = with_shape(a.experts, [&](auto L, auto PER) {
        return with_dtype(a.dtype, [&](auto DT) {
            constexpr int l = decltype(L)::value, per = decltype(PER)::value, dt = decltype(DT)::value;
            if (whole_vectors<per, dt>(a.logits, a.experts))
                hipLaunchKernelGGL((balance_kernel<l, per, dt, true>), dim3((unsigned)parts), dim3(RB_THREADS), 0, s, a);
            else
                hipLaunchKernelGGL((balance_kernel<l, per, dt, false>), dim3((unsigned)parts), dim3(RB_THREADS), 0, s, a);
            return hipGetLastError();
        });
    });
    if (e != hipSuccess || parts == 1) return e;
    hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(BF_THREADS), 0, s, a, parts);
    return hipGetLastError();
}

hipError_t run_router_backward(const RouterGradArgs &a, hipStream_t s) {
    const int at_once = RB_THREADS / lanes_of(a.experts);
    const long groups = ((long)a.rows + at_once - 1) / at_once;
    const unsigned grid = (unsigned)(groups < 4096 ? groups : 4096);
    return with_shape(a.experts, [&](auto L, auto PER) {
        return with_dtype(a.dtype, [&](auto DT) {
            constexpr int l = decltype(L)::value, per = decltype(PER)::value, dt = decltype(DT)::value;
            if (whole_vectors<per, dt>(a.logits, a.experts))
                hipLaunchKernelGGL((router_backward_kernel<l, per, dt, true>), dim3(grid), dim3(RB_THREADS), 0, s, a);
            else
                hipLaunchKernelGGL((router_backward_kernel<l, per, dt, false>), dim3(grid), dim3(RB_THREADS), 0, s, a);
            return hipGetLastError();
        });
    });
}

}  // namespace exl3
