#include "exl3_router.h"

namespace exl3 {

// The choice of experts: exl3_route.h.  A launch takes up to 2^24 rows (its threads are numbered in 32 bits).
hipError_t run_route(const RouteArgs &a, hipStream_t s) {
    constexpr int most = 1 << 24;
    for (int r = 0; r < a.rows; r += min(most, a.rows - r)) {
        RouteArgs c = a;
        c.rows = min(most, a.rows - r);
        c.logits = static_cast<const char *>(a.logits) + (size_t)r * a.experts * (a.dtype == DT_F32 ? 4 : 2);
        c.mask = a.mask ? a.mask + r : nullptr;
        c.inds = a.inds + (size_t)r * a.topk;
        c.scores = a.scores + (size_t)r * a.topk;
        const hipError_t e = a.dtype == DT_F16 ? run_route_f16(c, s) : a.dtype == DT_BF16 ? run_route_bf16(c, s) : run_route_f32(c, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// ---------------------------------------------------------------------------------------------------------------
// The gradient of the logits through the scores, with ds the scores' gradient times scale, p as above and r = p / sum over
// the row's slots of p:
//   softmax, renorm:  dx_e = sum over slots i on e of r_i (ds_i - sum_j r_j ds_j)
//   sigmoid, renorm:  the same times 1 - p_i
//   sigmoid:          dx_e = sum over slots i on e of p_i (1 - p_i) ds_i
//   softmax:          dx_e = sum over slots i on e of p_i ds_i - p_e sum_j p_j ds_j
// A slot whose id is past the experts has no score.  All but the last (DENSE) read the picked logits alone, and write a row
// of zeros with the slots' terms in it.
//
// A row is held by L lanes as in the balance loss's kernel, lane l holding PER experts and SPL slots.
constexpr int RT_THREADS = 256;

template <int L, int PER, int SPL, int DT, bool VEC, bool DENSE>
__global__ __launch_bounds__(RT_THREADS) void route_backward_kernel(RouteGradArgs a) {
    constexpr int G = RT_THREADS / L;
    const int l = threadIdx.x & (L - 1), grp = threadIdx.x / L, e0 = l * PER;
    __shared__ __align__(16) float rows_lds[G][L * PER];
    float *at = rows_lds[grp];
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * G;
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < rows; r0 += step) {
        const size_t r = r0 + grp;
        const bool in = r < rows, live = in && (!a.mask || a.mask[r] != 0);
        float d[PER], ds[SPL], x[SPL];
        int ind[SPL];
#pragma unroll
        for (int i = 0; i < SPL; i++) {
            const int j = l + i * L;
            const size_t slot = r * a.topk + j;
            const bool has = live && j < a.topk;
            ind[i] = has && a.inds[has ? slot : 0] < (uint32_t)a.experts ? (int)a.inds[slot] : -1;
            ds[i] = ind[i] >= 0 ? a.dscores[slot] * a.scale : 0.f;
            x[i] = ind[i] >= 0 ? load_act<DT>(a.logits, r * a.experts + ind[i]) : -INFINITY;
        }
        float mx = -INFINITY, inv = 0.f;
        if constexpr (DENSE) {
            Logits<PER, DT, VEC> row = {};
            if (live) row.load(a.logits, r * a.experts, a.experts, e0);
            row.unpack(a.experts, e0, live, d);
            mx = d[0];
#pragma unroll
            for (int q = 1; q < PER; q++) mx = fmaxf(mx, d[q]);
            mx = group_max<L>(mx);
            const float base = mx == -INFINITY ? 0.f : mx;
            float den = 0.f;
#pragma unroll
            for (int q = 0; q < PER; q++) {
                d[q] = __expf(d[q] - base);
                den += d[q];
            }
            den = group_sum<L>(den);
            inv = den == 0.f ? 0.f : 1.f / den;
            mx = base;
        } else {
            if (a.renorm) {
#pragma unroll
                for (int i = 0; i < SPL; i++) mx = fmaxf(mx, a.sigmoid ? fminf(x[i], 0.f) : x[i]);
                mx = group_max<L>(mx);
                mx = mx == -INFINITY ? 0.f : mx;
            }
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] = 0.f;
        }
        // the slots' terms
        float t[SPL], dot = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < SPL; i++) {
            float w;
            if constexpr (DENSE) w = expf(x[i] - mx) * inv;
            else if (!a.sigmoid) w = expf(x[i] - mx);
            else {
                const float e = expf(-fabsf(x[i]));
                w = a.renorm ? expf(fminf(x[i], 0.f) - mx) / (1.f + e) : (x[i] >= 0.f ? 1.f : e) / (1.f + e);
            }
            w = ind[i] >= 0 ? w : 0.f;
            t[i] = w;
            sum += w;
            dot += w * ds[i];
        }
        if (DENSE || a.renorm) dot = group_sum<L>(dot);
        if constexpr (!DENSE) {
            if (a.renorm) {
                sum = group_sum<L>(sum);
                inv = sum == 0.f ? 0.f : 1.f / sum;
                dot *= inv;
            }
        }
#pragma unroll
        for (int i = 0; i < SPL; i++) {
            if constexpr (DENSE) t[i] *= ds[i];
            else {
                t[i] = a.renorm ? t[i] * inv * (ds[i] - dot) : t[i] * ds[i];
                if (a.sigmoid) {
                    const float e = expf(-fabsf(x[i]));
                    t[i] *= (x[i] >= 0.f ? e : 1.f) / (1.f + e);
                }
            }
        }
        if constexpr (DENSE) {
            const float c = dot * inv;
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] *= -c;
        }
        // Into the row by way of LDS (a wave's own rows: no barrier).  Every slot leaves its number at its expert: where two
        // of a row's slots name one expert, some slot does not find its own again.
        wave_order();
#pragma unroll
        for (int i = 0; i < SPL; i++)
            if (ind[i] >= 0) at[ind[i]] = __int_as_float(l + i * L + 1);
        wave_order();
        bool twice = false;
#pragma unroll
        for (int i = 0; i < SPL; i++) twice |= ind[i] >= 0 && __float_as_int(at[max(ind[i], 0)]) != l + i * L + 1;
        wave_order();
        if (__any(twice)) {  // slot by slot, so equal experts' terms always add in slot order
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                const int n = min(L, a.topk - i * L);
                for (int j = 0; j < n; j++) {
                    const int e = __shfl(ind[i], j, L) - e0;
                    const float v = __shfl(t[i], j, L);
#pragma unroll
                    for (int q = 0; q < PER; q++) d[q] += e == q ? v : 0.f;
                }
            }
        } else {
#pragma unroll
            for (int q = 0; q < PER; q++) at[e0 + q] = d[q];
            wave_order();
#pragma unroll
            for (int i = 0; i < SPL; i++)
                if (ind[i] >= 0) at[ind[i]] += t[i];
            wave_order();
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] = at[e0 + q];
        }
        wave_order();
        if (in) store_logits<PER, DT, VEC>(a.dlogits, r * a.experts, a.experts, e0, live, d);
    }
}

hipError_t run_route_backward(const RouteGradArgs &a, hipStream_t s) {
    const bool dense = !a.sigmoid && !a.renorm;
    return with_shape(a.experts, [&](auto L, auto PER) {
        return with_dtype(a.dtype, [&](auto DT) {
            constexpr int l = decltype(L)::value, per = decltype(PER)::value, dt = decltype(DT)::value;
            const long groups = ((long)a.rows + RT_THREADS / l - 1) / (RT_THREADS / l);
            const dim3 grid((unsigned)(groups < 2048 ? groups : 2048));
            const bool vec = whole_vectors<per, dt>(a.logits, a.experts) && whole_vectors<per, dt>(a.dlogits, a.experts);
            auto launch = [&](auto SPL) {
                constexpr int spl = decltype(SPL)::value;
                auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(RT_THREADS), 0, s, a); };
                if (dense) vec ? go(route_backward_kernel<l, per, spl, dt, true, true>) : go(route_backward_kernel<l, per, spl, dt, false, true>);
                else vec ? go(route_backward_kernel<l, per, spl, dt, true, false>) : go(route_backward_kernel<l, per, spl, dt, false, false>);
                return hipGetLastError();
            };
            if constexpr (l < 32)
                if (a.topk > l) return launch(std::integral_constant<int, 32 / l>{});
            return launch(std::integral_constant<int, 1>{});
        });
    });
}

}  // namespace exl3
