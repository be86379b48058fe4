// The choice of experts.  With x a row of logits, p = softmax(x) or sigmoid(x) and c = p + bias:
//   of G groups of E / G experts the `taken` with the largest value (the sum of a group's one or two largest c),
//   of their experts the k with the largest c, listed in falling order, equal ones by their number,
//   score_i = scale p_i / (renorm ? sum over the picks of p : 1).
// Without bias, and with one group or a group's largest c as its value, the order of c is the order of x.  A logit of -inf
// takes its expert out; so do a bias of -inf or NaN, a NaN logit and, under softmax, +inf, and the last two make the row's
// scores NaN.  Slots that no expert is left for, and all slots of a row that `mask` leaves out, hold 0xFFFFFFFF and 0.
#include "exl3_router.h"

namespace exl3 {

constexpr int RT_THREADS = 256;
constexpr int NO_EXPERT = 0x7FFFFFFF;

// The better of two candidates: the larger value, of equal ones the lower number (NO_EXPERT, with -inf, is worse than any).
__device__ __forceinline__ bool better(double c, int i, double d, int j) { return c > d || (c == d && i < j); }

// The best of the wave's candidates, in every lane.
__device__ __forceinline__ void wave_best(double &c, int &i) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const double d = __shfl_xor(c, m);
        const int j = __shfl_xor(i, m);
        const bool take = better(d, j, c, i);
        c = take ? d : c;
        i = take ? j : i;
    }
}

// The score's part of pick x before the sum: p for a score that keeps its value, else p over a factor that the row's picks
// share (`top`: their largest x or min(x, 0)), so that far negative logits keep their ratios.
__device__ __forceinline__ float pick_weight(const RouteArgs &a, float x, float top, float row_max, float row_den) {
    if (!a.sigmoid) return a.renorm ? expf(x - top) : expf(x - row_max) / row_den;
    const float e = expf(-fabsf(x));
    if (a.renorm) return expf(fminf(x, 0.f) - top) / (1.f + e);
    return (x >= 0.f ? 1.f : e) / (1.f + e);
}

// A row by one wave, lane l holding experts l, l + 64, ...; everything that decides in 64 bits.
template <int PER, int DT>
__device__ __forceinline__ void route_row(const RouteArgs &a, size_t row, int lane) {
    const size_t at = row * a.experts;
    float x[PER];
    double c[PER];
    uint32_t out = 0;  // bit i: expert lane + 64 i is out of the choice
    bool bad = false;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 64 * i;
        x[i] = load_act<DT>(a.logits, at + min(e, a.experts - 1));
        const bool nan = x[i] != x[i] || (!a.sigmoid && x[i] == INFINITY);
        bad |= nan && e < a.experts;
        const float b = a.bias && e < a.experts ? a.bias[e] : 0.f;
        const bool off = e >= a.experts || nan || x[i] == -INFINITY || !(b > -INFINITY);
        out |= off ? 1u << i : 0u;
        // (an expert that its bias takes out still has its share of the softmax)
        if (e < a.experts && !nan) mx = fmaxf(mx, x[i]);
    }
    bad = __any(bad);
    mx = group_max<64>(mx);
    const bool by_logit = !a.bias && (a.groups == 1 || a.group_top == 1);
    double den = 1.;
    if (!a.sigmoid && !(by_logit && a.renorm)) {
        den = 0.;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const bool in = lane + 64 * i < a.experts && x[i] > -INFINITY && x[i] < INFINITY;
            c[i] = in ? exp((double)x[i] - (double)mx) : 0.;
            den += c[i];
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) den += __shfl_xor(den, m);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane + 64 * i;
        if (by_logit) c[i] = (double)x[i];
        else {
            const double p = a.sigmoid ? 1. / (1. + exp(-(double)x[i])) : c[i] / den;
            c[i] = p + (a.bias && e < a.experts ? (double)a.bias[e] : 0.);
        }
    }
    auto best_of = [&](int first, int end, uint32_t without, double &bc, int &bi) {
        bc = -INFINITY;
        bi = NO_EXPERT;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane + 64 * i;
            const bool take = e >= first && e < end && !((without >> i) & 1u) && better(c[i], e, bc, bi);
            bc = take ? c[i] : bc;
            bi = take ? e : bi;
        }
        wave_best(bc, bi);
    };
    if (a.groups > 1) {
        const int size = a.experts / a.groups;
        double worth = -INFINITY;
        for (int g = 0; g < a.groups; g++) {
            double c1, c2 = 0.;
            int i1, i2 = NO_EXPERT;
            best_of(g * size, (g + 1) * size, out, c1, i1);
            if (a.group_top == 2) {
                const uint32_t mine = (i1 & 63) == lane && i1 != NO_EXPERT ? 1u << (i1 >> 6) : 0u;
                best_of(g * size, (g + 1) * size, out | mine, c2, i2);
            }
            if (lane == g) worth = i2 == NO_EXPERT ? c1 : c1 + c2;
        }
        int ahead = 0;
        for (int g = 0; g < a.groups; g++) {
            const double w = __shfl(worth, g);
            ahead += better(w, g, worth, lane) ? 1 : 0;
        }
        const uint64_t open = __ballot(lane < a.groups && ahead < a.taken && worth > -INFINITY);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int g = min(lane + 64 * i, a.experts - 1) / size;
            out |= (open >> g) & 1 ? 0u : 1u << i;
        }
    }
    int mine = NO_EXPERT;
    for (int j = 0; j < a.topk; j++) {
        double bc;
        int bi;
        best_of(0, a.experts, out, bc, bi);
        if (bi == NO_EXPERT) break;
        out |= (bi & 63) == lane ? 1u << (bi >> 6) : 0u;
        mine = lane == j ? bi : mine;
    }
    const bool has = mine != NO_EXPERT;
    const float px = has ? load_act<DT>(a.logits, at + mine) : -INFINITY;
    const float top = group_max<64>(a.sigmoid ? fminf(px, 0.f) : px);
    float w = has ? pick_weight(a, px, top, mx, (float)den) : 0.f;
    if (a.renorm) {
        const float sum = group_sum<64>(w);
        w = has ? w / sum : 0.f;
    }
    if (lane < a.topk) {
        a.inds[row * a.topk + lane] = has ? (uint32_t)mine : 0xFFFFFFFFu;
        a.scores[row * a.topk + lane] = bad ? NAN : w * a.scale;
    }
}

template <int PER, int DT>
__global__ __launch_bounds__(RT_THREADS) void route_kernel(RouteArgs a) {
    const int lane = threadIdx.x & 63;
    const size_t row = (size_t)blockIdx.x * (RT_THREADS / 64) + (threadIdx.x >> 6);
    if (row >= (size_t)a.rows) return;
    if (a.mask && !a.mask[row]) {
        if (lane < a.topk) {
            a.inds[row * a.topk + lane] = 0xFFFFFFFFu;
            a.scores[row * a.topk + lane] = 0.f;
        }
        return;
    }
    route_row<PER, DT>(a, row, lane);
}

hipError_t run_route(const RouteArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)(((long)a.rows + RT_THREADS / 64 - 1) / (RT_THREADS / 64));
    return with_dtype(a.dtype, [&](auto DT) {
        constexpr int dt = decltype(DT)::value;
        auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(grid), dim3(RT_THREADS), 0, s, a); };
        if (a.experts <= 64) go(route_kernel<1, dt>);
        else if (a.experts <= 128) go(route_kernel<2, dt>);
        else if (a.experts <= 256) go(route_kernel<4, dt>);
        else if (a.experts <= 512) go(route_kernel<8, dt>);
        else go(route_kernel<16, dt>);
        return hipGetLastError();
    });
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
