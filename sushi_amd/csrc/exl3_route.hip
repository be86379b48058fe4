// The choice of experts.  With x a row of logits, p = softmax(x) or sigmoid(x) and c = p + bias:
//   of G groups of E / G experts the `taken` with the largest value (the sum of a group's one or two largest c),
//   of their experts the k with the largest c, listed in falling order, equal ones by their number,
//   score_i = scale p_i / (renorm ? sum over the picks of p : 1).
// Without bias, and with one group or a group's largest c as its value, the order of c is the order of x.  A logit of -inf
// takes its expert out; so do a bias of -inf or NaN, a NaN logit and, under softmax, +inf, and the last two make the row's
// scores NaN.  Slots that no expert is left for, and all slots of a row that `mask` leaves out, hold 0xFFFFFFFF and 0.
#include "exl3_router.h"
#include "exl3_vec.h"

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

// ---------------------------------------------------------------------------------------------------------------
// Up to eight picks, many rows a wave.  A row is held by L lanes in units of eight experts, unit u = i L + l the i-th of lane l;
// a unit's experts are one group's (a group's last unit may be short).  Each lane sorts its units' values and merges them into
// its best T, then log2(L) merges with other lanes leave the row's best T in every lane.
//
// A value and its expert are one f64: the f32's bits in the high word, which order as they do in f32, and the number below, so
// that of equal values the lower number is the larger f64.  A comparator of a sorting network is then one maximum and one
// minimum, at the f64 rate that is the f32's here.
__device__ __forceinline__ double key_of(float v, int e) {
    const int hi = __float_as_int(v);
    return __hiloint2double(hi, e ^ ~(hi >> 31));
}
__device__ __forceinline__ float value_of(double key) { return __int_as_float(__double2hiint(key)); }
__device__ __forceinline__ int expert_of(double key) { return __double2loint(key) ^ ~(__double2hiint(key) >> 31); }

__device__ __forceinline__ void comparator(double &a, double &b) {
    const double hi = fmax(a, b), lo = fmin(a, b);
    a = hi;
    b = lo;
}
// Into falling order: eight by the network of 19 comparators in 6 steps, four by 5 in 3.
__device__ __forceinline__ void sort_keys(double (&k)[8]) {
    constexpr int net[19][2] = {{0, 2}, {1, 3}, {4, 6}, {5, 7}, {0, 4}, {1, 5}, {2, 6}, {3, 7}, {0, 1}, {2, 3},
                                {4, 5}, {6, 7}, {2, 4}, {3, 5}, {1, 4}, {3, 6}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
    for (int i = 0; i < 19; i++) comparator(k[net[i][0]], k[net[i][1]]);
}
__device__ __forceinline__ void sort_keys(double (&k)[4]) {
    comparator(k[0], k[2]);
    comparator(k[1], k[3]);
    comparator(k[0], k[1]);
    comparator(k[2], k[3]);
    comparator(k[1], k[2]);
}
// The T largest of two falling lists, falling: the maxima of one list and the other backwards rise and then fall or the other
// way round, which log2(T) steps sort.
template <int T>
__device__ __forceinline__ void merge_keys(double (&k)[T], const double (&o)[T]) {
#pragma unroll
    for (int i = 0; i < T; i++) k[i] = fmax(k[i], o[T - 1 - i]);
#pragma unroll
    for (int d = T / 2; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i < T; i++)
            if (!(i & d)) comparator(k[i], k[i | d]);
}

template <int H>
__device__ __forceinline__ int xor_lane_int(int v) {
    if constexpr (H < 4) return __float_as_int(xor_lane_row<H>(__int_as_float(v)));
    // (quads hold one list by then, so the mirror of 8 or 16 lanes serves for the exchange by 4 or 8)
    else if constexpr (H == 4) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, false);
    else if constexpr (H == 8) return __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, false);
    else return __shfl_xor(v, H);
}
template <int H, int T>
__device__ __forceinline__ void merge_lanes(double (&k)[T]) {
    double o[T];
#pragma unroll
    for (int i = 0; i < T; i++) o[i] = __hiloint2double(xor_lane_int<H>(__double2hiint(k[i])), xor_lane_int<H>(__double2loint(k[i])));
    merge_keys(k, o);
}

// The sum over a row's L lanes, and whether any of them holds true.
template <int L>
__device__ __forceinline__ bool group_any(bool v) {
    const uint64_t all = __ballot(v);
    if constexpr (L == 64) return all != 0;
    else return (all >> (threadIdx.x & 63 & ~(L - 1))) & ((uint64_t(1) << L) - 1);
}

// c in f32 is within half of this of its 64-bit value.  sigmoid: the exponent's argument is off by 2^-23 |x|, which moves p by
// p (1 - p) |x| 2^-23 < 2^-25, its exp2 and rcp an ulp each, with room 2^-21; softmax: the row's sum of up to 1024 terms and
// its exps are within 2^-18 of themselves, as in the balance loss, and every p is below the largest, 1 / den; the sum with the
// bias 2^-24 of itself.
__device__ __forceinline__ float near_of(const RouteArgs &a, float inv_den, float c) {
    return (a.sigmoid ? 0x1p-20f : 0x1p-17f * inv_den) + 0x1p-22f * c;
}

constexpr int RL_THREADS = 256;

template <int L, int NU, int T, int DT, bool BY_LOGIT, bool GROUPED>
__global__ __launch_bounds__(RL_THREADS) void route_lists_kernel(RouteArgs a) {
    constexpr int ROWS = 64 / L, WAVES = RL_THREADS / 64, PER = (L * NU * 8 + 63) / 64;
    constexpr float LOG2E = 1.4426950408889634f;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & (L - 1), grp = lane / L;
    __shared__ __align__(16) float bias_lds[BY_LOGIT ? 1 : L * NU * 8];
    __shared__ float2 unit_top[GROUPED ? WAVES : 1][GROUPED ? ROWS : 1][GROUPED ? L * NU + 1 : 1];
    __shared__ float worth_lds[GROUPED ? WAVES : 1][GROUPED ? ROWS : 1][GROUPED ? kRouteMaxGroups + 1 : 1];
    const int size = a.experts / a.groups, units = (size + 7) / 8;
    int first[NU], n[NU];  // a unit's first expert and how many it holds
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int u = i * L + l, g = GROUPED ? u / units : 0, part = u - g * units;
        first[i] = g * size + part * 8;
        n[i] = g < a.groups ? max(0, min(8, size - part * 8)) : 0;
    }
    if constexpr (!BY_LOGIT) {
        if (wave == 0 && grp == 0)
#pragma unroll
            for (int i = 0; i < NU; i++)
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float b = q < n[i] && a.bias ? a.bias[first[i] + q] : 0.f;
                    // (NaN is out of the choice; what passes 2^125 goes by 64 bits where it decides, and adds up in f32)
                    bias_lds[(i * L + l) * 8 + q] = b > -INFINITY ? fminf(fmaxf(b, -0x1p125f), 0x1p125f) : -INFINITY;
                }
        __syncthreads();
    }
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * WAVES * ROWS;
    for (size_t r0 = ((size_t)blockIdx.x * WAVES + wave) * ROWS; r0 < rows; r0 += step) {
        const size_t r = r0 + grp;
        const bool in = r < rows, live = in && (!a.mask || a.mask[in ? r : 0] != 0);
        const char *row = static_cast<const char *>(a.logits) + (in ? r : r0) * a.experts * (DT == DT_F32 ? 4 : 2);
        Raw8<DT> raw[NU];
#pragma unroll
        for (int i = 0; i < NU; i++) {
            if (first[i] + 8 <= a.experts) raw[i].load(elem<DT>(row, first[i]));
            else raw[i].load_some(elem<DT>(row, first[i]), n[i]);
        }
        // the values that the choice goes by, -inf for an expert that is out of it
        float v[NU][8], mx = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < NU; i++)
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const float x = raw[i].get(q) + 0.f;  // (-0 is 0)
                const bool nan = x != x || (!a.sigmoid && x == INFINITY);
                bad |= nan && q < n[i];
                v[i][q] = q < n[i] && !nan ? x : -INFINITY;
                mx = fmaxf(mx, v[i][q]);
            }
        bad = group_any<L>(bad);
        float inv = 1.f;
        const bool whole = !a.sigmoid && !(BY_LOGIT && a.renorm);  // the softmax over the row
        if (whole || !BY_LOGIT) {
            mx = group_max<L>(mx);
            mx = mx == -INFINITY ? 0.f : mx;
            float den = 0.f;
#pragma unroll
            for (int i = 0; i < NU; i++)
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float x = v[i][q];
                    const float e = __builtin_amdgcn_exp2f(a.sigmoid ? -LOG2E * x : LOG2E * (x - mx));
                    den += e;
                    if constexpr (!BY_LOGIT) v[i][q] = x == -INFINITY ? x : a.sigmoid ? rcp(1.f + e) : e;
                }
            if (whole) {
                den = group_sum<L>(den);
                inv = rcp(den);
            }
            if constexpr (!BY_LOGIT) {
                const float p = a.sigmoid ? 1.f : inv;
#pragma unroll
                for (int i = 0; i < NU; i++)
#pragma unroll
                    for (int q = 0; q < 8; q++) v[i][q] = v[i][q] * p + bias_lds[(i * L + l) * 8 + q];
            }
        }
        bool near = false;
        if constexpr (GROUPED) {
            // each unit's two largest, each group's, its place among the groups
#pragma unroll
            for (int i = 0; i < NU; i++) {
                float m1 = v[i][0], m2 = -INFINITY;
#pragma unroll
                for (int q = 1; q < 8; q++) {
                    m2 = fmaxf(m2, fminf(m1, v[i][q]));
                    m1 = fmaxf(m1, v[i][q]);
                }
                unit_top[wave][grp][i * L + l] = float2{m1, m2};
            }
            wave_order();
            for (int g = l; g < a.groups; g += L) {
                float m1 = -INFINITY, m2 = -INFINITY;
                for (int u = g * units; u < (g + 1) * units; u++) {
                    const float2 o = unit_top[wave][grp][u];
                    m2 = fmaxf(fmaxf(m2, o.y), fminf(m1, o.x));
                    m1 = fmaxf(m1, o.x);
                }
                worth_lds[wave][grp][g] = a.group_top == 2 && m2 > -INFINITY ? m1 + m2 : m1;
            }
            wave_order();
            uint64_t open = 0;
            for (int g0 = 0; g0 < a.groups; g0 += L) {
                const int g = g0 + l;
                const float w = g < a.groups ? worth_lds[wave][grp][g] : -INFINITY;
                const float tol = BY_LOGIT ? 0.f : near_of(a, inv, fabsf(w)) * 2.f;
                int ahead = 0, surely = 0, maybe = 0;
                for (int o = 0; o < a.groups; o++) {
                    const float x = worth_lds[wave][grp][o];
                    ahead += x > w || (x == w && o < g) ? 1 : 0;
                    if constexpr (!BY_LOGIT) {
                        surely += x > w + tol ? 1 : 0;
                        maybe += x >= w - tol && o != g ? 1 : 0;
                    }
                }
                const bool is = g < a.groups && w > -INFINITY;
                if constexpr (!BY_LOGIT) near |= is && surely < a.taken && maybe >= a.taken;
                const uint64_t b = __ballot(is && ahead < a.taken);
                open |= ((b >> (lane & ~(L - 1))) & (L == 64 ? ~uint64_t(0) : (uint64_t(1) << (L & 63)) - 1)) << g0;
            }
            wave_order();
#pragma unroll
            for (int i = 0; i < NU; i++) {
                const bool is = n[i] > 0 && (open >> min((i * L + l) / units, 63)) & 1;
#pragma unroll
                for (int q = 0; q < 8; q++) v[i][q] = is ? v[i][q] : -INFINITY;
            }
        }
        double best[T];
#pragma unroll
        for (int i = 0; i < NU; i++) {
            double k[T];
#pragma unroll
            for (int part = 0; part < 8 / T; part++) {
#pragma unroll
                for (int q = 0; q < T; q++) k[q] = key_of(v[i][part * T + q], first[i] + part * T + q);
                sort_keys(k);
                if (i == 0 && part == 0) {
#pragma unroll
                    for (int q = 0; q < T; q++) best[q] = k[q];
                } else {
                    merge_keys(best, k);
                }
            }
        }
        if constexpr (L > 1) merge_lanes<1>(best);
        if constexpr (L > 2) merge_lanes<2>(best);
        if constexpr (L > 4) merge_lanes<4>(best);
        if constexpr (L > 8) merge_lanes<8>(best);
        if constexpr (L > 16) merge_lanes<16>(best);
        if constexpr (L > 32) merge_lanes<32>(best);
        if constexpr (!BY_LOGIT) {
            // Two values that decide and lie close: the row goes by 64 bits.
            float last = value_of(best[0]);
            const float big = fabsf(last);
            float gap = INFINITY;
#pragma unroll
            for (int i = 1; i < T; i++) {
                const float x = value_of(best[i]);
                gap = i <= a.topk ? fminf(gap, last - x) : gap;  // (NaN, of two experts that are out, is no gap)
                last = i < a.topk ? x : last;
            }
            const float tol = near_of(a, inv, fmaxf(big, last > -INFINITY ? fabsf(last) : 0.f));
            near |= gap <= tol;
            if (a.topk == T) {
                int above = 0;
#pragma unroll
                for (int i = 0; i < NU; i++)
#pragma unroll
                    for (int q = 0; q < 8; q++) above += v[i][q] >= last - tol ? 1 : 0;
                above = (int)group_sum<L>((float)above);
                near |= above > T && last > -INFINITY;
            }
            near = group_any<L>(near) && live;
        }
        // a lane a slot: its expert and its logit
        int e = -1;
        float px = -INFINITY;
#pragma unroll
        for (int i = 0; i < T; i++) {
            const bool me = (l & (T - 1)) == i;
            const float c = value_of(best[i]);
            e = me ? (c > -INFINITY && i < a.topk ? expert_of(best[i]) : -1) : e;
            px = me ? c : px;
        }
        const bool has = e >= 0 && l < T;
        if constexpr (!BY_LOGIT) px = has ? load_act<DT>(elem<DT>(row, e), 0) : -INFINITY;
        px = has ? px : -INFINITY;
        const float top = group_max<(T < L ? T : L)>(a.sigmoid ? fminf(px, 0.f) : px);
        float w = has ? pick_weight(a, px, top, mx, 1.f) * (a.sigmoid || a.renorm ? 1.f : inv) : 0.f;
        if (a.renorm) {
            const float sum = group_sum<(T < L ? T : L)>(w);
            w = has ? w / sum : 0.f;
        }
        if (l < a.topk && in && !near) {
            a.inds[r * a.topk + l] = has && live ? (uint32_t)e : 0xFFFFFFFFu;
            a.scores[r * a.topk + l] = !live ? 0.f : bad ? NAN : w * a.scale;
        }
        if constexpr (!BY_LOGIT) {
            uint64_t again = __ballot(near && l == 0);
            while (again) {
                const int at = __ffsll((unsigned long long)again) - 1;
                again &= again - 1;
                route_row<PER, DT>(a, r0 + at / L, lane);
            }
        }
    }
}

template <int L, int NU, int T, int DT>
static hipError_t launch_lists(const RouteArgs &a, hipStream_t s) {
    constexpr int at_once = RL_THREADS / L;
    const long wgs = ((long)a.rows + at_once - 1) / at_once;
    const dim3 grid((unsigned)(wgs < 2048 ? wgs : 2048));
    const bool grouped = a.groups > 1, by_logit = !a.bias && (!grouped || a.group_top == 1);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(RL_THREADS), 0, s, a); };
    if (by_logit) grouped ? go(route_lists_kernel<L, NU, T, DT, true, true>) : go(route_lists_kernel<L, NU, T, DT, true, false>);
    else grouped ? go(route_lists_kernel<L, NU, T, DT, false, true>) : go(route_lists_kernel<L, NU, T, DT, false, false>);
    return hipGetLastError();
}

template <int T, int DT>
static hipError_t with_units(const RouteArgs &a, int units, hipStream_t s) {
    if (units <= 8) return launch_lists<8, 1, T, DT>(a, s);
    if (units <= 16) return launch_lists<8, 2, T, DT>(a, s);
    if (units <= 32) return launch_lists<8, 4, T, DT>(a, s);
    if (units <= 64) return launch_lists<16, 4, T, DT>(a, s);
    return launch_lists<32, 4, T, DT>(a, s);
}

constexpr int kListUnits = 128;

hipError_t run_route(const RouteArgs &a, hipStream_t s) {
    const int units = a.groups * ((a.experts / a.groups + 7) / 8);
    return with_dtype(a.dtype, [&](auto DT) {
        constexpr int dt = decltype(DT)::value;
        if (a.topk <= 8 && units <= kListUnits) return a.topk <= 4 ? with_units<4, dt>(a, units, s) : with_units<8, dt>(a, units, s);
        const unsigned grid = (unsigned)(((long)a.rows + RT_THREADS / 64 - 1) / (RT_THREADS / 64));
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
