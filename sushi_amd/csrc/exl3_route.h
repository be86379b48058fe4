// The choice of experts: kernels, instantiated for one type of logits by each exl3_route_*.hip.  With x a row of logits,
// p = softmax(x) or sigmoid(x) and c = p + bias:
//   of G groups of E / G experts the `taken` with the largest value (the sum of a group's one or two largest c),
//   of their experts the k with the largest c, listed in falling order, equal ones by their number,
//   score_i = scale p_i / (renorm ? sum over the picks of p : 1).
// Without bias, and with one group or a group's largest c as its value, the order of c is the order of x.  A logit of -inf
// takes its expert out; so do a bias of -inf or NaN, a NaN logit and, under softmax, +inf, and the last two make the row's
// scores NaN.  Slots that no expert is left for, and all slots of a row that `mask` leaves out, hold 0xFFFFFFFF and 0.
#pragma once
#include "exl3_router.h"
#include "exl3_vec.h"

namespace exl3 {

constexpr int RT_THREADS = 256;
constexpr int RT_WAVES = RT_THREADS / 64;
constexpr int NO_EXPERT = 0x7FFFFFFF;

// The value of lane (lane ^ H) where the lanes that differ below bit H hold the same: the mirror of 8 or 16 lanes then serves
// for the exchange by 4 or 8.
template <int H>
__device__ __forceinline__ int xor_lane_int(int v) {
    if constexpr (H < 4) return __float_as_int(xor_lane_row<H>(__int_as_float(v)));
    else if constexpr (H == 4) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, false);
    else if constexpr (H == 8) return __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, false);
    else return __shfl_xor(v, H);
}

// The better of two candidates: the larger value, of equal ones the lower number (NO_EXPERT, with -inf, is worse than any).
__device__ __forceinline__ bool better(double c, int i, double d, int j) { return c > d || (c == d && i < j); }

// The best of the wave's candidates, in every lane.
template <int H>
__device__ __forceinline__ void best_step(double &c, int &i) {
    const double d = __hiloint2double(xor_lane_int<H>(__double2hiint(c)), xor_lane_int<H>(__double2loint(c)));
    const int j = xor_lane_int<H>(i);
    const bool take = better(d, j, c, i);
    c = take ? d : c;
    i = take ? j : i;
}
__device__ __forceinline__ void wave_best(double &c, int &i) {
    best_step<1>(c, i);
    best_step<2>(c, i);
    best_step<4>(c, i);
    best_step<8>(c, i);
    best_step<16>(c, i);
    best_step<32>(c, i);
}

// The score's part of pick x before the sum: p for a score that keeps its value, else p over a factor that the row's picks
// share (`top`: their largest x or min(x, 0)), so that far negative logits keep their ratios.
__device__ __forceinline__ float pick_weight(const RouteArgs &a, float x, float top, float row_max, float inv_den) {
    if (!a.sigmoid) return a.renorm ? expf(x - top) : expf(x - row_max) * inv_den;
    const float e = expf(-fabsf(x));
    if (a.renorm) return expf(fminf(x, 0.f) - top) / (1.f + e);
    return (x >= 0.f ? 1.f : e) / (1.f + e);
}

// A row by one wave, lane l holding experts l, l + 64, ...; everything that decides in 64 bits.  buf: 64 PER values of the
// wave's, with groups.
template <int PER, int DT>
__device__ __forceinline__ void route_row(const RouteArgs &a, size_t row, int lane, double *buf) {
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
    if (a.groups > 1) {
        // a lane a group
        const int size = a.experts / a.groups;
#pragma unroll
        for (int i = 0; i < PER; i++) buf[lane + 64 * i] = (out >> i) & 1u ? -INFINITY : c[i];
        wave_order();
        double c1 = -INFINITY, c2 = -INFINITY;
        const int g0 = min(lane, a.groups - 1) * size;
        for (int j = 0; j < size; j++) {
            const double v = buf[g0 + j];
            c2 = v > c1 ? c1 : v > c2 ? v : c2;
            c1 = v > c1 ? v : c1;
        }
        const double worth = lane >= a.groups ? -INFINITY : a.group_top == 2 && c2 > -INFINITY ? c1 + c2 : c1;
        wave_order();
        int ahead = 0;
        for (int g = 0; g < a.groups; g++) {
            const double w = __shfl(worth, g);
            ahead += better(w, g, worth, lane) ? 1 : 0;
        }
        const uint64_t open = __ballot(ahead < a.taken && worth > -INFINITY);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int g = min(lane + 64 * i, a.experts - 1) / size;
            out |= (open >> g) & 1 ? 0u : 1u << i;
        }
    }
    int mine = NO_EXPERT;
    for (int j = 0; j < a.topk; j++) {
        double bc = -INFINITY;
        int bi = NO_EXPERT;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane + 64 * i;
            const bool take = !((out >> i) & 1u) && better(c[i], e, bc, bi);
            bc = take ? c[i] : bc;
            bi = take ? e : bi;
        }
        wave_best(bc, bi);
        if (bi == NO_EXPERT) break;
        out |= (bi & 63) == lane ? 1u << (bi >> 6) : 0u;
        mine = lane == j ? bi : mine;
    }
    const bool has = mine != NO_EXPERT;
    const float px = has ? load_act<DT>(a.logits, at + mine) : -INFINITY;
    const float top = group_max<64>(a.sigmoid ? fminf(px, 0.f) : px);
    float w = has ? pick_weight(a, px, top, mx, 1.f / (float)den) : 0.f;
    if (a.renorm) {
        const float sum = group_sum<64>(w);
        w = has ? w / sum : 0.f;
    }
    if (lane < a.topk) {
        a.inds[row * a.topk + lane] = has ? (uint32_t)mine : 0xFFFFFFFFu;
        a.scores[row * a.topk + lane] = bad ? NAN : w * a.scale;
    }
}

// More than eight picks (or more units than the lists hold): a wave a row.
template <int PER, int DT>
__global__ __launch_bounds__(RT_THREADS) void route_kernel(RouteArgs a) {
    __shared__ double buf[RT_WAVES][64 * PER];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t row = (size_t)blockIdx.x * RT_WAVES + wave;
    if (row >= (size_t)a.rows) return;
    if (a.mask && !a.mask[row]) {
        if (lane < a.topk) {
            a.inds[row * a.topk + lane] = 0xFFFFFFFFu;
            a.scores[row * a.topk + lane] = 0.f;
        }
        return;
    }
    route_row<PER, DT>(a, row, lane, buf[wave]);
}

// ---------------------------------------------------------------------------------------------------------------
// Up to eight picks, several rows a wave.  A row is held by L lanes in units of eight experts, unit u = i L + l the i-th of lane l;
// a unit's experts are one group's (a group's last unit may be short).  Each lane sorts its units' keys and merges them into
// its best T, then log2(L) merges with other lanes leave the row's best T in every lane.
//
// A key is 32 bits: a value and, in the low bits, the complement of its expert's number, so a comparator of a sorting network
// is one maximum and one minimum of integers.  (A whole f32 above a number, as an f64, costs four times as much a comparator:
// 65521 rows of 256 bf16 logits 23.6 us.)
//   EXACT: the choice is by 16-bit logits, whose f32 bits leave the low ones free; the keys' order is the choice's.
//   Otherwise a key holds M - v, M the row's largest value, as a float of 5 exponent bits (2^-20 .. 2^12) and what mantissa is
//   left (18 bits for 256 experts).  Where two values that decide lie closer than that or than v's own f32 error tells, the
//   wave takes the row again in 64 bits.
__device__ __forceinline__ void comparator(int &a, int &b) {
    const int hi = max(a, b), lo = min(a, b);
    a = hi;
    b = lo;
}
// Into falling order: eight by the network of 19 comparators in 6 steps, four by 5 in 3.
__device__ __forceinline__ void sort_keys(int (&k)[8]) {
    constexpr int net[19][2] = {{0, 2}, {1, 3}, {4, 6}, {5, 7}, {0, 4}, {1, 5}, {2, 6}, {3, 7}, {0, 1}, {2, 3},
                                {4, 5}, {6, 7}, {2, 4}, {3, 5}, {1, 4}, {3, 6}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
    for (int i = 0; i < 19; i++) comparator(k[net[i][0]], k[net[i][1]]);
}
__device__ __forceinline__ void sort_keys(int (&k)[4]) {
    comparator(k[0], k[2]);
    comparator(k[1], k[3]);
    comparator(k[0], k[1]);
    comparator(k[2], k[3]);
    comparator(k[1], k[2]);
}
// The T largest of two falling lists, falling: the maxima of one list and the other backwards rise and then fall or the other
// way round, which log2(T) steps sort.
template <int T>
__device__ __forceinline__ void merge_keys(int (&k)[T], const int (&o)[T]) {
#pragma unroll
    for (int i = 0; i < T; i++) k[i] = max(k[i], o[T - 1 - i]);
#pragma unroll
    for (int d = T / 2; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i < T; i++)
            if (!(i & d)) comparator(k[i], k[i | d]);
}
template <int H, int T>
__device__ __forceinline__ void merge_lanes(int (&k)[T]) {
    int o[T];
#pragma unroll
    for (int i = 0; i < T; i++) o[i] = xor_lane_int<H>(k[i]);
    merge_keys(k, o);
}

// Whether any of a row's L lanes holds true.
template <int L>
__device__ __forceinline__ bool group_any(bool v) {
    const uint64_t all = __ballot(v);
    if constexpr (L == 64) return all != 0;
    else return (all >> (threadIdx.x & 63 & ~(L - 1))) & ((uint64_t(1) << (L & 63)) - 1);
}

// c in f32 is within half of this of its 64-bit value.  sigmoid: exp2's argument is off by 2^-23 |x|, which moves p by
// p (1 - p) |x| 2^-23 < 2^-25, exp2, the sum and rcp move it by at most 2^-23 p each and less where p is small; softmax: the
// row's sum of up to 1024 terms and its exps are within 2^-18 of themselves, as in the balance loss, and every p is below the
// largest, 1 / den; the sum with the bias 2^-24 of itself.
__device__ __forceinline__ float near_of(const RouteArgs &a, float inv_den, float c) {
    return (a.sigmoid ? 0x1p-21f : 0x1p-17f * inv_den) + 0x1p-22f * c;
}

// M - v as 31 bits, and back (to its truncation): 0 below 2^-20, 0x7FFFFFFF for an expert that is out.
constexpr uint32_t kDistBase = 107u << 23, kDistOut = (1u << 28) - 1;
template <int ID_BITS>  // (of which a key keeps 28 - (ID_BITS - 3))
__device__ __forceinline__ uint32_t dist_bits(float d) {
    return min(__builtin_elementwise_sub_sat(__float_as_uint(d), kDistBase), kDistOut - (1u << (ID_BITS - 3)));
}
__device__ __forceinline__ float bits_dist(uint32_t b) { return b == 0 ? 0.f : __uint_as_float(b + kDistBase); }

template <int L, int NU, int T, int DT, bool BY_LOGIT, bool GROUPED>
__global__ __launch_bounds__(RT_THREADS) void route_lists_kernel(RouteArgs a) {
    constexpr int ROWS = 64 / L, PER = (L * NU * 8 + 63) / 64;
    constexpr bool EXACT = BY_LOGIT && DT != DT_F32;
    constexpr int ID_BITS = L * NU * 8 <= 64 ? 6 : L * NU * 8 <= 128 ? 7 : L * NU * 8 <= 256 ? 8 : L * NU * 8 <= 512 ? 9 : 10;
    constexpr int ID = (1 << ID_BITS) - 1;  // numbers are units' places, 8 u + q
    constexpr float LOG2E = 1.4426950408889634f;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & (L - 1), grp = lane / L;
    __shared__ __align__(16) float bias_lds[BY_LOGIT ? 4 : L * NU * 8];
    __shared__ float2 unit_top[GROUPED ? RT_WAVES : 1][GROUPED ? ROWS : 1][GROUPED ? L * NU + 1 : 1];
    __shared__ float worth_lds[GROUPED ? RT_WAVES : 1][GROUPED ? ROWS : 1][GROUPED ? kRouteMaxGroups + 1 : 1];
    __shared__ double buf[GROUPED && !EXACT ? RT_WAVES : 1][GROUPED && !EXACT ? 64 * PER : 1];
    const int size = a.experts / a.groups, units = (size + 7) / 8;
    auto first_of = [&](int u) { return GROUPED ? u / units * size + u % units * 8 : u * 8; };
    auto count_of = [&](int u) {
        const int left = GROUPED ? (u < a.groups * units ? size - u % units * 8 : 0) : size - u * 8;
        return max(0, min(8, left));
    };
    int first[NU], n[NU];  // a unit's first expert and how many it holds
#pragma unroll
    for (int i = 0; i < NU; i++) {
        first[i] = first_of(i * L + l);
        n[i] = count_of(i * L + l);
    }
    if constexpr (!BY_LOGIT) {
        for (int s = threadIdx.x; s < L * NU * 8; s += RT_THREADS) {
            const bool is = (s & 7) < count_of(s / 8);
            const float b = is && a.bias ? a.bias[first_of(s / 8) + (s & 7)] : 0.f;
            // (NaN is out of the choice; what passes 2^125 goes by 64 bits where it decides, and adds up in f32)
            bias_lds[s] = b > -INFINITY ? fminf(fmaxf(b, -0x1p125f), 0x1p125f) : -INFINITY;
        }
        __syncthreads();
    }
    const int bad_class = a.sigmoid ? 0x003 : 0x203;  // NaN; under softmax +inf too
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * RT_WAVES * ROWS;
    for (size_t r0 = ((size_t)blockIdx.x * RT_WAVES + wave) * ROWS; r0 < rows; r0 += step) {
        const size_t r = r0 + grp;
        const bool in = r < rows, live = in && (!a.mask || a.mask[in ? r : 0] != 0);
        const char *row = static_cast<const char *>(a.logits) + (in ? r : r0) * a.experts * (DT == DT_F32 ? 4 : 2);
        Raw8<DT> raw[NU];
#pragma unroll
        for (int i = 0; i < NU; i++) {
            if (n[i] > 0 && first[i] + 8 <= a.experts) raw[i].load(elem<DT>(row, first[i]));
            else raw[i].load_some(elem<DT>(row, first[i]), n[i]);
        }
#pragma unroll
        for (int i = 0; i < NU; i++)
            if (n[i] < 8) raw[i].keep(n[i]);  // -inf past a unit's experts
        // the values that the choice goes by, -inf for an expert that is out of it
        float v[NU][8], mx = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < NU; i++)
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const float x = raw[i].get(q);
                const bool nan = __builtin_amdgcn_classf(x, bad_class);
                bad |= nan;
                v[i][q] = nan ? -INFINITY : x;
                mx = fmaxf(mx, v[i][q]);
            }
        bad = group_any<L>(bad);
        float inv = 1.f;
        const bool whole = !a.sigmoid && !(BY_LOGIT && a.renorm);  // the softmax over the row
        if (whole || !EXACT) {
            mx = group_max<L>(mx);
            mx = mx == -INFINITY ? 0.f : mx;
        }
        float top_v = mx;  // the largest value
        if (whole || !BY_LOGIT) {
            float den = 0.f;
            if (!BY_LOGIT) top_v = -INFINITY;
            const float by = a.sigmoid ? -LOG2E : LOG2E, from = a.sigmoid ? 0.f : mx;
#pragma unroll
            for (int i = 0; i < NU; i++)
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float x = v[i][q], e = __builtin_amdgcn_exp2f(by * (x - from));
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
                for (int i = 0; i < NU; i++) {
                    const float4 *b = reinterpret_cast<const float4 *>(bias_lds + (i * L + l) * 8);
                    const float4 lo = b[0], hi = b[1];
                    const float bias[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        v[i][q] = v[i][q] * p + bias[q];
                        top_v = fmaxf(top_v, v[i][q]);
                    }
                }
                top_v = group_max<L>(top_v);
                top_v = top_v == -INFINITY ? 0.f : top_v;
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
                    m2 = __builtin_amdgcn_fmed3f(m1, m2, v[i][q]);
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
        int best[T];
#pragma unroll
        for (int i = 0; i < NU; i++) {
            int k[T];
#pragma unroll
            for (int part = 0; part < 8 / T; part++) {
#pragma unroll
                for (int q = 0; q < T; q++) {
                    const int not_id = ~((i * L + l) * 8 + part * T + q) & ID;
                    const float x = v[i][part * T + q];
                    if constexpr (EXACT) {
                        const int b = __float_as_int(x + 0.f);  // (-0 is 0)
                        k[q] = b ^ (((b >> 31) & (0x7FFFFFFF & ~ID)) | not_id);
                    } else {
                        const uint32_t d = x == -INFINITY ? kDistOut : dist_bits<ID_BITS>(top_v - x);
                        k[q] = (int)(((~d << 3) & (0x7FFFFFFF & ~ID)) | not_id);
                    }
                }
                sort_keys(k);
                if (i == 0 && part == 0) {
#pragma unroll
                    for (int q = 0; q < T; q++) best[q] = k[q];
                } else {
                    merge_keys(best, k);
                }
            }
        }
        merge_lanes<1>(best);
        merge_lanes<2>(best);
        merge_lanes<4>(best);
        if constexpr (L > 8) merge_lanes<8>(best);
        if constexpr (L > 16) merge_lanes<16>(best);
        if constexpr (L > 32) merge_lanes<32>(best);
        // keys of experts that are out: what -inf, or kDistOut, makes
        constexpr int OUT = EXACT ? (int)(0xFF800000u ^ (0x7FFFFFFFu & ~ID)) | ID : ID;
        if constexpr (!EXACT) {
            // Two values that decide and lie close: the row goes by 64 bits.
            auto dist = [](int key) { return bits_dist((~(uint32_t)key & (0x7FFFFFFFu & ~ID)) >> 3); };
            constexpr float STEP = 1.f / (float)(1 << (26 - ID_BITS));  // two truncations, relative
            const float tol = BY_LOGIT ? 0x1p-22f * fabsf(top_v) : near_of(a, inv, fabsf(top_v));
            float last = 0.f, bound = 0.f;
#pragma unroll
            for (int i = 0; i < T; i++) {
                if (i > a.topk) continue;
                const float d = dist(best[i]);
                const bool is = best[i] > OUT;
                if (i > 0) near |= is && d * (1.f - STEP) - last <= tol + (d < 0x1p-19f ? 0x1p-20f : 0.f);
                if (i < a.topk) {
                    near |= is && d >= 0x1p11f;  // at the end of the distances
                    last = d;
                    bound = is ? d : -1.f;
                }
            }
            if (a.topk == T) {
                const float edge = top_v - (bound * (1.f + STEP) + tol + 0x1p-20f);
                int above = 0;
#pragma unroll
                for (int i = 0; i < NU; i++)
#pragma unroll
                    for (int q = 0; q < 8; q++) above += v[i][q] >= edge ? 1 : 0;
                above = (int)group_sum<L>((float)above);
                near |= above > T && bound >= 0.f;
            }
            near = group_any<L>(near) && live;
        }
        // a lane a slot: its expert and its logit
        int key = best[0];
#pragma unroll
        for (int i = 1; i < T; i++) key = (l & (T - 1)) == i ? best[i] : key;
        const bool has = l < T && l < a.topk && key > OUT;
        const int place = ~key & ID, e = GROUPED ? first_of(place >> 3) + (place & 7) : place;
        float px;
        if constexpr (EXACT) {
            const int b = (key & ~ID);
            px = __int_as_float(b ^ ((b >> 31) & (0x7FFFFFFF & ~ID)));
        } else {
            px = load_act<DT>(elem<DT>(row, has ? e : 0), 0);
        }
        px = has ? px : -INFINITY;
        const float top = group_max<T>(a.sigmoid ? fminf(px, 0.f) : px);
        float w = has ? pick_weight(a, px, top, mx, inv) : 0.f;
        if (a.renorm) {
            const float sum = group_sum<T>(w);
            w = has ? w / sum : 0.f;
        }
        if (l < a.topk && in && !near) {
            a.inds[r * a.topk + l] = has && live ? (uint32_t)e : 0xFFFFFFFFu;
            a.scores[r * a.topk + l] = !live ? 0.f : bad ? NAN : w * a.scale;
        }
        if constexpr (!EXACT) {
            uint64_t again = __ballot(near && l == 0);
            while (again) {
                const int at = __ffsll((unsigned long long)again) - 1;
                again &= again - 1;
                route_row<PER, DT>(a, r0 + at / L, lane, buf[GROUPED ? wave : 0]);
            }
        }
    }
}

template <int L, int NU, int T, int DT>
static hipError_t launch_lists(const RouteArgs &a, hipStream_t s) {
    constexpr int at_once = RT_THREADS / L;
    const long wgs = ((long)a.rows + at_once - 1) / at_once;
    const dim3 grid((unsigned)(wgs < 2048 ? wgs : 2048));
    const bool grouped = a.groups > 1, by_logit = !a.bias && (!grouped || a.group_top == 1);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(RT_THREADS), 0, s, a); };
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

template <int DT>
static hipError_t route_of_type(const RouteArgs &a, hipStream_t s) {
    const int units = a.groups * ((a.experts / a.groups + 7) / 8);
    if (a.topk <= 8 && units <= kListUnits) return a.topk <= 4 ? with_units<4, DT>(a, units, s) : with_units<8, DT>(a, units, s);
    const unsigned grid = (unsigned)(((long)a.rows + RT_WAVES - 1) / RT_WAVES);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(grid), dim3(RT_THREADS), 0, s, a); };
    if (a.experts <= 64) go(route_kernel<1, DT>);
    else if (a.experts <= 128) go(route_kernel<2, DT>);
    else if (a.experts <= 256) go(route_kernel<4, DT>);
    else if (a.experts <= 512) go(route_kernel<8, DT>);
    else go(route_kernel<16, DT>);
    return hipGetLastError();
}

}  // namespace exl3
