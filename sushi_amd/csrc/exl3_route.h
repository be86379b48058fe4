// The choice of experts: kernels, instantiated for one type of logits by each exl3_route_*.hip.  With x a row of logits,
// p = softmax(x) or sigmoid(x) and c = p + bias:
//   of G groups of E / G experts the `taken` with the largest value (the sum of a group's one or two largest c),
//   of their experts the k with the largest c, listed in falling order, equal ones by their number,
//   score_i = scale p_i / (renorm ? sum over the picks of p : 1).
// Without bias, or with one that is the same for every expert, the experts' order is that of x, and the groups' too where their
// value is one c.  A logit of -inf takes its expert out; so do a bias of -inf or NaN, a NaN logit and, under softmax, +inf, and
// the last two make the row's scores NaN.  Slots that no expert is left for, and all slots of a row that `mask` leaves out, hold
// 0xFFFFFFFF and 0.
#pragma once
#include "exl3_router.h"
#include "exl3_vec.h"

namespace exl3 {

constexpr int RT_THREADS = 256;
constexpr int RT_WAVES = RT_THREADS / 64;
constexpr int kListUnits = 128;  // units of eight experts that the lists serve
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

// exp(x) for x <= 0 to about an ulp: exp2 of the product with log2 e in two f32, as Cody and Waite split a constant, times what
// the product's rounding left out.
__device__ __forceinline__ float exp_near(float x) {
    constexpr float HI = 1.44269504f, LO = 1.92596299e-8f, LN2 = 0.693147181f;
    const float n = x * HI, rest = fmaf(x, HI, -n) + x * LO, e = __builtin_amdgcn_exp2f(n);
    return x > -104.f ? fmaf(e, rest * LN2, e) : 0.f;  // (the rest of -inf is NaN)
}
// a / b for b of f32's middle range: a reciprocal and one Newton step, by the quotient's remainder.
__device__ __forceinline__ float quotient(float a, float b) {
    const float r = rcp(b), q = a * r;
    return fmaf(fmaf(-q, b, a), r, q);
}

// The score's part of pick x before the sum: p for a score that keeps its value, else p over a factor that the row's picks
// share (`top`: their largest x or min(x, 0)), so that far negative logits keep their ratios.
__device__ __forceinline__ float pick_weight(const RouteArgs &a, float x, float top, float row_max, float inv_den) {
    if (!a.sigmoid) return a.renorm ? exp_near(x - top) : exp_near(x - row_max) * inv_den;
    const float e = exp_near(-fabsf(x));
    if (a.renorm) return quotient(exp_near(fminf(x, 0.f) - top), 1.f + e);
    return quotient(x >= 0.f ? 1.f : e, 1.f + e);
}

// A row's values by one wave in 64 bits, lane l taking experts l, l + 64, ...: x or c, -inf for an expert that is out by its logit
// or its bias.  In `buf`, the wave's.
struct RowInfo {
    float mx, inv;  // the softmax's
    bool bad;
};
template <int DT>
__device__ __forceinline__ RowInfo row_values(const RouteArgs &a, size_t row, int lane, double *buf, bool by_logit) {
    const size_t at = row * a.experts;
    const bool whole = !a.sigmoid && !(by_logit && a.renorm);
    bool bad = false;
    float mx = -INFINITY;
#pragma unroll 2
    for (int e = lane; e < a.experts; e += 64) {
        const float x = load_act<DT>(a.logits, at + e);
        const bool nan = x != x || (!a.sigmoid && x == INFINITY);
        bad |= nan;
        mx = fmaxf(mx, nan ? -INFINITY : x);
        buf[e] = nan ? -INFINITY : (double)x;
    }
    mx = group_max<64>(mx);
    mx = mx == -INFINITY ? 0.f : mx;
    double den = 0.;
    if (!by_logit || whole) {
#pragma unroll 2
        for (int e = lane; e < a.experts; e += 64) {
            const double x = buf[e], y = exp(a.sigmoid ? -x : x - (double)mx);
            den += y;
            if (!by_logit) buf[e] = x == -INFINITY ? x : a.sigmoid ? 1. / (1. + y) : y;
        }
    }
    if (whole) {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) den += __shfl_xor(den, m);
    }
    if (!by_logit) {
        for (int e = lane; e < a.experts; e += 64) {
            const double c = buf[e];
            const float b = a.bias ? a.bias[e] : 0.f;
            // (an expert that its bias takes out still has its share of the softmax)
            const bool off = c == -INFINITY || !(b > -INFINITY);
            buf[e] = off ? -INFINITY : (whole ? c / den : c) + (double)b;
        }
    }
    return RowInfo{mx, whole ? (float)(1. / den) : 1.f, (bool)__any(bad)};
}

// Whether the bias is one finite value for every expert, or there is none.
__device__ __forceinline__ bool same_bias(const RouteArgs &a, int lane) {
    if (!a.bias) return true;
    const float first = a.bias[0];
    bool same = fabsf(first) < INFINITY;
    for (int e = lane; e < a.experts; e += 64) same &= a.bias[e] == first;
    return __all(same);
}

// A lane's pick of a row by one wave: its slot (past topk: none), its expert (NO_EXPERT: a slot without one).
template <int DT>
__device__ __forceinline__ void write_picks(const RouteArgs &a, size_t row, const RowInfo &info, int slot, int expert) {
    const bool has = slot < a.topk && expert != NO_EXPERT;
    const float px = has ? load_act<DT>(a.logits, row * a.experts + expert) : -INFINITY;
    const float top = group_max<64>(a.sigmoid ? fminf(px, 0.f) : px);
    float w = has ? pick_weight(a, px, top, info.mx, info.inv) : 0.f;
    if (a.renorm) {
        const float sum = group_sum<64>(w);
        w = has ? quotient(w, sum) : 0.f;
    }
    if (slot < a.topk) {
        a.inds[row * a.topk + slot] = has ? (uint32_t)expert : 0xFFFFFFFFu;
        a.scores[row * a.topk + slot] = info.bad ? NAN : w * a.scale;
    }
}

// A row by one wave, whatever it holds; by_logit: the experts' order is their logits'.
template <int DT>
__device__ __forceinline__ void route_row(const RouteArgs &a, size_t row, int lane, double *buf, bool by_logit) {
    const bool groups_too = by_logit && a.group_top == 1;
    RowInfo info = row_values<DT>(a, row, lane, buf, a.groups > 1 ? groups_too : by_logit);
    if (a.groups > 1) {
        // a lane a group
        const int size = a.experts / a.groups;
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
        if (by_logit && !groups_too) info = row_values<DT>(a, row, lane, buf, true);
        for (int e = lane; e < a.experts; e += 64)
            if (!((open >> (e / size)) & 1)) buf[e] = -INFINITY;
    }
    int mine = NO_EXPERT;
    for (int j = 0; j < a.topk; j++) {
        double bc = -INFINITY;
        int bi = NO_EXPERT;
        for (int e = lane; e < a.experts; e += 64) {
            const double c = buf[e];
            const bool take = c > bc;  // (of a lane's equal ones the first)
            bc = take ? c : bc;
            bi = take ? e : bi;
        }
        wave_best(bc, bi);
        if (bi == NO_EXPERT) break;
        if ((bi & 63) == lane) buf[bi] = -INFINITY;
        mine = lane == j ? bi : mine;
    }
    write_picks<DT>(a, row, info, lane, mine);
}

// A row whose groups are settled (bit g of `open`) and whose picks are all at least `least`, by one wave: the few experts that may
// be stand in a list, a lane each, which counts those ahead of its own.  False with more than a wave of them.  A sigmoid is a
// logit's own, so only those of the list are taken in 64 bits.
constexpr int kSettleLds = 64 * 4;  // the list, behind a row's values
template <int DT>
__device__ __forceinline__ bool settle_row(const RouteArgs &a, size_t row, int lane, double *buf, bool by_logit, uint64_t open,
                                           double least) {
    const bool own = a.sigmoid && !by_logit;
    RowInfo info = {0.f, 1.f, false};
    if (!own) info = row_values<DT>(a, row, lane, buf, by_logit);
    int *const list = reinterpret_cast<int *>(buf + a.experts);
    const int size = a.experts / a.groups;
    wave_order();
    int count = 0;
    bool bad = false;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
        const int e = e0 + lane, at = min(e, a.experts - 1);
        bool is = e < a.experts && ((open >> (a.groups > 1 ? at / size : 0)) & 1);
        double c = -INFINITY;
        if (own) {
            const float x = load_act<DT>(a.logits, row * a.experts + at), b = a.bias ? a.bias[at] : 0.f;
            bad |= x != x;
            // (to twice what near_of allows)
            const float near = rcp(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x)) + b;
            is = is && x > -INFINITY && b > -INFINITY && (double)near + (double)(0x1p-20f + 0x1p-21f * fabsf(near)) >= least;
        } else {
            c = buf[at];
            is = is && c >= least && c > -INFINITY;
        }
        const uint64_t who = __ballot(is);
        const int place = count + (int)__popcll(who & ((uint64_t(1) << lane) - 1));
        count += (int)__popcll(who);
        if (count > 64) return false;
        if (is) {  // (a value's place is never past its expert's)
            list[place] = e;
            if (!own) buf[place] = c;
        }
        wave_order();
    }
    const int expert = lane < count ? list[lane] : NO_EXPERT;
    double mine = -INFINITY;
    if (own) {
        info.bad = (bool)__any(bad);
        if (lane < count) mine = 1. / (1. + exp(-(double)load_act<DT>(a.logits, row * a.experts + expert))) + (double)(a.bias ? a.bias[expert] : 0.f);
    } else if (lane < count) {
        mine = buf[lane];
    }
    int ahead = 0;
    for (int i = 0; i < count; i++) {
        const double c = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(mine), i), __builtin_amdgcn_readlane(__double2loint(mine), i));
        ahead += better(c, __builtin_amdgcn_readlane(expert, i), mine, expert) ? 1 : 0;
    }
    // lanes behind the list take the slots that no expert is left for
    write_picks<DT>(a, row, info, lane < count ? ahead : lane, expert);
    return true;
}

// More than eight picks (or more units than the lists hold): a wave a row, each pick a pass over the row's values.  Bound by the
// issue of those: 65521 bf16 rows of 256 with 12 picks take 125 us by the logits, 160 with a bias, 202 with groups too.
template <int DT>
__global__ __launch_bounds__(RT_THREADS) void route_kernel(RouteArgs a) {
    extern __shared__ double row_buf[];
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
    route_row<DT>(a, row, lane, row_buf + wave * a.experts, same_bias(a, lane));
}

// ---------------------------------------------------------------------------------------------------------------
// Up to eight picks, several rows a wave.  A row is held by L lanes in units of eight experts, unit u = i L + l the i-th of lane l;
// a unit's experts are one group's (a group's last unit may be short).  Each lane sorts its units' keys and merges them into
// its best T, then log2(L) merges with other lanes leave the row's best T in every lane, and the best of the others beside them.
//
// A key is 32 bits: a value and, in the low bits, the complement of its expert's place, so a comparator of a sorting network
// is one maximum and one minimum of integers.  (A whole f32 above a number, as an f64, costs four times as much a comparator:
// 65521 rows of 256 bf16 logits 23.6 us.)  The value is
//   a 16-bit logit, whose f32 bits leave the low ones free (the keys' order is the choice's),
//   an f32 logit without its low bits (6 to 10 of them): those that share a key are put in order by the logits themselves,
//   or c in steps of the range that p and the bias span.
// Where two values of c decide and lie closer than c's steps or its f32 error tell, and where f32 logits at the edge of the picks
// share a key and differ, the wave takes the row again in 64 bits.
//
// The loops over a lane's units stay rolled: the kernel is short, so a call of few rows fetches less of it, and few registers
// leave room for more waves.
//
// Long calls are bound by the issue of vector instructions more than by their bytes: 65521 bf16 rows of 256 experts by the logits
// alone take 12.7 us, 97 instructions a row and 10.4 us of issue (7.3 for the bytes); of f32 logits 20 to 22, 111 a row, 11.8 of
// issue and 13 for the bytes; with bias and groups 32, 180 a row, 20 of issue, the rest of it the rows that go by 64 bits after the
// others and a second generation of workgroups (36 KB of LDS each).  A masked row is computed as any other.  Short calls are a
// launch and one row's latency: 6.1 us for 32 rows with bias and groups, 2.6 to 4 by the logits.
//
// The steps of c span the whole bias, so one expert far from the others leaves them few: with one at -100 / -1e4 / -1e9 the 32 us
// become 47 / 145 / 248, as more and more rows go by 64 bits.  An expert at -inf is out and costs nothing.
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
// way round, which log2(T) steps sort.  The largest of those left out goes into `next`.
template <int T>
__device__ __forceinline__ void merge_keys(int (&k)[T], const int (&o)[T], int &next) {
#pragma unroll
    for (int i = 0; i < T; i++) {
        next = max(next, min(k[i], o[T - 1 - i]));
        k[i] = max(k[i], o[T - 1 - i]);
    }
#pragma unroll
    for (int d = T / 2; d > 0; d /= 2)
#pragma unroll
        for (int i = 0; i < T; i++)
            if (!(i & d)) comparator(k[i], k[i | d]);
}
template <int H, int T>
__device__ __forceinline__ void merge_lanes(int (&k)[T], int &next) {
    int o[T];
#pragma unroll
    for (int i = 0; i < T; i++) o[i] = xor_lane_int<H>(k[i]);
    next = max(next, xor_lane_int<H>(next));
    merge_keys(k, o, next);
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

// An integer of c's steps: 0 for what is not above it, NaN too (the conversion saturates, which C++ does not say).
__device__ __forceinline__ uint32_t to_steps(float x) {
    uint32_t r;
    asm("v_cvt_u32_f32 %0, %1" : "=v"(r) : "v"(x));
    return r;
}

template <int L, int T, int DT, bool BY_LOGIT, bool GROUPED>
__global__ __launch_bounds__(RT_THREADS) void route_lists_kernel(RouteArgs a, int nu, int id_bits, int wave_lds) {
    constexpr int ROWS = 64 / L;
    constexpr float LOG2E = 1.4426950408889634f;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & (L - 1), grp = lane / L;
    extern __shared__ __align__(16) double row_buf[];  // wave_lds bytes a wave
    char *const mem = reinterpret_cast<char *>(row_buf) + wave * wave_lds;
    float *const bias_lds = reinterpret_cast<float *>(reinterpret_cast<char *>(row_buf) + RT_WAVES * wave_lds);  // behind the waves'
    __shared__ float range[RT_WAVES][3];
    const int size = a.experts / a.groups, units = (size + 7) / 8;
    const uint32_t over = (65536 + units - 1) / units;  // u / units = u over >> 16 for the units here
    auto group_of = [&](int u) { return GROUPED ? (int)(u * over >> 16) : 0; };
    auto first_of = [&](int u) { return GROUPED ? group_of(u) * (size - units * 8) + u * 8 : u * 8; };
    auto count_of = [&](int u) {
        const int g = group_of(u);
        return g < a.groups ? max(0, min(8, size - (u - g * units) * 8)) : 0;
    };
    const int id_mask = (1 << id_bits) - 1;       // a key's low bits: the complement of the expert's place, 8 u + q
    const int value_mask = 0x7FFFFFFF & ~id_mask;
    float lo = 0.f, steps = 0.f, largest = 0.f;   // c's steps: (c - lo) steps + 1; no |c| is above `largest`
    // A bias that is the same for every expert does not move the choice among experts: it goes by the logits, whose ties are ties.
    bool by_logit = BY_LOGIT;
    bool far = false;  // a bias past 2^125: keys and groups' values do not tell it from others, so every row goes by 64 bits
    if constexpr (!BY_LOGIT) {
        float least = INFINITY, most = -INFINITY;
        bool out = false;
        for (int s = threadIdx.x; s < L * nu * 8; s += RT_THREADS) {
            const bool is = (s & 7) < count_of(s / 8);
            const float b = is ? a.bias ? a.bias[first_of(s / 8) + (s & 7)] : 0.f : -INFINITY;
            out |= is && !(b > -INFINITY);
            // (NaN is out of the choice; what passes 2^125 ends there, so that sums stay in f32: see `far`)
            bias_lds[s] = b > -INFINITY ? fminf(fmaxf(b, -0x1p125f), 0x1p125f) : -INFINITY;
            least = fminf(least, b > -INFINITY ? b : INFINITY);
            most = fmaxf(most, b);
        }
        least = -group_max<64>(-least);
        most = group_max<64>(most);
        range[wave][0] = least;
        range[wave][1] = most;
        range[wave][2] = __any(out) ? 1.f : 0.f;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < RT_WAVES; w++) {
            out |= range[w][2] != 0.f;
            least = fminf(least, range[w][0]);
            most = fmaxf(most, range[w][1]);
        }
        by_logit = !out && least == most && fabsf(most) < INFINITY;
        far = least < -0x1p125f || most > 0x1p125f;
        least = fminf(fmaxf(least, -0x1p125f), 0x1p125f);
        most = fminf(fmaxf(most, -0x1p125f), 0x1p125f);
        lo = least;
        largest = fmaxf(fabsf(least), fabsf(most) + 1.f);
        steps = most >= least ? (float)((1u << (31 - id_bits)) - 16) / (1.0625f + (most - least)) : 0.f;
    }
    const bool exact = DT != DT_F32 && by_logit;      // keys that order as the choice does
    const bool groups_by_logit = BY_LOGIT || (by_logit && a.group_top == 1);
    const int bad_class = a.sigmoid ? 0x003 : 0x203;  // NaN; under softmax +inf too
    // (One set of rows a wave: in a loop over sets the compiler keeps the 64-bit path's constants in registers throughout.)
    const size_t rows = (size_t)a.rows, r0 = ((size_t)blockIdx.x * RT_WAVES + wave) * ROWS;
    if (r0 >= rows) return;
    const size_t r = r0 + grp;
    const bool in = r < rows, live = in && (!a.mask || a.mask[in ? r : 0] != 0);
    const char *row = static_cast<const char *>(a.logits) + (in ? r : r0) * a.experts * (DT == DT_F32 ? 4 : 2);
    // A vector may pass the row's end into the next rows, and its values there go; past the last row it goes by elements.
    const int reach = (int)min(rows - (in ? r : r0), (size_t)8) * a.experts;
    bool bad = false;
    // A unit's logits, -inf for experts that are out by them and past the unit's own; whether the wave has any of those.
    auto load = [&](int u, float (&v)[8]) {
        Raw8<DT> raw;
        const int first = first_of(u), n = count_of(u);
        if (n > 0 && first + 8 <= reach) raw.load(elem<DT>(row, first));
        else raw.load_some(elem<DT>(row, first), n);
        if (n < 8) raw.keep(n);
        bool odd = false;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            v[q] = raw.get(q);
            odd |= __builtin_amdgcn_classf(v[q], bad_class | 0x004);
        }
        odd = __any(odd);
        if (odd)
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const bool nan = __builtin_amdgcn_classf(v[q], bad_class);
                bad |= nan;
                v[q] = nan ? -INFINITY : v[q];
            }
        return odd;
    };
    const bool whole = !a.sigmoid && !(BY_LOGIT && a.renorm);  // the softmax over the row
    float mx = -INFINITY, inv = 1.f;
    if (whole) {
#pragma unroll 1
        for (int i = 0; i < nu; i++) {
            float v[8];
            load(i * L + l, v);
#pragma unroll
            for (int q = 0; q < 8; q++) mx = fmaxf(mx, v[q]);
        }
        mx = group_max<L>(mx);
        mx = mx == -INFINITY ? 0.f : mx;
    }
    if (whole) {
        float den = 0.f;
#pragma unroll 1
        for (int i = 0; i < nu; i++) {
            float v[8];
            load(i * L + l, v);
#pragma unroll
            for (int q = 0; q < 8; q++) den += __builtin_amdgcn_exp2f(LOG2E * (v[q] - mx));
        }
        inv = rcp(group_sum<L>(den));
    }
    // The values that the choice goes by, -inf for an expert that is out of it.
    auto values = [&](int u, float (&v)[8]) {
        float x[8];
        const bool odd = load(u, x);
        if constexpr (BY_LOGIT) {
#pragma unroll
            for (int q = 0; q < 8; q++) v[q] = x[q];
        } else {
            const float4 *b = reinterpret_cast<const float4 *>(bias_lds + u * 8);
            const float4 b0 = b[0], b1 = b[1];
            const float bias[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
            if (a.sigmoid) {
#pragma unroll
                for (int q = 0; q < 8; q++) v[q] = rcp(1.f + __builtin_amdgcn_exp2f(-LOG2E * x[q])) + bias[q];
            } else {
#pragma unroll
                for (int q = 0; q < 8; q++) v[q] = fmaf(__builtin_amdgcn_exp2f(LOG2E * (x[q] - mx)), inv, bias[q]);
            }
            if (odd)
#pragma unroll
                for (int q = 0; q < 8; q++) v[q] = x[q] == -INFINITY ? x[q] : v[q];
        }
    };
    bool near = false, near_group = far;
    uint64_t open = ~uint64_t(0);
    float *const vals = reinterpret_cast<float *>(mem) + grp * (L * nu * 8 + 8);  // (rows at different banks)
    int *const list = reinterpret_cast<int *>(mem + 2048 * nu + 32 * ROWS) + grp * a.groups;  // the open groups, in order
    int opened = 0, units_left = nu;
    if constexpr (GROUPED) {
        // each group's two largest, its place among the groups
        float *const worth = reinterpret_cast<float *>(list);
#pragma unroll 1
        for (int i = 0; i < nu; i++) {
            float v[8];
            const int u = i * L + l;
            if (groups_by_logit) load(u, v);
            else values(u, v);
            float4 *o = reinterpret_cast<float4 *>(vals + u * 8);
            o[0] = float4{v[0], v[1], v[2], v[3]};
            o[1] = float4{v[4], v[5], v[6], v[7]};
        }
        wave_order();
        for (int g = l; g < a.groups; g += L) {
            float m1 = -INFINITY, m2 = -INFINITY;
            int u = g % units;  // (lanes begin at different units, so at different banks)
#pragma unroll 1
            for (int j = 0; j < units; j++) {
                const float4 *o = reinterpret_cast<const float4 *>(vals + (g * units + u) * 8);
                const float4 v0 = o[0], v1 = o[1];
                const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    m2 = __builtin_amdgcn_fmed3f(m1, m2, v[q]);
                    m1 = fmaxf(m1, v[q]);
                }
                u = u + 1 == units ? 0 : u + 1;
            }
            worth[g] = a.group_top == 2 && m2 > -INFINITY ? m1 + m2 : m1;
        }
        wave_order();
        open = 0;
        const float tol = near_of(a, inv, largest) * 2.f;
        for (int g0 = 0; g0 < a.groups; g0 += L) {
            const int g = g0 + l;
            const float w = g < a.groups ? worth[g] : -INFINITY;
            int ahead = 0, surely = 0, maybe = 0;
            for (int o = 0; o < a.groups; o++) {
                const float x = worth[o];
                ahead += x > w || (x == w && o < g) ? 1 : 0;
                if (!groups_by_logit) {
                    surely += x > w + tol ? 1 : 0;
                    maybe += x >= w - tol && o != g ? 1 : 0;
                }
            }
            const bool is = g < a.groups && w > -INFINITY;
            if (!groups_by_logit) near_group |= is && surely < a.taken && maybe >= a.taken;
            const uint64_t b = __ballot(is && ahead < a.taken);
            open |= ((b >> (lane & ~(L - 1))) & (L == 64 ? ~uint64_t(0) : (uint64_t(1) << (L & 63)) - 1)) << g0;
        }
        wave_order();
        opened = __popcll(open);
        for (int g = l; g < a.groups; g += L)
            if ((open >> g) & 1) list[__popcll(open & ((uint64_t(1) << g) - 1))] = g;
        wave_order();
        units_left = (a.taken * units + L - 1) / L;
    }
    // The lane's i-th unit of those left, and whether there is one; its kept values; its logits, -inf for what is out.
    auto unit_of = [&](int i, int &u) {
        u = i * L + l;
        bool is = true;
        if constexpr (GROUPED) {  // the u-th unit of the open groups
            const int nth = group_of(u);
            is = nth < opened;
            u += is ? (list[nth] - nth) * units : -u;
        }
        return is;
    };
    auto kept = [&](int u, float (&v)[8]) {
        const float4 *o = reinterpret_cast<const float4 *>(vals + u * 8);
        const float4 v0 = o[0], v1 = o[1];
        v[0] = v0.x, v[1] = v0.y, v[2] = v0.z, v[3] = v0.w, v[4] = v1.x, v[5] = v1.y, v[6] = v1.z, v[7] = v1.w;
    };
    auto logits_of = [&](int u, bool is, float (&v)[8]) {
        if (GROUPED && groups_by_logit) kept(u, v);
        else load(u, v);
        if constexpr (GROUPED)
            if (!is)
#pragma unroll
                for (int q = 0; q < 8; q++) v[q] = -INFINITY;
    };
    // A logit's part of its key: its bits in the order of integers (-0 is 0), an f32's without the low ones.
    auto logit_key = [&](float v) {
        const int b = __float_as_int(v + 0.f);
        return (b ^ ((b >> 31) & value_mask)) & ~id_mask;
    };
    int best[T], next = INT32_MIN;
#pragma unroll 1
    for (int i = 0; i < units_left; i++) {
        int u;
        const bool is = unit_of(i, u);
        float v[8];
        int k8[8];
        const int not_id = ~(u * 8 + 7) & id_mask;
        if (by_logit) {
            logits_of(u, is, v);
#pragma unroll
            for (int q = 0; q < 8; q++) k8[q] = logit_key(v[q]) | not_id | (7 - q);
        } else {
            if constexpr (GROUPED) kept(u, v);
            else values(u, v);
            const float by = is ? steps : 0.f, one = is ? 1.f : 0.f;
#pragma unroll
            for (int q = 0; q < 8; q++) k8[q] = (int)(to_steps(fmaf(v[q] - lo, by, one)) << id_bits) | not_id | (7 - q);
        }
#pragma unroll
        for (int part = 0; part < 8 / T; part++) {
            int k[T];
#pragma unroll
            for (int j = 0; j < T; j++) k[j] = k8[part * T + j];
            sort_keys(k);
            if (part == 0 && i == 0) {
#pragma unroll
                for (int q = 0; q < T; q++) best[q] = k[q];
            } else {
                merge_keys(best, k, next);
            }
        }
    }
    merge_lanes<1>(best, next);
    merge_lanes<2>(best, next);
    merge_lanes<4>(best, next);
    if constexpr (L > 8) merge_lanes<8>(best, next);
    if constexpr (L > 16) merge_lanes<16>(best, next);
    if constexpr (L > 32) merge_lanes<32>(best, next);
    bad = group_any<L>(bad);
    // keys of experts that are out: what -inf or no step makes
    const int out = by_logit ? (int)(0xFF800000u ^ (uint32_t)value_mask) | id_mask : id_mask;
    // Two values of c that decide and lie close: the row goes by 64 bits.  `least`: no pick is below it.  f32 logits are out of
    // order only among those that share a key: `tied` picks, or the last pick and the next at the `edge`.
    double least = -INFINITY;
    bool tied = false, edge = false;
    if (!exact) {
        int last = 0;
        if (by_logit) {
#pragma unroll
            for (int i = 0; i <= T; i++) {
                const int key = i < T ? best[i < T ? i : 0] : next;
                const bool same = i > 0 && key > out && !((key ^ last) & ~id_mask);
                tied |= same && i < a.topk;
                edge |= same && i == a.topk;
                last = key;
            }
        } else {
            const float err = near_of(a, inv, largest);
            const int tol = (int)fminf(err * steps, 0x1p30f) + 3;
#pragma unroll
            for (int i = 0; i <= T; i++) {
                const int key = (i < T ? best[i < T ? i : 0] : next) >> id_bits;
                if (i > 0 && i <= a.topk && key > 0) near |= last - key <= tol;
                if (i == a.topk - 1 && key > 0) least = (double)lo + (double)(key - 5) / (double)steps - (double)err;
                last = key;
            }
        }
    }
    // a lane a slot: its expert and its logit
    int key = best[0], slot = l & (T - 1);
    asm volatile("" : "+v"(slot));  // (its comparisons are not kept over the rows)
#pragma unroll
    for (int i = 1; i < T; i++) key = slot == i ? best[i] : key;
    const bool has = l < T && l < a.topk && key > out;
    const int place = ~key & id_mask, e = GROUPED ? first_of(place >> 3) + (place & 7) : place;
    float px;
    if (exact) {
        const int b = key & ~id_mask;
        px = __int_as_float(b ^ ((b >> 31) & value_mask));
    } else {
        px = load_act<DT>(elem<DT>(row, has ? e : 0), 0);
    }
    px = has ? px : -INFINITY;
    int to = l;
    if constexpr (DT == DT_F32) {
        if (__any(edge)) {  // in order all the same if what shares the last pick's key is equal to it
            const float x = __shfl(px, a.topk - 1, L);
            const int shared = __shfl(key, a.topk - 1, L) & ~id_mask;
            bool other = false;
#pragma unroll 1
            for (int i = 0; i < units_left; i++) {
                int u;
                const bool is = unit_of(i, u);
                float v[8];
                logits_of(u, is, v);
#pragma unroll
                for (int q = 0; q < 8; q++) other |= logit_key(v[q]) == shared && v[q] != x;
            }
            if (edge && group_any<L>(other)) {
                near = true;
                least = __int_as_float(shared < 0 ? (shared ^ value_mask) | id_mask : shared);
            }
        }
        if (__any(tied)) {
            int ahead = 0;
            for (int j = 0; j < a.topk; j++) {
                const float x = __shfl(px, j, L);
                const int o = __shfl(e, j, L);
                ahead += x > px || (x == px && o < e) ? 1 : 0;
            }
            to = has ? ahead : l;
        }
    }
    if (!BY_LOGIT || DT == DT_F32) {
        near = group_any<L>(near || near_group) && live;
        near_group = group_any<L>(near_group);
    }
    const float top = group_max<T>(a.sigmoid ? fminf(px, 0.f) : px);
    float w = has ? pick_weight(a, px, top, mx, inv) : 0.f;
    if (a.renorm) {
        const float sum = group_sum<T>(w);
        w = has ? quotient(w, sum) : 0.f;
    }
    if (l < a.topk && in && !near) {
        a.inds[r * a.topk + to] = has && live ? (uint32_t)e : 0xFFFFFFFFu;
        a.scores[r * a.topk + to] = !live ? 0.f : bad ? NAN : w * a.scale;
    }
    uint64_t again = __ballot(near && l == 0);
#pragma unroll 1
    while (again) {
        const int at = __ffsll((unsigned long long)again) - 1;
        again &= again - 1;
        wave_order();
        double *const buf = reinterpret_cast<double *>(mem);
        const uint64_t its_open = (uint64_t)__shfl((uint32_t)(open >> 32), at) << 32 | __shfl((uint32_t)open, at);
        if (__shfl(near_group ? 1 : 0, at) || !settle_row<DT>(a, r0 + at / L, lane, buf, by_logit, its_open, __shfl(least, at)))
            route_row<DT>(a, r0 + at / L, lane, buf, by_logit);
        wave_order();
    }
}

// Lanes a row: so many that a lane has at most four units, and up to 2048 rows one each.  256 f32 experts with bias and groups / by
// the logits, us with 32 and with 8 lanes a row: 32 rows 6.4 / 3.6 and 7.9 / 4.8, 2048 rows 11.7 / 4.1 and 13.2 / 5.3, 4096 rows
// 12.7 / 8.1 and 13.4 / 5.3, 65521 rows 71 / 32 and 32 / 21.
template <int L, int T, int DT>
static hipError_t launch_lists(const RouteArgs &a, int units, hipStream_t s) {
    constexpr int at_once = RT_THREADS / L;
    const long wgs = ((long)a.rows + at_once - 1) / at_once;
    const dim3 grid((unsigned)wgs);
    const bool grouped = a.groups > 1, by_logit = !a.bias && (!grouped || a.group_top == 1);
    const int nu = (units + L - 1) / L;
    int id_bits = 6;
    while ((1 << id_bits) < L * nu * 8) id_bits++;
    // the values and the groups' worths of a wave's rows; a row's values in 64 bits and the list that settles it
    const int lists = grouped ? nu * 2048 + 64 / L * 32 + (64 / L * a.groups * 4 + 15) / 16 * 16 : 0, row = (a.experts * 8 + kSettleLds + 15) / 16 * 16;
    const int lds = lists > row ? lists : row;
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(RT_THREADS), RT_WAVES * lds + (by_logit ? 0 : L * nu * 32), s, a, nu, id_bits, lds); };
    if (by_logit) grouped ? go(route_lists_kernel<L, T, DT, true, true>) : go(route_lists_kernel<L, T, DT, true, false>);
    else grouped ? go(route_lists_kernel<L, T, DT, false, true>) : go(route_lists_kernel<L, T, DT, false, false>);
    return hipGetLastError();
}

template <int T, int DT>
static hipError_t with_lanes(const RouteArgs &a, int units, hipStream_t s) {
    const bool few = a.rows <= 2048;
    if (units <= 8 || (!few && units <= 32)) return launch_lists<8, T, DT>(a, units, s);
    if (units <= 16 || (!few && units <= 64)) return launch_lists<16, T, DT>(a, units, s);
    if (units <= 32 || !few) return launch_lists<32, T, DT>(a, units, s);
    return launch_lists<64, T, DT>(a, units, s);
}

template <int DT>
static hipError_t route_of_type(const RouteArgs &a, hipStream_t s) {
    const int units = a.groups * ((a.experts / a.groups + 7) / 8);
    if (a.topk <= 8 && units <= kListUnits) return a.topk <= 4 ? with_lanes<4, DT>(a, units, s) : with_lanes<8, DT>(a, units, s);
    const dim3 grid((unsigned)(((long)a.rows + RT_WAVES - 1) / RT_WAVES));
    hipLaunchKernelGGL(route_kernel<DT>, grid, dim3(RT_THREADS), RT_WAVES * a.experts * sizeof(double), s, a);
    return hipGetLastError();
}

}  // namespace exl3
