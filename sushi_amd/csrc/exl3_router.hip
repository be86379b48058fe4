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
//
// Measured: balance loss of 65521 rows of 128 bf16 logits 13.4 us (16.8 MB of logits; about 5 us are the two-level join),
// of 32 rows of 256 f32 logits 4.1; the gradient of 65521 x 128 15.7 us (36.6 MB; vector instructions fill 60% of the
// kernel), of 2048 x 256 4.5.  Sixteen experts a lane in place of eight spend a fifth less on each row's sums but hold
// fewer waves: the gradient 14.4 and 6.2 us there, the balance loss 14.3 and 4.75.  Without the loop over rows (a
// workgroup for every set of them, no loads ahead) the gradient of 65521 rows takes 21 us.
#include "exl3_router.h"

namespace exl3 {

constexpr int RB_THREADS = 256;
constexpr int BL_THREADS = 512;

// What one workgroup leaves for another of the same launch is written through to memory and read past the caches.
// (Device-wide release and acquire fences instead write back and drop whole L2s: 16 workgroups' worth of them took 50 us.)
template <class T>
__device__ __forceinline__ void put(T *p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
template <class T>
__device__ __forceinline__ T get(const T *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// An expert's sum of probabilities and its count, as one word of a part.
__device__ __forceinline__ uint64_t pair_of(float sum, int count) { return (uint64_t)__float_as_uint(sum) << 32 | (uint32_t)count; }

// One expert's sum and count over n parts from `first` on, in their order, B parts' loads at a time.
template <int B>
__device__ __forceinline__ void sum_parts(const BalanceArgs &a, int first, int n, int e, float &sum, int &count) {
    float x = 0.f;
    int c = 0;
    for (int i0 = 0; i0 < n; i0 += B) {
        uint64_t w[B];
#pragma unroll
        for (int i = 0; i < B; i++) w[i] = get(a.parts + (size_t)(first + min(i0 + i, n - 1)) * a.experts + e);
#pragma unroll
        for (int i = 0; i < B; i++) {
            x += i0 + i < n ? __uint_as_float((uint32_t)(w[i] >> 32)) : 0.f;
            c += i0 + i < n ? (int)(uint32_t)w[i] : 0;
        }
    }
    sum = x;
    count = c;
}

// The live rows of parts first .. first + n - 1 (n <= 64, one wave).
__device__ __forceinline__ int live_parts(const BalanceArgs &a, int first, int n, int lane) {
    int v = lane < n ? get(a.part_live + first + lane) : 0;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// Counts this workgroup at *ctr once its stores are acknowledged; true in the last of `n` to arrive, which leaves the
// counter at zero.
__device__ __forceinline__ bool last_to_arrive(uint32_t *ctr, int n, int *shared) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t old = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *shared = old == (uint32_t)(n - 1);
        if (*shared) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *shared != 0;
}

// Workgroup b sums rows b G, b G + gridDim.x G, ... (G rows at once, the next ones' logits in flight) into its part: E sums,
// E counts and its live rows.  The parts are joined in two levels by whoever arrives last: of kBalanceJoin consecutive
// workgroups the last sums their parts into one, and of those the last sums them and writes the results (its threads in
// JT shares of the parts, so that every load is in flight at once).  Each sum runs in a fixed order, whoever does it.  (As
// a second launch of one workgroup the join took 22 us over 512 parts of 128 experts.)
static_assert(kBalanceJoin <= 64 && kBalanceMaxParts <= 64 * kBalanceJoin, "one wave joins the live rows");
template <int L, int PER, int DT, bool VEC>
__global__ __launch_bounds__(BL_THREADS) void balance_kernel(BalanceArgs a) {
    constexpr int G = BL_THREADS / L;  // rows at once
    constexpr int E_MAX = L * PER;
    __shared__ float sums[BL_THREADS / 64][E_MAX];
    constexpr int JT = E_MAX >= BL_THREADS ? 1 : BL_THREADS / E_MAX < 8 ? BL_THREADS / E_MAX : 8;
    constexpr int JB = kBalanceMaxParts / kBalanceJoin / JT < kBalanceJoin ? kBalanceMaxParts / kBalanceJoin / JT : kBalanceJoin;
    __shared__ int hist[E_MAX], join_count[JT][E_MAX];
    __shared__ int live_rows, flag;
    __shared__ float red[BL_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = tid & (L - 1), grp = tid / L, e0 = l * PER;
    for (int e = tid; e < E_MAX; e += BL_THREADS) hist[e] = 0;
    if (tid == 0) live_rows = 0;
    __syncthreads();
    float acc[PER] = {};
    int mine = 0;
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * G;
    // the next row's logits, mask and first slot of the lane; a row past the end is not live
    Logits<PER, DT, VEC> next = {};
    bool next_live = false;
    uint32_t next_ind = 0;
    size_t r = (size_t)blockIdx.x * G + grp;
    auto fetch = [&](size_t row) __attribute__((always_inline)) {
        next_live = row < rows;
        if (next_live) {
            next.load(a.logits, row * a.experts, a.experts, e0);
            next_ind = a.inds[row * a.topk + min(l, a.topk - 1)];
            if (a.mask) next_live = a.mask[row] != 0;
        }
    };
    fetch(r);
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < rows; r0 += step, r += step) {
        float v[PER];
        const bool live = next_live;
        const uint32_t ind = next_ind;
        next.unpack(a.experts, e0, live, v);
        if (r0 + step < rows) fetch(r + step);
        if (live) {
            if (l < a.topk && ind < (uint32_t)a.experts) atomicAdd(&hist[ind], 1);
            for (int j = l + L; j < a.topk; j += L) {
                const uint32_t e = a.inds[r * a.topk + j];
                if (e < (uint32_t)a.experts) atomicAdd(&hist[e], 1);
            }
        }
        const float den = group_sum<L>(row_exp<L, PER>(v));
        const float inv = den == 0.f || !live ? 0.f : rcp(den);
#pragma unroll
        for (int q = 0; q < PER; q++) acc[q] += v[q] * inv;
        mine += live && l == 0 ? 1 : 0;
    }
    if (mine) atomicAdd(&live_rows, mine);
    // the row groups of a wave, then the waves in order
#pragma unroll
    for (int q = 0; q < PER; q++) {
        if constexpr (L < 16) acc[q] += xor_lane_row<8>(acc[q]);
        if constexpr (L < 32) acc[q] += __shfl_xor(acc[q], 16);
        if constexpr (L < 64) acc[q] += __shfl_xor(acc[q], 32);
        if (lane < L) sums[wave][e0 + q] = acc[q];
    }
    __syncthreads();
    for (int e = tid; e < E_MAX; e += BL_THREADS) {
        float s = sums[0][e];
#pragma unroll
        for (int w = 1; w < BL_THREADS / 64; w++) s += sums[w][e];
        sums[0][e] = s;
    }
    __syncthreads();
    if (gridDim.x > 1) {
        const int b = blockIdx.x, join = b / kBalanceJoin * kBalanceJoin, n = min(kBalanceJoin, (int)gridDim.x - join);
        const int joins = ((int)gridDim.x + kBalanceJoin - 1) / kBalanceJoin;
        for (int e = tid; e < a.experts; e += BL_THREADS) put(a.parts + (size_t)b * a.experts + e, pair_of(sums[0][e], hist[e]));
        if (tid == 0) put(a.part_live + b, live_rows);
        if (!last_to_arrive(a.counters + (size_t)(1 + join / kBalanceJoin) * COUNTER_STRIDE, n, &flag)) return;
        // (the joined parts land in a row of their own past the workgroups')
        const size_t out = gridDim.x + join / kBalanceJoin;
        for (int e = tid; e < a.experts; e += BL_THREADS) {
            float x;
            int c;
            sum_parts<kBalanceJoin>(a, join, n, e, x, c);
            put(a.parts + out * a.experts + e, pair_of(x, c));
        }
        if (wave == 0) {
            const int v = live_parts(a, join, n, lane);
            if (lane == 0) put(a.part_live + out, v);
        }
        if (!last_to_arrive(a.counters, joins, &flag)) return;
        const int share = tid / E_MAX, per = (joins + JT - 1) / JT;
        if (share < JT) {
            for (int e = JT > 1 ? tid % E_MAX : tid; e < a.experts; e += JT > 1 ? E_MAX : BL_THREADS) {
                float x = 0.f;
                int c = 0;
                const int n2 = min(per, joins - share * per);
                if (n2 > 0) sum_parts<JB>(a, gridDim.x + share * per, n2, e, x, c);
                sums[share][e] = x;
                join_count[share][e] = c;
            }
        }
        if (wave == 0) {
            const int v = live_parts(a, gridDim.x, joins, lane);
            if (lane == 0) live_rows = v;
        }
        __syncthreads();
        for (int e = tid; e < a.experts; e += BL_THREADS) {
            float x = sums[0][e];
            int c = join_count[0][e];
#pragma unroll
            for (int i = 1; i < JT; i++) x += sums[i][e], c += join_count[i][e];
            sums[0][e] = x;
            hist[e] = c;
        }
        __syncthreads();
    }
    // the results from the sums and counts in LDS
    const float T = (float)live_rows;
    const float scale = live_rows > 0 ? a.coef * (float)a.experts / (T * (float)a.topk) / T : 0.f;
    float part = 0.f;
    for (int e = tid; e < a.experts; e += BL_THREADS) {
        const float w = scale * (float)hist[e];
        a.weight[e] = w;
        a.counts[e] = hist[e];
        part += w * sums[0][e];
    }
    part = group_sum<64>(part);
    if (lane == 0) red[wave] = part;
    __syncthreads();
    if (tid == 0) {
        float s = 0.f;
        for (int w = 0; w < BL_THREADS / 64; w++) s += red[w];
        *a.loss = s;
    }
}

// What a row brings: its lane's logits and SPL slots (lane l holds slots l, l + L, ...), and whether it is live.
template <int L, int PER, int SPL, int DT, bool VEC>
struct RouterRow {
    Logits<PER, DT, VEC> logits;
    uint32_t ind[SPL];
    float ds[SPL];
    bool live;
    __device__ __forceinline__ void load(const RouterGradArgs &a, size_t r, int l) {
        live = r < (size_t)a.rows;
        if (!live) return;
        logits.load(a.logits, r * a.experts, a.experts, l * PER);
        if (a.dscores) {
#pragma unroll
            for (int i = 0; i < SPL; i++) {  // a slot past the row's as its last one, dropped below
                const size_t at = r * a.topk + min(l + i * L, a.topk - 1);
                ind[i] = a.inds[at];
                ds[i] = a.dscores[at];
            }
        }
        if (a.mask) live = a.mask[r] != 0;
    }
};

// dlogits: each group of L lanes takes rows in strides of the grid, the next row's loads in flight (eight workgroups a CU:
// within 64 registers where rows are whole vectors and a lane has one slot and eight experts).  A row's lanes are one
// wave's, so its row of LDS needs no barrier: it carries the logits to the slots that picked them and the slots' terms
// back to the lanes that hold their experts.
template <int L, int PER, int SPL, int DT, bool VEC>
__global__ __launch_bounds__(RB_THREADS) void router_backward_kernel(RouterGradArgs a) {
    constexpr int G = RB_THREADS / L;
    using Row = RouterRow<L, PER, SPL, DT, VEC>;
    const int l = threadIdx.x & (L - 1), grp = threadIdx.x / L, e0 = l * PER;
    __shared__ __align__(16) float rows_lds[G][L * PER];
    float *at = rows_lds[grp];
    float w[PER];
    const float dloss = a.weight ? *a.dloss : 0.f;
#pragma unroll
    for (int q = 0; q < PER; q++) w[q] = a.weight && e0 + q < a.experts ? a.weight[e0 + q] : 0.f;
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * G;
    size_t r = (size_t)blockIdx.x * G + grp;
    Row next = {};
    next.load(a, r, l);
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < rows; r0 += step, r += step) {
        const bool live = next.live;
        float d[PER];
        next.logits.unpack(a.experts, e0, live, d);
        float ds[SPL], s[SPL];
        int ind[SPL];
#pragma unroll
        for (int i = 0; i < SPL; i++) {  // a slot with no expert has no score
            ind[i] = live && l + i * L < a.topk && next.ind[i] < (uint32_t)a.experts ? (int)next.ind[i] : -1;
            ds[i] = next.ds[i];
        }
        if (r0 + step < rows) next.load(a, r + step, l);
        bool twice = false;
        if (a.dscores) {
#pragma unroll
            for (int q = 0; q < PER; q++) at[e0 + q] = d[q];
            wave_order();
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                const float x = at[max(ind[i], 0)];
                s[i] = ind[i] >= 0 ? x : -INFINITY;
                mx = fmaxf(mx, s[i]);
            }
            // Every slot leaves its number at its expert: where two of a row's slots name one expert, some slot does not
            // find its own again.
            wave_order();
#pragma unroll
            for (int i = 0; i < SPL; i++)
                if (ind[i] >= 0) at[ind[i]] = __int_as_float(l + i * L + 1);
            wave_order();
#pragma unroll
            for (int i = 0; i < SPL; i++)
                twice |= ind[i] >= 0 && __float_as_int(at[max(ind[i], 0)]) != l + i * L + 1;
            mx = group_max<L>(mx);
            const float base = mx == -INFINITY ? 0.f : mx;
            float den = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                s[i] = __expf(s[i] - base);
                den += s[i];
                dot += ind[i] >= 0 ? s[i] * ds[i] : 0.f;
            }
            den = group_sum<L>(den);
            dot = group_sum<L>(dot);
            const float inv = den == 0.f ? 0.f : rcp(den);
            dot *= inv;
#pragma unroll
            for (int i = 0; i < SPL; i++) s[i] = s[i] * inv * (ds[i] - dot);  // the slot's term
        }
        if (a.weight) {
            float den = row_exp<L, PER>(d), dot = 0.f;
#pragma unroll
            for (int q = 0; q < PER; q++) dot += w[q] * d[q];
            den = group_sum<L>(den);
            dot = group_sum<L>(dot);
            const float inv = den == 0.f ? 0.f : rcp(den);
            const float c = dloss * inv;
            const float cdot = c * (dot * inv);
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] *= c * w[q] - cdot;
        } else {
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] = 0.f;
        }
        if (a.dscores) {
            wave_order();
            if (__any(twice)) {  // slot by slot, so equal experts' terms always add in slot order
#pragma unroll
                for (int i = 0; i < SPL; i++) {
                    const int n = min(L, a.topk - i * L);
                    for (int j = 0; j < n; j++) {
                        const int e = __shfl(ind[i], j, L) - e0;
                        const float t = __shfl(s[i], j, L);
#pragma unroll
                        for (int q = 0; q < PER; q++) d[q] += e == q ? t : 0.f;
                    }
                }
            } else {
#pragma unroll
                for (int q = 0; q < PER; q++) at[e0 + q] = d[q];
                wave_order();
#pragma unroll
                for (int i = 0; i < SPL; i++)
                    if (ind[i] >= 0) at[ind[i]] += s[i];
                wave_order();
#pragma unroll
                for (int q = 0; q < PER; q++) d[q] = at[e0 + q];
            }
            wave_order();
        }
        if (r < rows) store_logits<PER, DT, VEC>(a.dlogits, r * a.experts, a.experts, e0, live, d);
    }
}

static int lanes_of(int experts) {
    return experts <= 64 ? 8 : experts <= 128 ? 16 : experts <= 256 ? 32 : 64;
}

// Workgroups of the balance loss: one for up to eight sets of the rows it holds at once (the join costs more), else one for
// each set, at most two a CU.  One workgroup against one for each set, us in a graph, top-8: 64 rows of 128 experts (two sets)
// 3.9 and 7.8, 128 rows (four) 4.8 and 7.9, 256 (eight) 7.0 and 7.7; eight sets of 64, 256 and 512 experts 7.0 and 7.8, 7.5 and
// 8.4, 7.5 and 8.7; from there on a set costs half a microsecond.
constexpr long kBalanceAlone = 8;
int balance_parts(int rows, int experts) {
    const int at_once = BL_THREADS / lanes_of(experts);
    const long sets = ((long)rows + at_once - 1) / at_once;
    return (int)(sets <= kBalanceAlone ? 1 : sets < kBalanceMaxParts ? sets : kBalanceMaxParts);
}

hipError_t run_balance_loss(const BalanceArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)balance_parts(a.rows, a.experts));
    return with_shape(a.experts, [&](auto L, auto PER) {
        return with_dtype(a.dtype, [&](auto DT) {
            constexpr int l = decltype(L)::value, per = decltype(PER)::value, dt = decltype(DT)::value;
            if (whole_vectors<per, dt>(a.logits, a.experts))
                hipLaunchKernelGGL((balance_kernel<l, per, dt, true>), grid, dim3(BL_THREADS), 0, s, a);
            else
                hipLaunchKernelGGL((balance_kernel<l, per, dt, false>), grid, dim3(BL_THREADS), 0, s, a);
            return hipGetLastError();
        });
    });
}

hipError_t run_router_backward(const RouterGradArgs &a, hipStream_t s) {
    const int at_once = RB_THREADS / lanes_of(a.experts);
    const long groups = ((long)a.rows + at_once - 1) / at_once;
    const unsigned grid = (unsigned)(groups < 2048 ? groups : 2048);  // eight workgroups a CU, then more rows each
    return with_shape(a.experts, [&](auto L, auto PER) {
        return with_dtype(a.dtype, [&](auto DT) {
            constexpr int l = decltype(L)::value, per = decltype(PER)::value, dt = decltype(DT)::value;
            const bool vec = whole_vectors<per, dt>(a.logits, a.experts) && whole_vectors<per, dt>(a.dlogits, a.experts);
            auto launch = [&](auto SPL) {
                constexpr int spl = decltype(SPL)::value;
                if (vec)
                    hipLaunchKernelGGL((router_backward_kernel<l, per, spl, dt, true>), dim3(grid), dim3(RB_THREADS), 0, s, a);
                else
                    hipLaunchKernelGGL((router_backward_kernel<l, per, spl, dt, false>), dim3(grid), dim3(RB_THREADS), 0, s, a);
                return hipGetLastError();
            };
            // slots a lane: one where the row's lanes hold them all, else enough for the 32 a row may have
            if constexpr (l < 32)
                if (a.topk > l) return launch(std::integral_constant<int, 32 / l>{});
            return launch(std::integral_constant<int, 1>{});
        });
    });
}

}  // namespace exl3
