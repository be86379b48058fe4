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

// Butterflies over the L lanes of a row: DPP within 16 lanes, a shuffle for the steps of 16 and 32.
template <int L, class F>
__device__ __forceinline__ float group_join(float v, F f) {
    if constexpr (L > 1) v = f(v, xor_lane_row<1>(v));
    if constexpr (L > 2) v = f(v, xor_lane_row<2>(v));
    if constexpr (L > 4) v = f(v, xor_lane_row<4>(v));
    if constexpr (L > 8) v = f(v, xor_lane_row<8>(v));
    if constexpr (L > 16) v = f(v, __shfl_xor(v, 16));
    if constexpr (L > 32) v = f(v, __shfl_xor(v, 32));
    return v;
}
template <int L>
__device__ __forceinline__ float group_max(float v) {
    return group_join<L>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    return group_join<L>(v, [](float a, float b) { return a + b; });
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

// Their counterpart: PER values of a row, rounded to the logits' type.
template <int PER, int DT, bool VEC>
__device__ __forceinline__ void store_logits(void *p, size_t row, int experts, int e0, const float (&v)[PER]) {
    const size_t at = row * (size_t)experts + e0;
    if constexpr (VEC && PER * (DT == DT_F32 ? 4 : 2) >= 4) {
        if (e0 >= experts) return;
        constexpr int W = PER * (DT == DT_F32 ? 4 : 2) / 4;
        uint32_t w[W];
#pragma unroll
        for (int q = 0; q < W; q++) {
            if constexpr (DT == DT_F32) w[q] = __float_as_uint(v[q]);
            else if constexpr (DT == DT_F16)
                w[q] = __half_as_ushort(__float2half_rn(v[2 * q])) | (uint32_t)__half_as_ushort(__float2half_rn(v[2 * q + 1])) << 16;
            else
                w[q] = __bfloat16_as_ushort(__float2bfloat16(v[2 * q])) |
                       (uint32_t)__bfloat16_as_ushort(__float2bfloat16(v[2 * q + 1])) << 16;
        }
        char *o = static_cast<char *>(p) + at * (DT == DT_F32 ? 4 : 2);
        if constexpr (W >= 4) {
#pragma unroll
            for (int q = 0; q < W / 4; q++)
                reinterpret_cast<uint4 *>(o)[q] = uint4{w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
        } else if constexpr (W == 2) {
            *reinterpret_cast<uint2 *>(o) = uint2{w[0], w[1]};
        } else {
            *reinterpret_cast<uint32_t *>(o) = w[0];
        }
    } else {
#pragma unroll
        for (int q = 0; q < PER; q++)
            if (e0 + q < experts) store_act<DT>(p, at + q, v[q]);
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
    const float inv = den == 0.f ? 0.f : rcp(den);
#pragma unroll
    for (int q = 0; q < PER; q++) v[q] *= inv;
}

// Orders a wave's LDS accesses across lanes: the hardware runs them in order, the compiler must too.
__device__ __forceinline__ void wave_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

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

// One expert's sum and count over parts first .. first + n - 1 (n <= kBalanceJoin or <= kBalanceMaxParts / kBalanceJoin), in
// their order, eight parts' loads at a time.
__device__ __forceinline__ void sum_parts(const BalanceArgs &a, int first, int n, int e, float &sum, int &count) {
    float x = 0.f;
    int c = 0;
    for (int i0 = 0; i0 < n; i0 += 8) {
        float xs[8];
        int cs[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const size_t at = (size_t)(first + min(i0 + i, n - 1)) * a.experts + e;
            xs[i] = get(a.part_sum + at);
            cs[i] = get(a.part_count + at);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x += i0 + i < n ? xs[i] : 0.f;
            c += i0 + i < n ? cs[i] : 0;
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
// workgroups the last sums their parts into one, and of those the last sums them and writes the results.  Each sum runs in the parts' order, whoever does it.  (As a second launch of one workgroup the join
// took 22 us over 512 parts of 128 experts.)
static_assert(kBalanceJoin <= 64 && kBalanceMaxParts <= 64 * kBalanceJoin, "one wave joins the live rows");
template <int L, int PER, int DT, bool VEC>
__global__ __launch_bounds__(BL_THREADS) void balance_kernel(BalanceArgs a) {
    constexpr int G = BL_THREADS / L;  // rows at once
    constexpr int E_MAX = L * PER;
    __shared__ float sums[BL_THREADS / 64][E_MAX];
    __shared__ int hist[E_MAX];
    __shared__ int live_rows, flag;
    __shared__ float red[BL_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = tid & (L - 1), grp = tid / L, e0 = l * PER;
    for (int e = tid; e < E_MAX; e += BL_THREADS) hist[e] = 0;
    if (tid == 0) live_rows = 0;
    __syncthreads();
    float acc[PER] = {};
    int mine = 0;
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * G;
    // the next row's logits, mask and first slot of the lane
    float next[PER];
    uint8_t next_live = 1;
    uint32_t next_ind = 0;
    size_t r = (size_t)blockIdx.x * G + grp;
    auto fetch = [&](size_t row) __attribute__((always_inline)) {
        load_logits<PER, DT, VEC>(a.logits, row, a.experts, e0, next);
        if (a.mask) next_live = a.mask[row];
        next_ind = a.inds[row * a.topk + min(l, a.topk - 1)];
    };
    if (rows) fetch(r < rows ? r : rows - 1);
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < rows; r0 += step, r += step) {
        float v[PER];
#pragma unroll
        for (int q = 0; q < PER; q++) v[q] = next[q];
        const bool live = r < rows && next_live;
        const uint32_t ind = next_ind;
        if (r0 + step < rows) fetch(r + step < rows ? r + step : rows - 1);
        if (live) {
            if (l < a.topk && ind < (uint32_t)a.experts) atomicAdd(&hist[ind], 1);
            for (int j = l + L; j < a.topk; j += L) {
                const uint32_t e = a.inds[r * a.topk + j];
                if (e < (uint32_t)a.experts) atomicAdd(&hist[e], 1);
            }
        }
        row_softmax<L, PER>(v);
#pragma unroll
        for (int q = 0; q < PER; q++) acc[q] += live ? v[q] : 0.f;
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
        for (int e = tid; e < a.experts; e += BL_THREADS) {
            put(a.part_sum + (size_t)b * a.experts + e, sums[0][e]);
            put(a.part_count + (size_t)b * a.experts + e, hist[e]);
        }
        if (tid == 0) put(a.part_live + b, live_rows);
        if (!last_to_arrive(a.counters + (size_t)(1 + join / kBalanceJoin) * COUNTER_STRIDE, n, &flag)) return;
        // (the joined parts land in a row of their own past the workgroups')
        const size_t out = gridDim.x + join / kBalanceJoin;
        for (int e = tid; e < a.experts; e += BL_THREADS) {
            float x;
            int c;
            sum_parts(a, join, n, e, x, c);
            put(a.part_sum + out * a.experts + e, x);
            put(a.part_count + out * a.experts + e, c);
        }
        if (wave == 0) {
            const int v = live_parts(a, join, n, lane);
            if (lane == 0) put(a.part_live + out, v);
        }
        if (!last_to_arrive(a.counters, joins, &flag)) return;
        for (int e = tid; e < a.experts; e += BL_THREADS) {
            float x;
            int c;
            sum_parts(a, gridDim.x, joins, e, x, c);
            sums[0][e] = x;
            hist[e] = c;
        }
        if (wave == 0) {
            const int v = live_parts(a, gridDim.x, joins, lane);
            if (lane == 0) live_rows = v;
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

// What a row brings: its lane's logits and slots (lane l holds slots l, l + L, ...), and whether it is live.
template <int L, int PER>
struct RouterRow {
    static constexpr int SPL = L >= 32 ? 1 : 32 / L;  // slots a lane holds (up to 32 a row)
    float v[PER];
    uint32_t ind[SPL];
    float ds[SPL];
    uint8_t live;
};
template <int L, int PER, int DT, bool VEC>
__device__ __forceinline__ void load_row(const RouterGradArgs &a, size_t r, int l, RouterRow<L, PER> &row) {
    load_logits<PER, DT, VEC>(a.logits, r, a.experts, l * PER, row.v);
    row.live = a.mask ? a.mask[r] : (uint8_t)1;
    if (a.dscores) {
#pragma unroll
        for (int i = 0; i < RouterRow<L, PER>::SPL; i++) {  // a slot past the row's as its last one, dropped below
            const size_t at = r * a.topk + min(l + i * L, a.topk - 1);
            row.ind[i] = a.inds[at];
            row.ds[i] = a.dscores[at];
        }
    }
}

// dlogits: each group of L lanes takes rows in strides of the grid, the next row's loads in flight.  A row's lanes are one
// wave's, so its row of LDS needs no barrier: it carries the logits to the slots that picked them and the slots' terms
// back to the lanes that hold their experts.
template <int L, int PER, int DT, bool VEC>
__global__ __launch_bounds__(RB_THREADS) void router_backward_kernel(RouterGradArgs a) {
    constexpr int G = RB_THREADS / L;
    constexpr int SPL = RouterRow<L, PER>::SPL;
    const int l = threadIdx.x & (L - 1), grp = threadIdx.x / L, e0 = l * PER;
    __shared__ __align__(16) float rows_lds[G][L * PER];
    float *at = rows_lds[grp];
    float w[PER];
    const float dloss = a.weight ? *a.dloss : 0.f;
#pragma unroll
    for (int q = 0; q < PER; q++) w[q] = a.weight && e0 + q < a.experts ? a.weight[e0 + q] : 0.f;
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * G;
    size_t r = (size_t)blockIdx.x * G + grp;
    RouterRow<L, PER> next;
    load_row<L, PER, DT, VEC>(a, r < rows ? r : rows - 1, l, next);
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < rows; r0 += step, r += step) {
        const RouterRow<L, PER> row = next;
        if (r0 + step < rows) load_row<L, PER, DT, VEC>(a, r + step < rows ? r + step : rows - 1, l, next);
        float d[PER];
        float g[SPL];
        int ind[SPL];
        bool twice = false;
        if (a.dscores) {
#pragma unroll
            for (int q = 0; q < PER; q++) at[e0 + q] = row.v[q];
            wave_order();
            float s[SPL], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < SPL; i++) {  // a slot with no expert has no score
                ind[i] = l + i * L < a.topk && row.ind[i] < (uint32_t)a.experts ? (int)row.ind[i] : -1;
                s[i] = ind[i] >= 0 ? at[ind[i]] : -INFINITY;
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
                if (ind[i] >= 0) twice = twice || __float_as_int(at[ind[i]]) != l + i * L + 1;
            mx = group_max<L>(mx);
            const float base = mx == -INFINITY ? 0.f : mx;
            float den = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                s[i] = __expf(s[i] - base);
                den += s[i];
            }
            den = group_sum<L>(den);
            const float inv = den == 0.f ? 0.f : rcp(den);
#pragma unroll
            for (int i = 0; i < SPL; i++) {
                s[i] *= inv;
                dot += ind[i] >= 0 ? s[i] * row.ds[i] : 0.f;
            }
            dot = group_sum<L>(dot);
#pragma unroll
            for (int i = 0; i < SPL; i++) g[i] = s[i] * (row.ds[i] - dot);
        }
#pragma unroll
        for (int q = 0; q < PER; q++) d[q] = a.weight ? row.v[q] : 0.f;
        if (a.weight) {
            row_softmax<L, PER>(d);
            float dot = 0.f;
#pragma unroll
            for (int q = 0; q < PER; q++) dot += w[q] * d[q];
            dot = group_sum<L>(dot);
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] = dloss * d[q] * (w[q] - dot);
        }
        if (a.dscores) {
            wave_order();
            if (__any(twice)) {  // slot by slot, so equal experts' terms always add in slot order
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
            } else {
#pragma unroll
                for (int q = 0; q < PER; q++) at[e0 + q] = d[q];
                wave_order();
#pragma unroll
                for (int i = 0; i < SPL; i++)
                    if (ind[i] >= 0) at[ind[i]] += g[i];
                wave_order();
#pragma unroll
                for (int q = 0; q < PER; q++) d[q] = at[e0 + q];
            }
            wave_order();
        }
        if (r < rows) {
#pragma unroll
            for (int q = 0; q < PER; q++) d[q] = row.live ? d[q] : 0.f;
            store_logits<PER, DT, VEC>(a.dlogits, r, a.experts, e0, d);
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

// Workgroups of the balance loss: one while a single pass or two of it hold the rows (the join costs more), else one for
// each set of rows it holds at once, at most two a CU.
int balance_parts(int rows, int experts) {
    const int at_once = BL_THREADS / lanes_of(experts);
    const long sets = ((long)rows + at_once - 1) / at_once;
    return (int)(sets <= 2 ? 1 : sets < kBalanceMaxParts ? sets : kBalanceMaxParts);
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
            if (whole_vectors<per, dt>(a.logits, a.experts) && whole_vectors<per, dt>(a.dlogits, a.experts))
                hipLaunchKernelGGL((router_backward_kernel<l, per, dt, true>), dim3(grid), dim3(RB_THREADS), 0, s, a);
            else
                hipLaunchKernelGGL((router_backward_kernel<l, per, dt, false>), dim3(grid), dim3(RB_THREADS), 0, s, a);
            return hipGetLastError();
        });
    });
}

}  // namespace exl3
