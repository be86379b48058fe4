#include "exl3_router.h"
#include "exl3_vec.h"

#include <algorithm>

namespace exl3 {

constexpr int RT_THREADS = 256;

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
// A slot whose id is past the experts has no score.

// The last form reads the whole row.  A row is held by L lanes as in the balance loss's kernel, lane l holding PER experts and
// SPL slots; its row of LDS takes the slots' terms to the lanes that hold their experts (a wave's own rows: no barrier).  333 rows
// of 160 f16 logits take 2.9 us, a launch and a row's latency; 65521 of 256 bf16 16.6, 4.0 TB/s of a read and a write.
template <int L, int PER, int SPL, int DT, bool VEC>
__global__ __launch_bounds__(RT_THREADS) void route_backward_row_kernel(RouteGradArgs a) {
    constexpr int G = RT_THREADS / L;
    const int l = threadIdx.x & (L - 1), grp = threadIdx.x / L, e0 = l * PER;
    __shared__ __align__(16) float rows_lds[G][L * PER];
    float *at = rows_lds[grp];
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * G;
    for (size_t r0 = (size_t)blockIdx.x * G; r0 < rows; r0 += step) {
        const size_t r = r0 + grp;
        const bool in = r < rows, live = in && (!a.mask || a.mask[r] != 0);
        float d[PER], t[SPL], x[SPL];
        int ind[SPL];
#pragma unroll
        for (int i = 0; i < SPL; i++) {
            const int j = l + i * L;
            const size_t slot = r * a.topk + j;
            const bool has = live && j < a.topk;
            ind[i] = has && a.inds[has ? slot : 0] < (uint32_t)a.experts ? (int)a.inds[slot] : -1;
            t[i] = ind[i] >= 0 ? a.dscores[slot] * a.scale : 0.f;
            x[i] = ind[i] >= 0 ? load_act<DT>(a.logits, r * a.experts + ind[i]) : -INFINITY;
        }
        Logits<PER, DT, VEC> row = {};
        if (live) row.load(a.logits, r * a.experts, a.experts, e0);
        row.unpack(a.experts, e0, live, d);
        float mx = d[0];
#pragma unroll
        for (int q = 1; q < PER; q++) mx = fmaxf(mx, d[q]);
        mx = group_max<L>(mx);
        mx = mx == -INFINITY ? 0.f : mx;
        float den = 0.f;
#pragma unroll
        for (int q = 0; q < PER; q++) {
            d[q] = __expf(d[q] - mx);
            den += d[q];
        }
        den = group_sum<L>(den);
        const float inv = den == 0.f ? 0.f : 1.f / den;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < SPL; i++) {  // the slots' terms
            t[i] = ind[i] >= 0 ? expf(x[i] - mx) * inv * t[i] : 0.f;
            dot += t[i];
        }
        dot = group_sum<L>(dot) * inv;
#pragma unroll
        for (int q = 0; q < PER; q++) d[q] *= -dot;
        // Every slot leaves its number at its expert: where two of a row's slots name one expert, some slot does not find its
        // own again.
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

// The other forms read the picked logits alone and write rows of zeros with the slots' terms in them.  A wave has 64 / LS rows, a
// lane a slot; the rows lie one after another in its LDS as they do in memory, so they leave in whole vectors whatever the
// row's length.  Bound by the rows' writes: 65521 rows of 256 bf16, sigmoid over eight slots, 10.9 us (3.6 TB/s with the slots'
// reads; as the kernel above does it, a row's lanes holding its experts, 16.5).
template <int LS, int DT>
__global__ __launch_bounds__(RT_THREADS) void route_backward_picked_kernel(RouteGradArgs a, int wave_lds) {
    constexpr int ROWS = 64 / LS, SIZE = DT == DT_F32 ? 4 : 2, N = 16 / SIZE;
    using Word = std::conditional_t<DT == DT_F32, uint32_t, uint16_t>;
    extern __shared__ __align__(16) char rows_mem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & (LS - 1);
    char *const mem = rows_mem + wave * wave_lds;
    const size_t rows = (size_t)a.rows, r0 = ((size_t)blockIdx.x * (RT_THREADS / 64) + wave) * ROWS, r = r0 + lane / LS;
    if (r0 >= rows) return;
    const bool has = r < rows && j < a.topk && (!a.mask || a.mask[r] != 0);
    const size_t slot = has ? r * a.topk + j : 0;
    const uint32_t id = has ? a.inds[slot] : 0xFFFFFFFFu;
    const bool is = id < (uint32_t)a.experts;
    const float ds = is ? a.dscores[slot] * a.scale : 0.f;
    const float x = is ? load_act<DT>(a.logits, r * a.experts + id) : -INFINITY;
    for (int i = lane * 16; i < wave_lds; i += 1024) *reinterpret_cast<uint4 *>(mem + i) = uint4{0, 0, 0, 0};
    float t = ds;
    const float e = a.sigmoid ? expf(-fabsf(x)) : 0.f;  // sigmoid(x) = (x < 0 ? e : 1) / (1 + e), 1 - sigmoid(x) the other way round
    if (a.renorm) {
        float mx = group_max<LS>(a.sigmoid ? fminf(x, 0.f) : x);
        mx = mx == -INFINITY ? 0.f : mx;
        float w = is ? (a.sigmoid ? expf(fminf(x, 0.f) - mx) / (1.f + e) : expf(x - mx)) : 0.f;
        const float sum = group_sum<LS>(w);
        w = sum == 0.f ? 0.f : w / sum;
        t = w * (ds - group_sum<LS>(w * ds));
    } else {
        t = ds * ((x >= 0.f ? 1.f : e) / (1.f + e));
    }
    if (a.sigmoid) t *= (x >= 0.f ? e : 1.f) / (1.f + e);
    // A slot leaves its number at its expert: where two of a row's slots name one expert, some slot does not find its own again.
    Word *const at = reinterpret_cast<Word *>(mem) + (lane / LS) * a.experts + (is ? id : 0);
    wave_order();
    if (is) *at = (Word)(j + 1);
    wave_order();
    if (__any(is && *at != (Word)(j + 1))) {  // equal experts' terms add in slot order, and each of their slots has the sum
        float sum = 0.f;
        for (int i = 0; i < LS; i++) sum += (uint32_t)__shfl((int)id, i, LS) == id ? __shfl(t, i, LS) : 0.f;
        t = sum;
    }
    wave_order();
    if (is) {
        if constexpr (DT == DT_F32) *at = __float_as_uint(t);
        else if constexpr (DT == DT_F16) *at = __half_as_ushort(__float2half_rn(t));
        else *at = __bfloat16_as_ushort(__float2bfloat16(t));
    }
    wave_order();
    const int count = (int)min((size_t)ROWS, rows - r0) * a.experts;
    char *const out = static_cast<char *>(a.dlogits) + r0 * a.experts * SIZE;
    for (int i = lane * N; i < count; i += 64 * N) {
        if (i + N <= count) {
            *reinterpret_cast<Words4At2 *>(out + i * SIZE) = *reinterpret_cast<const Words4 *>(mem + i * SIZE);
        } else {
            for (int q = i; q < count; q++) reinterpret_cast<Word *>(out)[q] = reinterpret_cast<const Word *>(mem)[q];
        }
    }
}

template <int LS, int DT>
static hipError_t launch_picked(const RouteGradArgs &a, hipStream_t s) {
    const int size = DT == DT_F32 ? 4 : 2, lds = (64 / LS * a.experts * size + 15) / 16 * 16;
    constexpr int at_once = RT_THREADS / LS, most = 1 << 24;  // rows a launch
    for (int r = 0; r < a.rows; r += std::min(most, a.rows - r)) {
        RouteGradArgs c = a;
        c.rows = std::min(most, a.rows - r);
        c.logits = static_cast<const char *>(a.logits) + (size_t)r * a.experts * size;
        c.inds = a.inds + (size_t)r * a.topk;
        c.dscores = a.dscores + (size_t)r * a.topk;
        c.mask = a.mask ? a.mask + r : nullptr;
        c.dlogits = static_cast<char *>(a.dlogits) + (size_t)r * a.experts * size;
        hipLaunchKernelGGL((route_backward_picked_kernel<LS, DT>), dim3((unsigned)((c.rows + at_once - 1) / at_once)), dim3(RT_THREADS),
                           RT_THREADS / 64 * lds, s, c, lds);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t run_route_backward(const RouteGradArgs &a, hipStream_t s) {
    if (a.sigmoid || a.renorm)
        return with_dtype(a.dtype, [&](auto DT) {
            constexpr int dt = decltype(DT)::value;
            // lanes a row: its slots, and so many that a wave's rows take 8 KiB at most
            const int row = a.experts * (dt == DT_F32 ? 4 : 2);
            if (a.topk <= 8 && row <= 1024) return launch_picked<8, dt>(a, s);
            if (a.topk <= 16 && row <= 2048) return launch_picked<16, dt>(a, s);
            return launch_picked<32, dt>(a, s);
        });
    return with_shape(a.experts, [&](auto L, auto PER) {
        return with_dtype(a.dtype, [&](auto DT) {
            constexpr int l = decltype(L)::value, per = decltype(PER)::value, dt = decltype(DT)::value;
            const long groups = ((long)a.rows + RT_THREADS / l - 1) / (RT_THREADS / l);
            const dim3 grid((unsigned)(groups < 8192 ? groups : 8192));
            const bool vec = whole_vectors<per, dt>(a.logits, a.experts) && whole_vectors<per, dt>(a.dlogits, a.experts);
            auto launch = [&](auto SPL) {
                constexpr int spl = decltype(SPL)::value;
                auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(RT_THREADS), 0, s, a); };
                vec ? go(route_backward_row_kernel<l, per, spl, dt, true>) : go(route_backward_row_kernel<l, per, spl, dt, false>);
                return hipGetLastError();
            };
            if constexpr (l < 32)
                if (a.topk > l) return launch(std::integral_constant<int, 32 / l>{});
            return launch(std::integral_constant<int, 1>{});
        });
    });
}

}  // namespace exl3
