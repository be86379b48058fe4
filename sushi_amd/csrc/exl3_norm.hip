// The norms before and after a block with its gate and residual, and their gradient.  With rms(v) = v / sqrt(mean v^2 + eps):
//   n = post ? rms(y) (o + post) : y,   h' = a h + b g n,   x' = rms(h') (o + pre)
// and backwards, from dh and dx, with r and q the factors of rms(h') and rms(y):
//   u = dx (o + pre),  H = dh + r (u - h' r^2 mean(u h')),  dpre = sum over rows of dx h' r,  dh_in = a H
//   dg = b H n (summed as the gate was broadcast),  z = b H g,  dpost = sum over rows of z y q,
//   v = post ? z (o + post) : z,   dy = post ? q (v - y q^2 mean(v y)) : z.
// Everything is f32 up to the one rounding of each output; x' comes of the h' that is not yet rounded, the gradient's r of
// the h' that was kept.
//
// Both passes are bound by the rows' bytes: a row stays in registers between its loads and its stores, whatever its norms need
// over it.  Forward, bf16 with both norms: 16384 rows of 4096 values 98 us (5.5 TB/s; a large copy reaches 5.2), 8192 rows of
// 8192 / 16384 96 / 191, 2047 rows of 5120 with an f32 stream and a gate 25; one row of 4096 3.5 us, a launch and two row sums.  Gradient:
// 16384 rows of 4096 155 us (5.2 TB/s); 333 rows of 2560, f16 with an f32 stream and a channel gate, 10.2: the latency of two rows
// (7.5) and the join's launch.
#include "exl3_vec.h"
#include "exl3_epilogue.h"

#include <algorithm>
#include <type_traits>

namespace exl3 {

// A wave's sum, in every lane: pairs, quads, 8 and 16 lanes by exchanges, then each row of 16 adds what the rows before it hold.
__device__ __forceinline__ float wave_total(float v) {
    v += xor_lane_row<1>(v);
    v += xor_lane_row<2>(v);
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, false));  // (quads hold one value)
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, false));
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x142, 0xA, 0xF, false));  // row_bcast:15
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x143, 0xC, 0xF, false));  // row_bcast:31
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// The row's sum of N values a thread: over a wave, then over the row's waves by way of LDS (in wave order; `red` is the
// reduction's own, so one barrier does; what of it stands for waves that the workgroup has not is zero).
template <int MAXT, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[N]) {
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = wave_total(v[k]);
    if constexpr (MAXT > 64) {
        const int wave = (MAXT <= 256 ? threadIdx.x % MAXT : threadIdx.x) >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; k++) red[wave][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; k++) {
            float s = red[0][k];
#pragma unroll
            for (int w = 1; w < MAXT / 64; w++) s += red[w][k];
            v[k] = s;
        }
    }
}

__host__ __device__ __forceinline__ const void *row_at(const void *p, size_t row, int width, int dt) {
    return p ? static_cast<const char *>(p) + row * width * (dt == DT_F32 ? 4 : 2) : nullptr;
}
__host__ __device__ __forceinline__ void *row_at(void *p, size_t row, int width, int dt) {
    return p ? static_cast<char *>(p) + row * width * (dt == DT_F32 ? 4 : 2) : nullptr;
}

// A row's gate: 8 values of a thread.
template <int DT, bool WHOLE>
__device__ __forceinline__ void gate8(const void *gate, int kind, int gate_dtype, size_t row, uint32_t c, uint32_t width, float (&g)[8]) {
    if (kind == GATE_CHANNEL) load8_any<WHOLE>(gate, gate_dtype, c, width, g);
    else if (kind == GATE_FULL) load8<DT, WHOLE>(row_at(gate, row, width, DT), c, width, g);
    else {
        const float v = kind == GATE_ROW ? load_any(gate, gate_dtype, row) : 1.f;
#pragma unroll
        for (int q = 0; q < 8; q++) g[q] = v;
    }
}

// A row by TPR threads (a wave, or a workgroup of up to MAXT), each NV vectors of 8.
template <int DT, int HT, int MAXT, int NV, bool WHOLE>
__global__ __launch_bounds__(MAXT == 64 ? 256 : MAXT) void norm_kernel(NormArgs a) {
    const int TPR = MAXT == 64 ? 64 : blockDim.x, t = MAXT == 64 ? threadIdx.x & 63 : threadIdx.x;
    const size_t row = MAXT == 64 ? (size_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x;
    __shared__ float red[2][MAXT / 64][1];
    if (MAXT == 64 && row >= (size_t)a.rows) return;  // a wave's row; else the grid is the rows
    if (MAXT > 64) {
        if (threadIdx.x < 2 * MAXT / 64) (&red[0][0][0])[threadIdx.x] = 0.f;
        __syncthreads();
    }
    const void *y = row_at(a.y, row, a.width, DT), *h = row_at(a.h, row, a.width, HT);
    float n[NV][8], s[NV][8];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        load8<DT, WHOLE>(y, (uint32_t)(i * TPR + t) * 8, a.width, n[i]);
        if (h) load8<HT, WHOLE>(h, (uint32_t)(i * TPR + t) * 8, a.width, s[i]);
    }
    const float inv_width = 1.f / (float)a.width;
    float f = 1.f;
    if (a.post) {
        float sum[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int q = 0; q < 8; q++) sum[0] += n[i][q] * n[i][q];
        row_sum<MAXT, 1>(sum, red[0]);
        f = __builtin_amdgcn_rsqf(sum[0] * inv_width + a.eps);
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
        float w[8];
        if (a.post) {
            load8_any<WHOLE>(a.post, a.post_dtype, (uint32_t)(i * TPR + t) * 8, a.width, w);
#pragma unroll
            for (int q = 0; q < 8; q++) n[i][q] *= f * (a.offset + w[q]);
        }
        if (a.gate_kind != GATE_NONE) {
            gate8<DT, WHOLE>(a.gate, a.gate_kind, a.gate_dtype, row, (uint32_t)(i * TPR + t) * 8, a.width, w);
#pragma unroll
            for (int q = 0; q < 8; q++) n[i][q] *= w[q];
        }
#pragma unroll
        for (int q = 0; q < 8; q++) {
            n[i][q] *= a.block_scale;
            if (h) n[i][q] += a.residual_scale * s[i][q];
            sum[0] += n[i][q] * n[i][q];
        }
        store8<HT, WHOLE>(row_at(a.h_out, row, a.width, HT), (uint32_t)(i * TPR + t) * 8, a.width, n[i]);
    }
    if (!a.pre) return;
    row_sum<MAXT, 1>(sum, red[1]);
    f = __builtin_amdgcn_rsqf(sum[0] * inv_width + a.eps);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        float w[8];
        load8_any<WHOLE>(a.pre, a.pre_dtype, (uint32_t)(i * TPR + t) * 8, a.width, w);
#pragma unroll
        for (int q = 0; q < 8; q++) n[i][q] *= f * (a.offset + w[q]);
        store8<DT, WHOLE>(row_at(a.x_out, row, a.width, DT), (uint32_t)(i * TPR + t) * 8, a.width, n[i]);
    }
}

// The gradient.  A workgroup takes rows blockIdx.x, + gridDim.x, ..., with the next row's values in flight, and keeps its columns'
// sums (dpre, dpost, a channel gate's) in registers, up to 16 a thread, or in its part, and leaves them there for the join.
// TEAMS rows at a time where rows are narrow, MAXT threads each: as many rows in flight in fewer parts.
template <int DT, int HT, int MAXT, int NV, bool WHOLE, bool CHANNEL, int TEAMS>
__global__ __launch_bounds__(MAXT *TEAMS, NV == 1 && MAXT * TEAMS <= 512 && HT != DT_F32 && !CHANNEL ? 4 : 2) void norm_backward_kernel(NormGradArgs a) {
    constexpr bool REGS = NV <= 2, AHEAD = NV == 1;
    constexpr bool GATE_AHEAD = AHEAD && !CHANNEL && (WHOLE || MAXT != 512);  // (there 128 registers do not hold it)
    const int TPR = TEAMS > 1 ? MAXT : blockDim.x, t = TEAMS > 1 ? threadIdx.x % MAXT : threadIdx.x;
    const int team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / MAXT) : 0;
    __shared__ float reds[TEAMS][2][MAXT / 64][3], reds2[TEAMS][2][MAXT / 64][1];
    auto &red = reds[team];
    auto &red2 = reds2[team];
    if (MAXT > 64 && TEAMS == 1) {
        for (int i = t; i < 6 * MAXT / 64; i += TPR) (&red[0][0][0])[i] = 0.f;
        if (t < 2 * MAXT / 64) (&red2[0][0][0])[t] = 0.f;
        __syncthreads();
    }
    const float inv_width = 1.f / (float)a.width;
    const int gate_kind = CHANNEL ? GATE_CHANNEL : a.gate_kind;
    // this workgroup's sums, one after another as they are wanted
    const int sums = (a.pre != nullptr) + (a.post != nullptr) + CHANNEL;
    float *part = a.part + (size_t)blockIdx.x * sums * a.width;
    float *part_post = part + (a.pre ? a.width : 0), *part_gate = part_post + (a.post ? a.width : 0);
    using Acc = float[REGS ? NV : 1][8];
    Acc acc_pre = {}, acc_post = {}, acc_gate = {};
    bool first = true, live = true;  // (a team past the last row takes that row and leaves nothing of it)
    int flip = 0;
    const size_t rows = (size_t)a.rows, step = (size_t)gridDim.x * TEAMS;
    auto row_of = [&](size_t row0) { return TEAMS > 1 ? min(row0 + team, rows - 1) : row0; };
    auto col = [&](int i) { return (uint32_t)(i * TPR + t) * 8; };
    auto add = [&](Acc &acc, float *at, int i, const float (&v)[8]) {
        if constexpr (REGS) {
            if (TEAMS > 1 && !live) return;
#pragma unroll
            for (int q = 0; q < 8; q++) acc[i][q] += v[q];
        } else {
            float o[8];
            if (first) {
                store8<DT_F32, WHOLE>(at, col(i), a.width, v);
                return;
            }
            load8<DT_F32, WHOLE>(at, col(i), a.width, o);
#pragma unroll
            for (int q = 0; q < 8; q++) o[q] += v[q];
            store8<DT_F32, WHOLE>(at, col(i), a.width, o);
        }
    };
    // the weights with their offset, kept where a thread has eight columns (their loads follow the first row's)
    float wpre[8], wpost[8], wgate[8];
    auto pre_of = [&](int i) {
        if constexpr (AHEAD) return;
        load8_any<WHOLE>(a.pre, a.pre_dtype, col(i), a.width, wpre);
#pragma unroll
        for (int q = 0; q < 8; q++) wpre[q] += a.offset;
    };
    auto post_of = [&](int i) {
        if constexpr (AHEAD) return;
        if (a.post) load8_any<WHOLE>(a.post, a.post_dtype, col(i), a.width, wpost);
#pragma unroll
        for (int q = 0; q < 8; q++) wpost[q] = a.post ? wpost[q] + a.offset : 1.f;
    };
    struct Row {
        Raw8<DT> y[NV], dx[REGS ? NV : 1];
        Raw8<HT> dh[1], h[REGS ? NV : 1];
        Raw8<DT> gate[1];  // like y
    };
    auto fetch = [&](size_t row, Row &r) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            load_raw<DT, WHOLE>(row_at(a.y, row, a.width, DT), col(i), a.width, r.y[i]);
            if (AHEAD && a.dh) load_raw<HT, WHOLE>(row_at(a.dh, row, a.width, HT), col(i), a.width, r.dh[0]);
            if (GATE_AHEAD && gate_kind == GATE_FULL)
                load_raw<DT, WHOLE>(row_at(a.gate, row, a.width, DT), col(i), a.width, r.gate[0]);
            if (REGS && a.pre) {
                load_raw<HT, WHOLE>(row_at(a.h, row, a.width, HT), col(i), a.width, r.h[i % (REGS ? NV : 1)]);
                load_raw<DT, WHOLE>(row_at(a.dx, row, a.width, DT), col(i), a.width, r.dx[i % (REGS ? NV : 1)]);
            }
        }
    };
    Row now;
    if constexpr (AHEAD) {
        fetch(row_of((size_t)blockIdx.x * TEAMS), now);
        RawAny pre, post, gate;
        if (a.pre) pre.load_row<WHOLE>(a.pre, a.pre_dtype, col(0), a.width);
        if (a.post) post.load_row<WHOLE>(a.post, a.post_dtype, col(0), a.width);
        if (CHANNEL) gate.load_row<WHOLE>(a.gate, a.gate_dtype, col(0), a.width);
        if (a.pre) pre.settle<WHOLE>(a.pre_dtype, col(0), a.width), pre.get(a.pre_dtype, a.offset, wpre);
        if (a.post) post.settle<WHOLE>(a.post_dtype, col(0), a.width), post.get(a.post_dtype, a.offset, wpost);
        else
#pragma unroll
            for (int q = 0; q < 8; q++) wpost[q] = 1.f;
        if (CHANNEL) gate.settle<WHOLE>(a.gate_dtype, col(0), a.width), gate.get(a.gate_dtype, 0.f, wgate);
    }
    for (size_t row0 = (size_t)blockIdx.x * TEAMS; row0 < rows; row0 += step, first = false, flip ^= 1) {
        const size_t row = row_of(row0);
        live = TEAMS == 1 || row0 + team < rows;
        auto again = [&](int i) -> int {  // where vector i of h and dx is
            if constexpr (REGS) return i;
            load_raw<HT, WHOLE>(row_at(a.h, row, a.width, HT), col(i), a.width, now.h[0]);
            load_raw<DT, WHOLE>(row_at(a.dx, row, a.width, DT), col(i), a.width, now.dx[0]);
            settle<HT, WHOLE>(col(i), a.width, now.h[0]);
            settle<DT, WHOLE>(col(i), a.width, now.dx[0]);
            return 0;
        };
        if constexpr (!AHEAD) fetch(row, now);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            settle<DT, WHOLE>(col(i), a.width, now.y[i]);
            if (AHEAD && a.dh) settle<HT, WHOLE>(col(i), a.width, now.dh[0]);
            if (GATE_AHEAD && gate_kind == GATE_FULL) settle<DT, WHOLE>(col(i), a.width, now.gate[0]);
            if (REGS && a.pre) {
                settle<HT, WHOLE>(col(i), a.width, now.h[i % (REGS ? NV : 1)]);
                settle<DT, WHOLE>(col(i), a.width, now.dx[i % (REGS ? NV : 1)]);
            }
        }
        const float row_gate = gate_kind == GATE_ROW ? load_any(a.gate, a.gate_dtype, row) : 1.f;
        Raw8<DT> y[NV];
        float H[NV][8];
        auto now_y = [&](int i, int q) { return y[i].get(q); };
        float s[3] = {0.f, 0.f, 0.f};  // of h'^2, u h', y^2
#pragma unroll
        for (int i = 0; i < NV; i++) {
#pragma unroll
            for (int q = 0; q < 8; q++) H[i][q] = AHEAD && a.dh ? now.dh[0].get(q) : 0.f;
            if (!AHEAD && a.dh) load8<HT, WHOLE>(row_at(a.dh, row, a.width, HT), col(i), a.width, H[i]);
            y[i] = now.y[i];
            if (a.pre) {
                const int k = again(i);
                pre_of(i);
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float h = now.h[k].get(q);
                    s[0] += h * h;
                    s[1] += now.dx[k].get(q) * wpre[q] * h;
                }
            }
            if (a.post)
#pragma unroll
                for (int q = 0; q < 8; q++) s[2] += now_y(i, q) * now_y(i, q);
        }
        // (a row's h and dx leave for good below where they are kept, so that the next row's may come)
        Raw8<HT> h1 = now.h[0];
        Raw8<DT> dx1 = now.dx[0], gate1 = now.gate[0];
        if constexpr (AHEAD) {
            if (row0 + step < rows) fetch(row_of(row0 + step), now);
        }
        if (a.pre || a.post) row_sum<MAXT, 3>(s, red[flip]);
        const float r = a.pre ? __builtin_amdgcn_rsqf(s[0] * inv_width + a.eps) : 0.f;
        const float along = r * r * (s[1] * inv_width);
        const float qf = a.post ? __builtin_amdgcn_rsqf(s[2] * inv_width + a.eps) : 1.f;
        float s2[1] = {0.f};  // of v y
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float d[8];
            if (a.pre) {
                const int k = AHEAD ? 0 : again(i);
                pre_of(i);
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float h = AHEAD ? h1.get(q) : now.h[k].get(q), dx = AHEAD ? dx1.get(q) : now.dx[k].get(q);
                    H[i][q] += r * (dx * wpre[q] - h * along);
                    d[q] = dx * (h * r);
                }
                add(acc_pre, part, i, d);
            }
            if (a.dres && live) {
#pragma unroll
                for (int q = 0; q < 8; q++) d[q] = a.residual_scale * H[i][q];
                store8<HT, WHOLE>(row_at(a.dres, row, a.width, HT), col(i), a.width, d);
            }
            post_of(i);
#pragma unroll
            for (int q = 0; q < 8; q++) H[i][q] *= a.block_scale;
            if (CHANNEL || gate_kind == GATE_FULL) {
                float g[8];
                if constexpr (CHANNEL && AHEAD) {
#pragma unroll
                    for (int q = 0; q < 8; q++) g[q] = wgate[q];
                } else if constexpr (GATE_AHEAD) {
#pragma unroll
                    for (int q = 0; q < 8; q++) g[q] = gate1.get(q);
                } else {
                    gate8<DT, WHOLE>(a.gate, gate_kind, a.gate_dtype, row, col(i), a.width, g);
                }
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    d[q] = H[i][q] * (now_y(i, q) * qf * wpost[q]);
                    H[i][q] *= g[q];
                }
                if (CHANNEL) add(acc_gate, part_gate, i, d);
                else if (live) store8<DT, WHOLE>(row_at(a.dgate, row, a.width, DT), col(i), a.width, d);
            }
            if (a.post) {
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    d[q] = H[i][q] * (now_y(i, q) * (qf * row_gate));
                    H[i][q] *= wpost[q];  // v, but for the row's gate
                    s2[0] += H[i][q] * now_y(i, q);
                }
                add(acc_post, part_post, i, d);
            } else if (gate_kind == GATE_ROW) {
#pragma unroll
                for (int q = 0; q < 8; q++) s2[0] += H[i][q] * now_y(i, q);
            }
        }
        if (a.post || gate_kind == GATE_ROW) row_sum<MAXT, 1>(s2, red2[flip]);
        // (a row's gate is a factor of the whole row: its gradient and the mean come of one sum)
        if (gate_kind == GATE_ROW && t == 0 && live) static_cast<float *>(a.dgate)[row] = s2[0] * qf;
        const float along_y = qf * qf * (s2[0] * inv_width), out = qf * row_gate;
#pragma unroll
        for (int i = 0; i < NV; i++) {
#pragma unroll
            for (int q = 0; q < 8; q++) H[i][q] = out * (a.post ? H[i][q] - now_y(i, q) * along_y : H[i][q]);
            if (live) store8<DT, WHOLE>(row_at(a.dy, row, a.width, DT), col(i), a.width, H[i]);
        }
    }
    if constexpr (TEAMS > 1) {  // the teams' sums, in order
        __shared__ __align__(16) float fold[TEAMS][MAXT * 8];
        auto join = [&](const float (&acc)[8], float *to) {
            store8<DT_F32, WHOLE>(fold[team], col(0), a.width, acc);
            __syncthreads();
            for (int c = threadIdx.x; c < a.width; c += MAXT * TEAMS) {
                float s = fold[0][c];
#pragma unroll
                for (int k = 1; k < TEAMS; k++) s += fold[k][c];
                to[c] = s;
            }
            __syncthreads();
        };
        if (a.pre) join(acc_pre[0], part);
        if (a.post) join(acc_post[0], part_post);
        if (CHANNEL) join(acc_gate[0], part_gate);
    } else if constexpr (REGS) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (a.pre) store8<DT_F32, WHOLE>(part, col(i), a.width, acc_pre[i]);
            if (a.post) store8<DT_F32, WHOLE>(part_post, col(i), a.width, acc_post[i]);
            if (CHANNEL) store8<DT_F32, WHOLE>(part_gate, col(i), a.width, acc_gate[i]);
        }
    }
}

// A column's sum over the parts: the lanes of a wave hold 64 columns, the workgroup's waves a share of the parts each, in
// order, NJ_AHEAD loads at a time; the shares add in wave order.
constexpr int NJ_WAVES = 16, NJ_AHEAD = 16;
__global__ __launch_bounds__(64 * NJ_WAVES) void norm_join_kernel(const float *part, int parts, int sums, int width, float *d0, float *d1,
                                                                  float *d2) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, total = sums * width, c = blockIdx.x * 64 + lane;
    __shared__ float share[NJ_WAVES][64];
    const float *at = part + min(c, total - 1);
    float s = 0.f;
    for (int p0 = wave; p0 < parts; p0 += NJ_WAVES * NJ_AHEAD) {
        float v[NJ_AHEAD];
#pragma unroll
        for (int i = 0; i < NJ_AHEAD; i++) v[i] = at[(size_t)min(p0 + i * NJ_WAVES, parts - 1) * total];
#pragma unroll
        for (int i = 0; i < NJ_AHEAD; i++) s += p0 + i * NJ_WAVES < parts ? v[i] : 0.f;
    }
    share[wave][lane] = s;
    __syncthreads();
    if (wave || c >= total) return;
    for (int w = 1; w < NJ_WAVES; w++) s += share[w][lane];
    const int k = c / width;
    (k == 0 ? d0 : k == 1 ? d1 : d2)[c - k * width] = s;
}

template <class F>
static hipError_t with_types(int dt, int ht, F f) {
    using std::integral_constant;
    if (dt == DT_F32) return f(integral_constant<int, DT_F32>{}, integral_constant<int, DT_F32>{});
    if (dt == DT_F16)
        return ht == DT_F32 ? f(integral_constant<int, DT_F16>{}, integral_constant<int, DT_F32>{})
                            : f(integral_constant<int, DT_F16>{}, integral_constant<int, DT_F16>{});
    return ht == DT_F32 ? f(integral_constant<int, DT_BF16>{}, integral_constant<int, DT_F32>{})
                        : f(integral_constant<int, DT_BF16>{}, integral_constant<int, DT_BF16>{});
}

// The threads of a row of `width` values at nv vectors each, in whole waves.
static int row_threads(int width, int nv) { return (width + 512 * nv - 1) / (512 * nv) * 64; }

static hipError_t launch_norm(const NormArgs &a, hipStream_t s) {
    return with_types(a.dtype, a.hdtype, [&](auto DT, auto HT) {
        constexpr int dt = decltype(DT)::value, ht = decltype(HT)::value;
        auto go = [&](auto MAXT, auto NV) {
            constexpr int maxt = decltype(MAXT)::value, nv = decltype(NV)::value;
            const dim3 grid((unsigned)(maxt == 64 ? ((long)a.rows + 3) / 4 : a.rows)), block(maxt == 64 ? 256 : row_threads(a.width, nv));
            if (a.width % 8 == 0) hipLaunchKernelGGL((norm_kernel<dt, ht, maxt, nv, true>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((norm_kernel<dt, ht, maxt, nv, false>), grid, block, 0, s, a);
            return hipGetLastError();
        };
        using std::integral_constant;
        if (a.width <= 512) return go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
        if (a.width <= 2048) return go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
        if (a.width <= 8192) return go(integral_constant<int, 512>{}, integral_constant<int, 2>{});
        return go(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
    });
}

// A launch takes up to 2^21 rows (its threads are numbered in 32 bits).
hipError_t run_norm(const NormArgs &a, hipStream_t s) {
    constexpr int most = 1 << 21;
    for (int r = 0; r < a.rows; r += std::min(most, a.rows - r)) {
        NormArgs c = a;
        c.rows = std::min(most, a.rows - r);
        c.y = row_at(a.y, r, a.width, a.dtype);
        c.h = row_at(a.h, r, a.width, a.hdtype);
        c.h_out = row_at(a.h_out, r, a.width, a.hdtype);
        c.x_out = row_at(a.x_out, r, a.width, a.dtype);
        if (a.gate_kind == GATE_ROW || a.gate_kind == GATE_FULL)
            c.gate = row_at(a.gate, r, a.gate_kind == GATE_ROW ? 1 : a.width, a.gate_dtype);
        const hipError_t e = launch_norm(c, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Rows of up to 2048 values go by teams of one, two or four waves, eight waves a workgroup: with a workgroup a row there would be
// four times the parts for as many rows in flight (8192 bf16 rows of 512 / 680 values: 20.0 / 24.4 us, by teams 13.7 / 19.6).
constexpr int backward_teams(int width) { return width <= 512 ? 8 : width <= 1024 ? 4 : width <= 2048 ? 2 : 1; }

// Workgroups of the gradient.  More of them hide a row's latency (1.0 us a row of 512 values, 1.5 of 4096, its loads ahead) and
// leave more parts to the join.  One a CU; two where both fit on it by their registers (without an f32 stream and a channel gate)
// and there are rows enough, each the same number of rows.  us in a graph at 256 / 512 / 1024 workgroups, bf16 with both norms:
// 8192 rows of 200 values 12.2 / 12.3 / 14.9, 16384 of 512 20.0 / 19.2 / 22.7; 2048 of 680 10.3 / 11.0 / 11.0, 8192 of 680
// 22.2 / 19.6 / 23.0; 333 rows of 4096 11.5 / 14.7 / -, 2048 rows 23.9 / 22.4 / 28.7, 8192 rows 65.8 / 62.2 / 66.1; 8192 rows of
// 6144 90.1 / 94.2 / 106.3; f32, 8192 rows of 1024 29.4 / 32.4 / 38.6.
static int backward_workgroups(int rows, int width, bool two) {
    const int teams = backward_teams(width), sets = (int)(((long)rows + teams - 1) / teams);
    const bool many = rows >= (width <= 512 ? 16384 : width <= 2048 ? 4096 : 2048) && width <= 4096;
    return std::min(sets, two && many ? 512 : 256);
}
int norm_backward_most(int rows, int width) { return backward_workgroups(rows, width, true); }
int norm_backward_parts(const NormGradArgs &a) {
    const int teams = backward_teams(a.width), sets = (int)(((long)a.rows + teams - 1) / teams);
    const int most = backward_workgroups(a.rows, a.width, a.hdtype != DT_F32 && a.gate_kind != GATE_CHANNEL);
    const int each = most ? (sets + most - 1) / most : 1;
    return (sets + each - 1) / each;
}

hipError_t run_norm_backward(const NormGradArgs &a, hipStream_t s) {
    hipError_t e = with_types(a.dtype, a.hdtype, [&](auto DT, auto HT) {
        constexpr int dt = decltype(DT)::value, ht = decltype(HT)::value;
        const bool whole = a.width % 8 == 0;
        auto go = [&](auto MAXT, auto NV) {
            constexpr int maxt = decltype(MAXT)::value, nv = decltype(NV)::value, teams = maxt <= 256 ? 512 / maxt : 1;
            auto kernel = [&](auto WHOLE, auto CHANNEL) {
                hipLaunchKernelGGL((norm_backward_kernel<dt, ht, maxt, nv, decltype(WHOLE)::value, decltype(CHANNEL)::value, teams>),
                                   dim3(a.parts), dim3(teams > 1 ? maxt * teams : row_threads(a.width, nv)), 0, s, a);
                return hipGetLastError();
            };
            using std::true_type, std::false_type;
            if constexpr (!(maxt == 768 && ht == DT_F32))
                if (!whole) return a.gate_kind == GATE_CHANNEL ? kernel(false_type{}, true_type{}) : kernel(false_type{}, false_type{});
            return a.gate_kind == GATE_CHANNEL ? kernel(true_type{}, true_type{}) : kernel(true_type{}, false_type{});
        };
        using std::integral_constant;
        if (a.width <= 512) return go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
        if (a.width <= 1024) return go(integral_constant<int, 128>{}, integral_constant<int, 1>{});
        if (a.width <= 2048) return go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
        if (a.width <= 4096) return go(integral_constant<int, 512>{}, integral_constant<int, 1>{});
        // (rows with an f32 stream that end inside a vector want more than the 168 registers of 12 waves)
        if (a.width <= 6144 && (whole || ht != DT_F32)) return go(integral_constant<int, 768>{}, integral_constant<int, 1>{});
        // (without the next row's loads ahead; past 8192 values the sums are kept in the part, and h and dx read twice: 8192 bf16
        // rows of 8192 / 16384 values take 198 / 654 us, 156 and 312 for the bytes)
        if (a.width <= 8192) return go(integral_constant<int, 512>{}, integral_constant<int, 2>{});
        return go(integral_constant<int, 512>{}, integral_constant<int, 4>{});
    });
    if (e != hipSuccess) return e;
    float *to[3], **next = to;
    if (a.pre) *next++ = a.dpre;
    if (a.post) *next++ = a.dpost;
    if (a.gate_kind == GATE_CHANNEL) *next++ = static_cast<float *>(a.dgate);
    const int sums = (int)(next - to);
    if (!sums) return hipSuccess;
    for (int k = sums; k < 3; k++) to[k] = to[0];
    hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)((sums * a.width + 63) / 64)), dim3(64 * NJ_WAVES), 0, s, a.part, a.parts, sums,
                       a.width, to[0], to[1], to[2]);
    return hipGetLastError();
}

}  // namespace exl3
