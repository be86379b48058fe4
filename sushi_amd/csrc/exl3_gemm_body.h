// (Kernels shared by exl3_gemm.hip and exl3_gemm_epilogue.hip.)
// Dense trellis GEMM for wide row counts (the prefill arm of linear.linear: prepareIndexed +
// innerGemmSortedTable + finishIndexedAs, beamivalice/sushi src/exl3/linear.zig:322-335 and
// src/exl3/expert_exl3_kernels.zig:1341-1620).
//
// MI355X layout.  A workgroup of 2 waves owns a 128-row x 128-column output tile (one Hadamard block wide, so
// the output FWHT + svh finish runs in its epilogue) over the whole k range, in k-steps of 32 (two trellis
// k-tiles).  The prepared input rows are staged through LDS; each wave owns 64 output columns (4 trellis tiles)
// and decodes its weights straight into v_mfma_f32_16x16x32_f16 B fragments: lane l = 16h + c needs column c of a
// 16-column block at k = 8h..8h+7, which is the codeword set {8q + 2p + e} (q = 0..3, e = 0..1) of chunk j = c % 8
// with p = 2*(c / 8) + h % 2 (tensorCorePerm), i.e. eight codewords from one 2n-bit run of the tile stream.
// Integer rates (n = 16K) use this reader; other rates are first decoded to a transposed f16 copy in workspace.
#pragma once
#include "exl3_gemm_tile.h"
#include "exl3_epilogue.h"

namespace exl3 {

constexpr int GM_WAVES = 2;
constexpr int GM_THREADS = 64 * GM_WAVES;
constexpr int GM_MT = 128;    // rows per workgroup
constexpr int GM_XP = 40;     // LDS pitch (halves) of a staged x row: 32 + 8 pad

// ---- prepare: xp[g][r][:] = f16(H128(f16(x) * suh) / sqrt(128))  (prepareIndexed / PREPARE_SOURCE :852-885)
static __global__ __launch_bounds__(64) void gemm_prepare_kernel(GemmArgs a) {
    const int b = blockIdx.x, r = blockIdx.y, g = blockIdx.z, lane = threadIdx.x;
    const size_t xi = ((size_t)g * a.rows + r) * a.in + (size_t)b * 128;
    const size_t si = (size_t)g * a.in + (size_t)b * 128;
    float v0, v1;
    if (a.x_dtype == DT_F16) {
        v0 = load_act<DT_F16>(a.x, xi + lane);
        v1 = load_act<DT_F16>(a.x, xi + lane + 64);
    } else if (a.x_dtype == DT_BF16) {
        v0 = f16r(load_act<DT_BF16>(a.x, xi + lane));
        v1 = f16r(load_act<DT_BF16>(a.x, xi + lane + 64));
    } else {
        v0 = f16r(load_act<DT_F32>(a.x, xi + lane));
        v1 = f16r(load_act<DT_F32>(a.x, xi + lane + 64));
    }
    v0 *= h2f(a.suh[si + lane]);
    v1 *= h2f(a.suh[si + lane + 64]);
    fwht128_wave(v0, v1, lane);
    a.xp[xi + lane] = __half_as_ushort(__float2half_rn(v0 * HAD_SCALE));
    a.xp[xi + lane + 64] = __half_as_ushort(__float2half_rn(v1 * HAD_SCALE));
}

// ---- prepare into MFMA A-fragment order: for 16-row tile rt and 32-k block kb of group g, the 1 KiB at
// xp[((g * RT + rt) * (in / 32) + kb) * 512] holds lane l = 16h + c's fragment (row 16 rt + c, k = 32 kb + 8h .. +7)
// at l * 8 halves, so one MFMA wave's load of a fragment is one contiguous 1 KiB.  RT = ceil(rows / 16); rows past
// the end of the last tile are zeros.  A workgroup (4 waves) prepares 16 rows x NB 128-blocks (two where they pair
// up): each wave loads its 4 rows of every block at once and runs their FWHTs together into an LDS tile, then every
// thread writes one 16-byte fragment per block.
template <int DT, int NB>
__global__ __launch_bounds__(256) void gemm_prepare_frag_kernel(GemmArgs a) {
    const int b0 = blockIdx.x * NB, rt = blockIdx.y, g = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int RT = (a.rows + 15) / 16;
    __shared__ __align__(16) uint16_t t[NB][16][128 + 8];
    const int m0 = rt * 16 + wave * 4;
    // every load in bounds (a row past the end reads the last row and is zeroed after), so a wave's four rows of
    // every block go out together with suh, with no branch to wait at
    float v0[NB][4], v1[NB][4], u0[NB], u1[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const size_t si = (size_t)g * a.in + (size_t)(b0 + nb) * 128;
        u0[nb] = h2f(a.suh[si + lane]);
        u1[nb] = h2f(a.suh[si + lane + 64]);
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const size_t xi = ((size_t)g * a.rows + min(m0 + rr, a.rows - 1)) * a.in + (size_t)(b0 + nb) * 128;
            v0[nb][rr] = load_act<DT>(a.x, xi + lane);
            v1[nb][rr] = load_act<DT>(a.x, xi + lane + 64);
        }
    }
    const float sc = fwht_relaid_sign(lane) * HAD_SCALE;
    const int c0 = fwht_relaid_col(lane, 0), c1 = fwht_relaid_col(lane, 1);
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const bool live = m0 + rr < a.rows;
            v0[nb][rr] = live ? f16r(v0[nb][rr]) * u0[nb] : 0.f;
            v1[nb][rr] = live ? f16r(v1[nb][rr]) * u1[nb] : 0.f;
        }
        fwht128_wave_rows_relaid<4>(v0[nb], v1[nb], lane);
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const int r = wave * 4 + rr;
            t[nb][r][c0] = __half_as_ushort(__float2half_rn(v0[nb][rr] * sc));
            t[nb][r][c1] = __half_as_ushort(__float2half_rn(v1[nb][rr] * sc));
        }
    }
    __syncthreads();
    const int kq = tid >> 6, c = lane & 15, h = lane >> 4;  // 32-k block kq of a 128-block, fragment lane (c, h)
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        const uint4 v = *reinterpret_cast<const uint4 *>(&t[nb][c][kq * 32 + 8 * h]);
        const size_t kb = (size_t)(b0 + nb) * 4 + kq;
        *reinterpret_cast<uint4 *>(a.xp + (((size_t)g * RT + rt) * (a.in / 32) + kb) * 512 + (size_t)lane * 8) = v;
    }
}

template <int DT>
static void launch_gemm_prepare_frag(const GemmArgs &a, hipStream_t s) {
    const int blocks = a.in / 128;
    const dim3 grid2((unsigned)(blocks / 2), (unsigned)((a.rows + 15) / 16), (unsigned)a.groups);
    const dim3 grid1((unsigned)blocks, (unsigned)((a.rows + 15) / 16), (unsigned)a.groups);
    if (blocks % 2 == 0) hipLaunchKernelGGL((gemm_prepare_frag_kernel<DT, 2>), grid2, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((gemm_prepare_frag_kernel<DT, 1>), grid1, dim3(256), 0, s, a);
}

// ---- dense fallback: tiles decoded to wt[g][out][in] f16 (transposed, so a B fragment is 16 contiguous bytes)
template <int FAM>
__global__ void gemm_decode_transposed_kernel(GemmArgs a, uint16_t *__restrict__ wt) {
    const int IT = a.in >> 4, OT = a.out >> 4;
    const int tile = blockIdx.x, g = blockIdx.y;
    const int tk = tile / OT, tn = tile % OT;
    const uint32_t *words =
        reinterpret_cast<const uint32_t *>(a.trellis + ((size_t)g * IT * OT + (size_t)tile) * a.n);
    const int t = 2 * threadIdx.x;
    uint32_t h = decode_pair_h2<FAM>(codeword_at(words, a.n, t), codeword_at(words, a.n, t + 1), a.k);
    const int T = t >> 3, i = t & 7, q = T & 3, j = T >> 2;
    const int row = 2 * q + ((i & 2) ? 8 : 0);
    const int col = j + ((i & 4) ? 8 : 0);
    uint32_t *dst = reinterpret_cast<uint32_t *>(wt + ((size_t)g * a.out + (size_t)tn * 16 + col) * a.in +
                                                 (size_t)tk * 16 + row);
    *dst = h;  // rows (row, row+1) of one column are adjacent in the transposed copy
}

template <int FAM, int N, bool EPI>
__device__ __forceinline__ void gemm_run(const GemmArgs &a, const uint16_t *__restrict__ wt, const EpilogueArgs *e) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int IT = a.in >> 4, OT = a.out >> 4;
    const int og = blockIdx.x, mb = blockIdx.y, g = blockIdx.z;
    const int m0 = mb * GM_MT;

    __shared__ __align__(16) uint16_t xs[GM_MT * GM_XP];
    __shared__ float outs[32][129];

    const int c = lane & 15, h = lane >> 4;
    const int kt_off = h >> 1, half = h & 1, j = c & 7, p = 2 * (c >> 3) + half;
    const DecodeK k = a.k;
    const uint16_t *tb = a.trellis + (size_t)g * IT * OT * a.n;

    f4_t acc[8][4];
#pragma unroll
    for (int rb = 0; rb < 8; rb++)
#pragma unroll
        for (int cb = 0; cb < 4; cb++) acc[rb][cb] = f4_t{0.f, 0.f, 0.f, 0.f};

    // Per-lane bit base of its eight codewords inside a tile: codeword (q, e) ends 32 + (e+1)K + q*n/2 bits past it.
    constexpr int K = N ? N / 16 : 1;
    constexpr int NW = N ? N / 2 : 1;
    constexpr int AW = N ? (32 + 2 * K + 3 * (N / 2) + 16 + 31) / 32 + 1 : 1;  // words covering the span, +1 to funnel
    const int span = 16 * (N ? N : 16);
    const int base = ((2 * j * (N ? N : 16) - 32 + 2 * p * K) % span + span) % span;
    const int wb = base >> 5, sb = base & 31;

    const int nks = IT / 2;
    for (int ks = 0; ks < nks; ks++) {
        // stage 128 rows x 32 k of the prepared input
        __syncthreads();
        {
            const int row = tid;  // GM_THREADS == GM_MT
            const int m = m0 + row;
            uint4 v0 = {0, 0, 0, 0}, v1 = v0, v2 = v0, v3 = v0;
            if (m < a.rows) {
                const uint4 *src = reinterpret_cast<const uint4 *>(a.xp + ((size_t)g * a.rows + m) * a.in + ks * 32);
                v0 = src[0];
                v1 = src[1];
                v2 = src[2];
                v3 = src[3];
            }
            uint4 *dst = reinterpret_cast<uint4 *>(&xs[row * GM_XP]);
            dst[0] = v0;
            dst[1] = v1;
            dst[2] = v2;
            dst[3] = v3;
        }
        // B fragments for this wave's 4 column blocks
        uint32_t B[4][4];
        const int tk = 2 * ks + kt_off;
#pragma unroll
        for (int cb = 0; cb < 4; cb++) {
            const int o = og * 8 + wave * 4 + cb;
            if constexpr (N != 0) {
                const uint32_t *words = reinterpret_cast<const uint32_t *>(tb + ((size_t)tk * OT + o) * N);
                uint32_t R[AW];
#pragma unroll
                for (int i = 0; i < AW; i++) R[i] = words[(wb + i) % NW];
                uint32_t A[AW - 1];
#pragma unroll
                for (int i = 0; i < AW - 1; i++) A[i] = sb ? __builtin_amdgcn_alignbit(R[i], R[i + 1], 32 - sb) : R[i];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t cw[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int end = 32 + (e + 1) * K + q * (N / 2);
                        const int aw = (end - 1) >> 5;
                        const int sh = 32 * (aw + 1) - end;
                        cw[e] = aw == 0 ? (A[0] >> sh) : __builtin_amdgcn_alignbit(A[aw - 1], A[aw], sh);
                    }
                    B[cb][q] = decode_pair_h2<FAM>(cw[0], cw[1], k);
                }
            } else {
                const uint4 v = *reinterpret_cast<const uint4 *>(
                    wt + ((size_t)g * a.out + (size_t)o * 16 + c) * a.in + (size_t)tk * 16 + 8 * half);
                B[cb][0] = v.x;
                B[cb][1] = v.y;
                B[cb][2] = v.z;
                B[cb][3] = v.w;
            }
        }
        __syncthreads();
#pragma unroll
        for (int rb = 0; rb < 8; rb++) {
            const uint4 av = *reinterpret_cast<const uint4 *>(&xs[(rb * 16 + c) * GM_XP + 8 * h]);
            const h8_t A8 = __builtin_bit_cast(h8_t, av);
#pragma unroll
            for (int cb = 0; cb < 4; cb++) {
                const uint4 bv = {B[cb][0], B[cb][1], B[cb][2], B[cb][3]};
                acc[rb][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A8, __builtin_bit_cast(h8_t, bv), acc[rb][cb], 0,
                                                                     0, 0);
            }
        }
    }

    // ---- epilogue: 32-row chunks through LDS, then FWHT-128 + svh per row
    const size_t sv = (size_t)g * a.out + (size_t)og * 128;
#pragma unroll
    for (int ch = 0; ch < 4; ch++) {
        __syncthreads();
#pragma unroll
        for (int rr = 0; rr < 2; rr++) {
            const int rb = ch * 2 + rr;
#pragma unroll
            for (int cb = 0; cb < 4; cb++)
#pragma unroll
                for (int i = 0; i < 4; i++) outs[rr * 16 + 4 * h + i][wave * 64 + cb * 16 + c] = acc[rb][cb][i];
        }
        __syncthreads();
        for (int r = wave; r < 32; r += GM_WAVES) {
            const int m = m0 + ch * 32 + r;
            if (m >= a.rows) break;
            float v0 = outs[r][lane], v1 = outs[r][lane + 64];
            fwht128_wave(v0, v1, lane);
            const size_t yo = ((size_t)g * a.rows + m) * a.out + (size_t)og * 128;
            float y0 = v0 * codebook_scale<FAM>() * HAD_SCALE * h2f(a.svh[sv + lane]);
            float y1 = v1 * codebook_scale<FAM>() * HAD_SCALE * h2f(a.svh[sv + lane + 64]);
            if constexpr (EPI) {
                const size_t col = (size_t)og * 128 + lane;
                const EpilogueWords w = epilogue_fetch(*e, a.y_dtype, col, yo + lane);
                y0 = epilogue_apply(*e, a.y_dtype, y0, w.b0, col, w.r0, yo + lane);
                y1 = epilogue_apply(*e, a.y_dtype, y1, w.b1, col + 64, w.r1, yo + lane + 64);
            }
            if (a.y_dtype == DT_F16) {
                store_act<DT_F16>(a.y, yo + lane, y0);
                store_act<DT_F16>(a.y, yo + lane + 64, y1);
            } else if (a.y_dtype == DT_BF16) {
                store_act<DT_BF16>(a.y, yo + lane, y0);
                store_act<DT_BF16>(a.y, yo + lane + 64, y1);
            } else {
                store_act<DT_F32>(a.y, yo + lane, y0);
                store_act<DT_F32>(a.y, yo + lane + 64, y1);
            }
        }
    }
}

template <int FAM, int N>
__global__ __launch_bounds__(GM_THREADS) void gemm_kernel(GemmArgs a, const uint16_t *__restrict__ wt) {
    gemm_run<FAM, N, false>(a, wt, nullptr);
}
template <int FAM, int N>
__global__ __launch_bounds__(GM_THREADS) void gemm_epilogue_kernel(GemmArgs a, const uint16_t *__restrict__ wt,
                                                                   EpilogueArgs e) {
    gemm_run<FAM, N, true>(a, wt, &e);
}

// Columns i and i + 64 (v[2 r], v[2 r + 1]) of the first `live` of four rows `pitch` elements apart, in dtype dt.
__device__ __forceinline__ void store_rows4(void *p, int dt, size_t i, size_t pitch, int live, const float (&v)[8]) {
    if (dt == DT_F32) {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (r < live) {
                store_act<DT_F32>(p, i + r * pitch, v[2 * r]);
                store_act<DT_F32>(p, i + r * pitch + 64, v[2 * r + 1]);
            }
        return;
    }
    const uint4 w = pack8(dt == DT_BF16, v);
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    uint16_t *q = static_cast<uint16_t *>(p) + i;
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (r < live) {
            q[r * pitch] = (uint16_t)ws[r];
            q[r * pitch + 64] = (uint16_t)(ws[r] >> 16);
        }
}

// EPI: with the epilogue e.  The bias words are fetched once; the residual's words of four rows go out together, while the
// four rows before them are finished.
template <int FAM, int N, bool EPI>
__device__ __forceinline__ void gemm4_run(const GemmArgs &a, const EpilogueArgs *e) {
    const int IT = a.in >> 4, OT = a.out >> 4;
    const int nog = a.out / 128, nm = (a.rows + G2_MT - 1) / G2_MT;
    const int L = blockIdx.x;
    int og, mt;
    if (nm <= 8 && 8 % nm == 0 && nog % (8 / nm) == 0) {
        const int xcd = L & 7, per = 8 / nm;
        mt = xcd / per;
        og = (L >> 3) * per + xcd % per;
    } else {
        og = L % nog;
        mt = L / nog;
    }
    const int g = blockIdx.z;
    constexpr int SLABS = 2 * 128 * G4_BP;  // halves
    __shared__ __align__(16) uint16_t lds[EPI && G4_STAGE_ALL / 2 > SLABS ? G4_STAGE_ALL / 2 : SLABS];
    uint16_t (*Bs)[128 * G4_BP] = reinterpret_cast<uint16_t (*)[128 * G4_BP]>(lds);
    const int RT = (a.rows + 15) / 16;
    const uint16_t *xfrag0 = a.xp + ((size_t)g * RT + (size_t)mt * (G2_MT / 16)) * (size_t)(a.in / 32) * 512;
    const size_t sv = (size_t)g * a.out + (size_t)og * 128;
    const int lane = threadIdx.x & 63;
    const float s0 = h2f(a.svh[sv + lane]), s1 = h2f(a.svh[sv + lane + 64]);
    const int tile_rows = min(G2_MT, a.rows - mt * G2_MT);
    uint32_t next0[4] = {}, next1[4] = {};  // EPI: the residual's words of the next four rows
    bool fetched = false;
    gemm4_tile<FAM, N, EPI>(a.in, a.out, og, a.trellis + (size_t)g * IT * OT * N, xfrag0, min(G2_MT, a.rows - mt * G2_MT),
                       nullptr, a.k, Bs,
                       [&](int m, int live, float (&v0)[4], float (&v1)[4], int ln, uint32_t)
                           __attribute__((always_inline)) {
                           if constexpr (EPI) {
                               const size_t col = (size_t)og * 128 + ln;
                               auto fetch = [&](int m4) __attribute__((always_inline)) {
#pragma unroll
                                   for (int i = 0; i < 4; i++) {
                                       const size_t o = ((size_t)mt * G2_MT + min(m4 + i, tile_rows - 1)) * a.out + col;
                                       next0[i] = act_word(e->residual, a.y_dtype, o);
                                       next1[i] = act_word(e->residual, a.y_dtype, o + 64);
                                   }
                               };
                               uint32_t rw[8];  // the rows' words of columns ln and ln + 64
                               if (e->residual && !fetched) fetch(m);
                               fetched = true;
                               float b0 = 0.f, b1 = 0.f;
                               if (e->bias) {
                                   b0 = load_any(e->bias, e->bias_dtype, col);
                                   b1 = load_any(e->bias, e->bias_dtype, col + 64);
                               }
#pragma unroll
                               for (int i = 0; i < 4; i++) {
                                   rw[2 * i] = next0[i];
                                   rw[2 * i + 1] = next1[i];
                               }
                               // a wave's rows are m, m + 4 of each 16
                               if (e->residual) fetch(m + ((m & 4) ? 12 : 4));
                               fwht128_wave_rows<4>(v0, v1, ln);
                               float z[8], y[8];
#pragma unroll
                               for (int i = 0; i < 4; i++) {
                                   z[2 * i] = v0[i] * codebook_scale<FAM>() * HAD_SCALE * s0 + b0;
                                   z[2 * i + 1] = v1[i] * codebook_scale<FAM>() * HAD_SCALE * s1 + b1;
                               }
                               act_eight(e->act, z, y);
                               if (e->residual) {
#pragma unroll
                                   for (int i = 0; i < 8; i++) y[i] += act_from_word(rw[i], a.y_dtype, col);
                               }
                               const size_t yo = ((size_t)mt * G2_MT + m) * a.out + col;
                               store_rows4(a.y, a.y_dtype, yo, a.out, live, y);
                               if (e->pre) store_rows4(e->pre, a.y_dtype, yo, a.out, live, z);
                               return;
                           }
                           fwht128_wave_rows<4>(v0, v1, ln);
                           for (int i = 0; i < live; i++) {
                               const size_t yo = ((size_t)g * a.rows + mt * G2_MT + m + i) * a.out + (size_t)og * 128;
                               store_y4(a.y, a.y_dtype, yo + ln, v0[i] * codebook_scale<FAM>() * HAD_SCALE * s0,
                                        v1[i] * codebook_scale<FAM>() * HAD_SCALE * s1);
                           }
                       });
}
template <int FAM, int N>
__global__ __launch_bounds__(G4_THREADS) void gemm4_kernel(GemmArgs a) {
    gemm4_run<FAM, N, false>(a, nullptr);
}
template <int FAM, int N>
__global__ __launch_bounds__(G4_THREADS) void gemm4_epilogue_kernel(GemmArgs a, EpilogueArgs e) {
    gemm4_run<FAM, N, true>(a, &e);
}

// A tile of sp.tile_rows rows x 128 columns over one split's k: the raw products to its plane.
template <int FAM, int N>
__global__ __launch_bounds__(G4_THREADS) void gemm4_split_kernel(GemmArgs a, GemmSplit sp) {
    const int OT = a.out >> 4, nog = a.out / 128, nm = (a.rows + sp.tile_rows - 1) / sp.tile_rows, nk = a.in / 128;
    const int s = (int)blockIdx.x / (nog * nm), L = (int)blockIdx.x - s * nog * nm;
    const int og = L % nog, mt = L / nog;
    const int k0 = (int)((long)nk * s / sp.splits), nsup = (int)((long)nk * (s + 1) / sp.splits) - k0;  // >= 1 each
    __shared__ __align__(16) uint16_t Bs[2][128 * G4_BP];
    const int rows = min(sp.tile_rows, a.rows - mt * sp.tile_rows);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int d = gemm4_decoder(wave, rows);
    if (d >= 0) {
        gemm4_decode_role<FAM>(rows <= G4_HELP_ROWS, d, nsup, lane, Bs, [&](int r, int rs, int loads) {
            return RateReader<FAM, N>(a.trellis + (size_t)k0 * 8 * OT * N, r, rs, OT, og, loads, lane, a.k);
        });
        return;
    }
    const uint16_t *xfrag0 =
        a.xp + (size_t)mt * (sp.tile_rows / 16) * (size_t)(a.in / 32) * 512 + (size_t)k0 * 4 * 512;
    float *plane = sp.part + ((size_t)s * a.rows + (size_t)mt * sp.tile_rows) * a.out + (size_t)og * 128;
    gemm4_mfma_waves<false>(
        a.in, 2 * nsup, xfrag0, rows, nullptr, Bs,
        [&](int m, int live, float (&v0)[4], float (&v1)[4], int ln, uint32_t) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < live) {
                    float *p = plane + (size_t)(m + i) * a.out + ln;
                    p[0] = v0[i];
                    p[64] = v1[i];
                }
        });
}

// Columns i and i + 1 (i even) of a row in dtype dt, 4-byte aligned.
__device__ __forceinline__ void load_pair(const void *p, int dt, size_t i, float &x, float &y) {
    if (dt == DT_F32) {
        x = static_cast<const float *>(p)[i];
        y = static_cast<const float *>(p)[i + 1];
        return;
    }
    const uint32_t w = act_word(p, dt, i);
    x = act_from_word(w, dt, 0);
    y = act_from_word(w, dt, 1);
}
__device__ __forceinline__ void store_pair(void *p, int dt, size_t i, float x, float y) {
    if (dt == DT_F32) {
        static_cast<float *>(p)[i] = x;
        static_cast<float *>(p)[i + 1] = y;
        return;
    }
    *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p) + i) = pack2(dt == DT_BF16, x, y);
}

// The outputs from the splits' planes, summed in split order: a wave takes R rows of an output block.  A lane holds columns
// 2 l and 2 l + 1 (the transform of any order of the index's bits is the same up to that order), so every access but the
// f32 rows' is one word or two of a lane.
template <int FAM, int R>
__global__ __launch_bounds__(256) void gemm_split_finish_kernel(GemmArgs a, GemmSplit sp, EpilogueArgs e) {
    const int og = blockIdx.x, row0 = (blockIdx.y * 4 + (int)(threadIdx.x >> 6)) * R, lane = threadIdx.x & 63;
    if (row0 >= a.rows) return;
    const int live = min(R, a.rows - row0);
    const size_t col = (size_t)og * 128 + 2 * lane;
    float r0[R] = {}, r1[R] = {}, b0 = 0.f, b1 = 0.f;
    if (e.residual) {
#pragma unroll
        for (int r = 0; r < R; r++)
            load_pair(e.residual, a.y_dtype, (size_t)(row0 + min(r, live - 1)) * a.out + col, r0[r], r1[r]);
    }
    if (e.bias) {
        b0 = load_any(e.bias, e.bias_dtype, col);
        b1 = load_any(e.bias, e.bias_dtype, col + 1);
    }
    constexpr float SC = codebook_scale<FAM>() * HAD_SCALE;
    const float s0 = h2f(a.svh[col]) * SC, s1 = h2f(a.svh[col + 1]) * SC;
    constexpr int CH = R == 1 ? 8 : 4;  // splits' loads in flight
    const size_t stride = (size_t)a.rows * a.out;
    float v0[R] = {}, v1[R] = {};
    for (int q0 = 0; q0 < sp.splits; q0 += CH) {
        float2 t[CH][R];
#pragma unroll
        for (int q = 0; q < CH; q++)
#pragma unroll
            for (int r = 0; r < R; r++)
                t[q][r] = *reinterpret_cast<const float2 *>(sp.part + (size_t)min(q0 + q, sp.splits - 1) * stride +
                                                            (size_t)(row0 + min(r, live - 1)) * a.out + col);
#pragma unroll
        for (int q = 0; q < CH; q++)
#pragma unroll
            for (int r = 0; r < R; r++) {
                v0[r] += q0 + q < sp.splits ? t[q][r].x : 0.f;
                v1[r] += q0 + q < sp.splits ? t[q][r].y : 0.f;
            }
    }
    float z[8] = {}, y[8];
    if constexpr (R == 1) fwht128_wave(v0[0], v1[0], lane);
    else fwht128_wave_rows<R>(v0, v1, lane);
#pragma unroll
    for (int r = 0; r < R; r++) {
        z[2 * r] = v0[r] * s0 + b0;
        z[2 * r + 1] = v1[r] * s1 + b1;
    }
    act_eight(e.act, z, y);
#pragma unroll
    for (int r = 0; r < R; r++)
        if (r < live) {
            const size_t i = (size_t)(row0 + r) * a.out + col;
            store_pair(a.y, a.y_dtype, i, y[2 * r] + r0[r], y[2 * r + 1] + r1[r]);
            if (e.pre) store_pair(e.pre, a.y_dtype, i, z[2 * r], z[2 * r + 1]);
        }
}

// ---- the ping-pong GEMM (hash-product families at the lane-reader rates)
//
// A workgroup of 8 waves owns an MT-row x 128-column output tile (MT = 256 or 512; one Hadamard block wide, so the
// FWHT + svh finish runs in its epilogue) over all of k, in k-steps of 64 (four trellis k-tiles).  Every wave owns
// RW = MT / 8 rows x all 128 columns (RW / 16 x 8 v_mfma_f32_16x16x32_f16 tiles) with its A fragments in registers, so
// each prepared row is loaded once per workgroup, and every wave also decodes: waves r and r + 4 decode the two column
// halves of k-tile row r of step s + 2 (the GEMV's lane decoder, half a chunk each) into a triple-buffered LDS slab.
// Waves r and r + 4 share a SIMD: wave r runs its step's MFMAs first and then decodes, wave r + 4 decodes first, so
// on every SIMD one wave feeds the matrix core while the other decodes on the VALU (a decode wave beside MFMA waves
// leaves their rate untouched).  One barrier per step: the slab read in step s was written in step s - 2 and the one
// written in step s was last read in step s - 1, each on the other side of a barrier.  The trellis words are loaded
// a step before their decode, the A fragments of step s + 1 as soon as step s's MFMAs of that half have issued.
// Every weight is decoded once per MT rows (twice per 1024 rows at MT = 512, against four times for the 256-row tile).
//
// KS = 2 splits k in halves over twice the workgroups (a grid of few 512-row tiles then fills the chip and still
// decodes every weight once per 512 rows).  Each half finishes half of every wave's rows: it writes the raw
// accumulators of the other half's rows through to memory, arrives at the tile's counter, adds the other half's
// partial of its own rows (a sum of two, so independent of which came first) and runs their epilogue.  The first to
// arrive waits, bounded, for the second; past the wait it hands the whole tile over.
constexpr int G5_WAVES = 8;
constexpr int G5_THREADS = 64 * G5_WAVES;
constexpr int G5_SLAB = 128 * G2_BP;                                        // halves per slab
constexpr int G5_SP = 144;  // epilogue stage pitch (halves): the four 16-lane groups' rows land 8 banks apart
constexpr int G5_EP = 132;  // its pitch (floats) for the sums of a launch with an epilogue: a read's eight rows spread
constexpr int lds_max(int a, int b) { return a > b ? a : b; }
constexpr int G5_LDS = lds_max(3 * G5_SLAB * 2, G5_WAVES * 16 * G5_SP * 2);
constexpr int G5_LDS_EPI = lds_max(G5_LDS, G5_WAVES * 16 * G5_EP * 4);

template <int FAM, int N, int MT, int KS, bool EPI>
__device__ __forceinline__ void gemm5_run(const GemmArgs &a, const EpilogueArgs *e) {
    static_assert(FAM != FAM_PAIR && FAM != FAM_MUL1, "hash-product families");
    static_assert(KS == 1 || KS == 2, "whole k or halves");
    constexpr int RW = MT / G5_WAVES;  // rows per wave
    constexpr int RB = RW / 16;        // row blocks per wave
    constexpr int AW = LaneBits<N>::AW;
    const int IT = a.in >> 4, OT = a.out >> 4;
    const int nog = a.out / 128, nm = (a.rows + MT - 1) / MT;
    // split ks of a tile: the grid's second half (its tile index repeats the first half's, so the same XCD map)
    const int ks = KS == 1 ? 0 : (int)blockIdx.x / (nm * nog);
    const int L = KS == 1 ? (int)blockIdx.x : (int)blockIdx.x - ks * nm * nog;
    int og, mt;
    if (nm <= 8 && 8 % nm == 0 && nog % (8 / nm) == 0) {  // a row tile's workgroups share an XCD (its A rows in one L2)
        const int xcd = L & 7, per = 8 / nm;
        mt = xcd / per;
        og = (L >> 3) * per + xcd % per;
    } else {
        og = L % nog;
        mt = L / nog;
    }
    const int g = blockIdx.z;
    __shared__ __align__(16) uint8_t lds[EPI ? G5_LDS_EPI : G5_LDS];
    uint16_t *slabs = reinterpret_cast<uint16_t *>(lds);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int RT = (a.rows + 15) / 16;
    const int nks = IT / 4 / KS;   // this split's k-steps (IT is a multiple of 8: whole 128-blocks)
    const int s0g = ks * nks;      // its first k-step
    const DecodeK k = a.k;
    const bool masked = k.wmask != 0xFFFFu;

    // ---- decode role: column half H of k-tile row r of each step
    const int r = wave & 3, H = wave >> 2;
    const int o = lane >> 3, j = lane & 7;
    const size_t kstep = (size_t)4 * OT * N;  // halves from one k-step's row r to the next
    const uint16_t *tb = a.trellis + (size_t)g * IT * OT * N + ((size_t)r * OT + og * 8) * N + (size_t)s0g * kstep;
    const uint32_t lane_words = (uint32_t)(o * N) >> 1;
    auto load_words = [&](int s, uint32_t (&W)[AW]) __attribute__((always_inline)) {
        load_lane_words_u<N>(reinterpret_cast<const uint32_t *>(tb + (size_t)min(s, nks - 1) * kstep), lane_words, j,
                             W);
    };
    // the slab column this lane writes (rows r * 16 .. + 15 of the step's 64 k)
    const int col = o * 16 + j + 8 * H;
    auto decode_into = [&](int s, const uint32_t (&W)[AW]) __attribute__((always_inline)) {
        uint32_t w[8];
        if (H) {
            if (masked) decode_weights_half<FAM, N, true, 1>(W, k, w);
            else decode_weights_half<FAM, N, false, 1>(W, k, w);
        } else {
            if (masked) decode_weights_half<FAM, N, true, 0>(W, k, w);
            else decode_weights_half<FAM, N, false, 0>(W, k, w);
        }
        uint16_t *dst = slabs + (size_t)(s % 3) * G5_SLAB + col * G2_BP + r * 16;
        *reinterpret_cast<uint4 *>(dst) = uint4{w[0], w[2], w[4], w[6]};
        *reinterpret_cast<uint4 *>(dst + 8) = uint4{w[1], w[3], w[5], w[7]};
    };

    // ---- MFMA role: rows m0 .. m0 + RW - 1 of the tile, all 128 columns
    const int m0 = mt * MT + wave * RW;
    // fragment (row tile rt, 32-k block kk) of group g: bytes ((rt in/32 + kk) 1024 + 16 lane) of the group's
    // prepared rows, read through a buffer resource (uniform base and offset in scalar registers, one lane offset)
    typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
    const size_t xp_group = (size_t)RT * (size_t)(a.in / 32) * 512;  // halves per group
    const __amdgpu_buffer_rsrc_t xrs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t *>(a.xp + (size_t)g * xp_group), (short)0, (int)(xp_group * 2), 0x00020000);
    const uint32_t a_lane = (uint32_t)lane * 16u;
    f4_t acc[RB][8];
#pragma unroll
    for (int rb = 0; rb < RB; rb++)
#pragma unroll
        for (int cb = 0; cb < 8; cb++) acc[rb][cb] = f4_t{0.f, 0.f, 0.f, 0.f};
    uint4 A[2][RB];
    auto load_a = [&](int s, int kb) __attribute__((always_inline)) {
        const int kk = (s0g + min(s, nks - 1)) * 2 + kb;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            const int rt = min(m0 / 16 + rb, RT - 1);
            const int soff = (rt * (a.in / 32) + kk) * 1024;
            const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(xrs, a_lane, soff, 0);
            A[kb][rb] = uint4{v.x, v.y, v.z, v.w};
        }
    };
    // B fragment f = kb * 8 + cb of step s; the first PD of a step are read before it starts (at the end of the
    // wave's previous decode phase), the rest PD fragments ahead of their MFMAs
    constexpr int PD = 3;
    auto frag = [&](int s, int f) __attribute__((always_inline)) {
        const uint16_t *bp = slabs + (size_t)(s % 3) * G5_SLAB + c * G2_BP + 8 * h;
        return *reinterpret_cast<const uint4 *>(bp + (f & 7) * 16 * G2_BP + (f >> 3) * 32);
    };
    uint4 bpre[PD];
    auto read_first = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < PD; f++) bpre[f] = frag(s, f);
    };
    auto mfma_phase = [&](int s) __attribute__((always_inline)) {
        uint4 bq[16];
#pragma unroll
        for (int f = 0; f < PD; f++) bq[f] = bpre[f];
#pragma unroll
        for (int f = 0; f < 16; f++) {
            if (f + PD < 16) bq[f + PD] = frag(s, f + PD);
            const int kb = f >> 3, cb = f & 7;
            const h8_t B8 = __builtin_bit_cast(h8_t, bq[f]);
#pragma unroll
            for (int rb = 0; rb < RB; rb++)
                acc[rb][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, A[kb][rb]), B8,
                                                                     acc[rb][cb], 0, 0, 0);
            if (f == 7) load_a(s + 1, 0);
            if (f == 15) load_a(s + 1, 1);
            if (f & 1) __builtin_amdgcn_sched_barrier(0);  // keep the B reads a few fragments ahead, not all at once
        }
    };

    // ---- the step loop.  Every wave runs the same order -- step s's MFMAs, then a decode -- and waves differ only in
    // where their barrier falls: waves 0-3 (H = 0) decode step s + 2 before barrier s, waves 4-7 (H = 1) decode step
    // s + 3 after it.  So between two barriers a SIMD's H = 0 wave runs its MFMAs and then decodes while its H = 1
    // wave decodes and then runs its MFMAs.  Slab t % 3 is read in step t after barrier t - 1; its H = 0 half is
    // written before barrier t - 2, its H = 1 half after barrier t - 3; both after the reads of step t - 3, which end
    // before barrier t - 3.  The words of step s + 2 + H sit in ring slot s % 3, loaded in the step before.
    uint32_t W0[AW], W1[AW], W2[AW];
    load_a(0, 0);
    load_a(0, 1);
    {
        uint32_t P0[AW], P1[AW];
        load_words(0, P0);
        load_words(1, P1);
        load_words(2, W2);
        load_words(2 + H, W0);
        decode_into(0, P0);
        decode_into(1, P1);
        if (H) decode_into(2, W2);
    }
    __syncthreads();
    read_first(0);
    auto step = [&](int s, const uint32_t (&Wd)[AW], uint32_t (&Wl)[AW]) __attribute__((always_inline)) {
        mfma_phase(s);
        __builtin_amdgcn_sched_barrier(0);
        if (H) __syncthreads();
        if (s + 2 + H < nks) decode_into(s + 2 + H, Wd);
        if (s + 3 + H < nks) load_words(s + 3 + H, Wl);
        if (s + 1 < nks) read_first(s + 1);  // slab s + 1 was complete before barrier s - 1
        __builtin_amdgcn_sched_barrier(0);
        if (!H) __syncthreads();
    };
    for (int s = 0; s < nks; s += 3) {
        step(s, W0, W1);
        if (s + 1 < nks) step(s + 1, W1, W2);
        if (s + 2 < nks) step(s + 2, W2, W0);
    }
    __syncthreads();  // the H = 1 waves' last decode (none: s + 3 >= nks) and every slab read are behind this

    // Row blocks this workgroup finishes: all of them, or with k in halves the half's own (set below).
    bool fin_lo = true, fin_hi = true;  // row blocks 0 .. RB/2 - 1 and RB/2 .. RB - 1 of every wave
    if constexpr (KS == 2) {
        // partial of split ks: [tile][ks][wave][rb][cb] blocks of 64 lanes x 4 floats, one 1 KiB store each.  Half ks
        // finishes row blocks RB/2 ks .. RB/2 ks + RB/2 - 1 of every wave: it writes the partner's row blocks of its
        // partial, arrives, and adds the partner's partial of its own.  The first to arrive waits (at most a.kwait
        // ticks) for the second; past the wait it writes its own row blocks too and hands the whole tile over, and
        // the second finishes every row.  Each output is the same sum of two either way.
        static_assert(RB % 2 == 0, "halves of the row blocks");
        constexpr int RH = RB / 2;
        const size_t tile = ((size_t)g * nm + mt) * nog + og;
        const size_t wave_f = (size_t)RB * 8 * 256;  // floats per wave
        float *mine = a.kpart + ((tile * 2 + ks) * G5_WAVES + wave) * wave_f;
        const float *other = a.kpart + ((tile * 2 + (ks ^ 1)) * G5_WAVES + wave) * wave_f;
        const __amdgpu_buffer_rsrc_t mr = __builtin_amdgcn_make_buffer_rsrc(mine, (short)0, (int)(wave_f * 4), 0x00020000);
        const __amdgpu_buffer_rsrc_t orr =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(other), (short)0, (int)(wave_f * 4), 0x00020000);
        // sc0 sc1: the stores go through to memory and the loads bypass the caches (the halves may sit on two XCDs)
        constexpr int SYS = 1 | 16;
        auto store_rows = [&](int half) __attribute__((always_inline)) {
#pragma unroll
            for (int rb = 0; rb < RB; rb++)
                if (rb / RH == half) {
#pragma unroll
                    for (int cb = 0; cb < 8; cb++)
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc[rb][cb]), mr, a_lane,
                                                               (rb * 8 + cb) * 1024, SYS);
                }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // acknowledged before the counter moves
        };
        constexpr uint32_t HANDED = 0x40000000u;  // the first half gave its whole tile to the second
        store_rows(ks ^ 1);
        __syncthreads();
        __shared__ uint32_t arrived;
        uint32_t *ctr = a.kctr + tile * COUNTER_STRIDE;
        if (tid == 0) arrived = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        const uint32_t st = arrived;
        __syncthreads();  // every wave has read `arrived` before wave 0 reuses it
        bool all = false;
        if (st == 0) {
            // first: wave 0 polls for the second's arrival, at most kwait ticks, so the wait always ends
            if (tid == 0) {
                const uint64_t t0 = __builtin_amdgcn_s_memrealtime();
                uint32_t v = __hip_atomic_load(ctr, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                while (v < 2u && __builtin_amdgcn_s_memrealtime() - t0 < (uint64_t)a.kwait) {
                    __builtin_amdgcn_s_sleep(2);
                    v = __hip_atomic_load(ctr, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                arrived = v;
            }
            __syncthreads();
            if (arrived < 2u) {
                // the second has not arrived: write this half's own row blocks, then hand the tile over unless the
                // second arrived meanwhile (then it has written this half's rows and finishes its own as usual)
                store_rows(ks);
                __syncthreads();
                if (tid == 0) {
                    uint32_t expect = 1u;
                    __hip_atomic_compare_exchange_strong(ctr, &expect, HANDED, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                         __HIP_MEMORY_SCOPE_AGENT);
                    arrived = expect;  // 1: handed over; 2: the second arrived first
                }
                __syncthreads();
                if (arrived == 1u) return;
            }
            if (tid == 0) *ctr = 0u;  // both arrived and the second never reads it again; the next launch reads it
                                      // after the kernel boundary
        } else if (st >= HANDED) {
            all = true;  // the first handed over the whole tile
            if (tid == 0) *ctr = 0u;
        }
        fin_lo = all || ks == 0;
        fin_hi = all || ks == 1;
#pragma unroll
        for (int rb = 0; rb < RB; rb++)
            if (rb < RH ? fin_lo : fin_hi) {
#pragma unroll
                for (int cb = 0; cb < 8; cb++) {
                    const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(orr, a_lane, (rb * 8 + cb) * 1024, SYS);
                    acc[rb][cb] += __builtin_bit_cast(f4_t, v);
                }
            }
    }

    // ---- epilogue: the output transform straight from the accumulators.  Column cb * 16 + c of the tile sits in
    // acc[.][cb] of lane c + 16 h (rows 4 h .. 4 h + 3), and H128 = H8 (over cb) x H16 (over c): the stages of bits
    // 6, 5, 4 are butterflies between a lane's own registers, those of bits 3 .. 0 the DPP stages within each 16-lane
    // row.  These are fwht128_wave's stages in its order with its sums, so the outputs equal the row-wise transform's
    // bit for bit, without staging rows through LDS or running one transform per row.
    const size_t sv = (size_t)g * a.out + (size_t)og * 128;
    float svc[8];
#pragma unroll
    for (int cb = 0; cb < 8; cb++) svc[cb] = h2f(a.svh[sv + cb * 16 + c]);
    const float sg8 = lane_sign<8>(lane), sg4 = lane_sign<4>(lane), sg2 = lane_sign<2>(lane), sg1 = lane_sign<1>(lane);
    // 16-bit outputs go out through a per-wave LDS stage of 16 rows (the slab ring is free past the last barrier):
    // one 16-byte store covers four rows' eighths, against a 2-byte store per lane from the lane layout
    // (and so does any y not 16-byte aligned: then every output goes out straight from the lane layout)
    const bool wide = a.y_dtype == DT_F32 || (reinterpret_cast<uintptr_t>(a.y) & 15) != 0, bf16 = a.y_dtype == DT_BF16;
    uint16_t *stage = reinterpret_cast<uint16_t *>(lds) + wave * 16 * G5_SP;
    // With an epilogue the f32 sums are staged instead, and each lane finishes eight columns of a row: where y is 16 bits
    // and every row 16-byte aligned, from 16-byte loads of the residual (issued ahead of the row block's transforms) to
    // 16-byte stores of y and pre.
    bool epi_wide = wide;
    if constexpr (EPI)
        epi_wide = epi_wide || ((reinterpret_cast<uintptr_t>(e->residual) | reinterpret_cast<uintptr_t>(e->pre)) & 15) != 0;
    float *estage = reinterpret_cast<float *>(lds) + wave * 16 * G5_EP;
    const size_t ecol = (size_t)og * 128 + (size_t)(lane & 15) * 8;
    float ebias[8];
    if constexpr (EPI) {
#pragma unroll
        for (int q = 0; q < 8; q++)
            ebias[q] = e->bias ? load_any(e->bias, e->bias_dtype, ecol + q) : 0.f;
    }
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        if (!(rb < RB / 2 ? fin_lo : fin_hi)) continue;
        uint4 res[4] = {};
        if constexpr (EPI) {
            if (!epi_wide && e->residual) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int m = min(m0 + rb * 16 + 4 * q + (lane >> 4), a.rows - 1);
                    res[q] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(e->residual) +
                                                              (size_t)m * a.out + ecol);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v[8];
#pragma unroll
            for (int cb = 0; cb < 8; cb++) v[cb] = acc[rb][cb][i];
#pragma unroll
            for (int hb = 4; hb >= 1; hb >>= 1)
#pragma unroll
                for (int cb = 0; cb < 8; cb++)
                    if (!(cb & hb)) {
                        const float lo = v[cb], hi = v[cb | hb];
                        v[cb] = lo + hi;
                        v[cb | hb] = lo - hi;
                    }
#pragma unroll
            for (int cb = 0; cb < 8; cb += 2) fwht_stage<8>(v[cb], v[cb + 1], sg8);
#pragma unroll
            for (int cb = 0; cb < 8; cb += 2) fwht_stage<4>(v[cb], v[cb + 1], sg4);
#pragma unroll
            for (int cb = 0; cb < 8; cb += 2) fwht_stage<2>(v[cb], v[cb + 1], sg2);
#pragma unroll
            for (int cb = 0; cb < 8; cb += 2) fwht_stage<1>(v[cb], v[cb + 1], sg1);
            if constexpr (EPI) {
#pragma unroll
                for (int cb = 0; cb < 8; cb++)
                    estage[(4 * h + i) * G5_EP + cb * 16 + c] = v[cb] * codebook_scale<FAM>() * HAD_SCALE * svc[cb];
            } else if (wide) {
                const int m = m0 + rb * 16 + 4 * h + i;
                if (m < a.rows) {
                    const size_t yo = ((size_t)g * a.rows + m) * a.out + (size_t)og * 128 + c;
#pragma unroll
                    for (int cb = 0; cb < 8; cb++) {
                        const float y = v[cb] * codebook_scale<FAM>() * HAD_SCALE * svc[cb];
                        if (a.y_dtype == DT_F16) store_act<DT_F16>(a.y, yo + cb * 16, y);
                        else if (bf16) store_act<DT_BF16>(a.y, yo + cb * 16, y);
                        else store_act<DT_F32>(a.y, yo + cb * 16, y);
                    }
                }
            } else {
#pragma unroll
                for (int cb = 0; cb < 8; cb++) {
                    // y is rounded to f32 first, as every other output path rounds it (the empty asm keeps the
                    // product from fusing into the 16-bit conversion, which would round once and differ at ties)
                    float y = v[cb] * codebook_scale<FAM>() * HAD_SCALE * svc[cb];
                    asm("" : "+v"(y));
                    stage[(4 * h + i) * G5_SP + cb * 16 + c] =
                        bf16 ? __bfloat16_as_ushort(__float2bfloat16(y)) : __half_as_ushort(__float2half_rn(y));
                }
            }
        }
        if constexpr (EPI) {
#pragma unroll 1
            for (int q = 0; q < 4; q++) {  // one body (the activations are long), the residual shifted through slot 0
                const int rr = 4 * q + (lane >> 4), m = min(m0 + rb * 16 + rr, a.rows - 1);
                const bool live = m0 + rb * 16 + rr < a.rows;
                const size_t yo = (size_t)m * a.out + ecol;
                const float *er = estage + rr * G5_EP + (lane & 15) * 8;
                if (epi_wide) {
#pragma unroll 1
                    for (int j = 0; j < 8 && live; j++) {
                        const float y = epilogue_apply(*e, a.y_dtype, er[j],
                                                       e->bias ? act_word(e->bias, e->bias_dtype, ecol + j) : 0u,
                                                       ecol + j, e->residual ? act_word(e->residual, a.y_dtype, yo + j) : 0u, yo + j);
                        store_any(a.y, a.y_dtype, yo + j, y);
                    }
                    continue;
                }
                float z[8], y[8];
                const uint32_t rw[4] = {res[0].x, res[0].y, res[0].z, res[0].w};
                res[0] = res[1];
                res[1] = res[2];
                res[2] = res[3];
#pragma unroll
                for (int j = 0; j < 8; j++) z[j] = er[j] + ebias[j];
                act_eight(e->act, z, y);
                if (e->residual) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint32_t h = j & 1 ? rw[j >> 1] >> 16 : rw[j >> 1] & 0xFFFFu;
                        y[j] += bf16 ? __uint_as_float(h << 16) : h2f((uint16_t)h);
                    }
                }
                if (live) {
                    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.y) + yo) = pack8(bf16, y);
                    if (e->pre) *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(e->pre) + yo) = pack8(bf16, z);
                }
            }
        } else if (!wide) {  // the wave's 16 rows, row-major in its LDS region: four rows per 16-byte store
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int rr = 4 * q + (lane >> 4), m = m0 + rb * 16 + rr;
                const uint4 val = *reinterpret_cast<const uint4 *>(stage + rr * G5_SP + (lane & 15) * 8);
                if (m < a.rows)
                    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.y) + ((size_t)g * a.rows + m) * a.out +
                                               (size_t)og * 128 + (lane & 15) * 8) = val;
            }
        }
    }
}
template <int FAM, int N, int MT, int KS>
__global__ __launch_bounds__(G5_THREADS, 1) void gemm5_kernel(GemmArgs a) {
    gemm5_run<FAM, N, MT, KS, false>(a, nullptr);
}
template <int FAM, int N, int MT, int KS>
__global__ __launch_bounds__(G5_THREADS, 1) void gemm5_epilogue_kernel(GemmArgs a, EpilogueArgs e) {
    gemm5_run<FAM, N, MT, KS, true>(a, &e);
}

// The launchers, for plain linears (EPI = false, e null) and those with an epilogue: exl3_gemm.hip builds the former,
// exl3_gemm_epilogue.hip the latter.
struct GemmEpilogue {
    EpilogueArgs args;
    GemmSplit split;
};
template <int FAM, int N, int MT, int KS, bool EPI>
static void launch_gemm5(const GemmArgs &a, const GemmEpilogue *e, dim3 grid, hipStream_t s) {
    if constexpr (EPI) hipLaunchKernelGGL((gemm5_epilogue_kernel<FAM, N, MT, KS>), grid, dim3(G5_THREADS), 0, s, a, e->args);
    else hipLaunchKernelGGL((gemm5_kernel<FAM, N, MT, KS>), grid, dim3(G5_THREADS), 0, s, a);
}

template <int FAM, int N, bool EPI>
static hipError_t launch_gemm_lane_n(const GemmArgs &a, const GemmEpilogue *e, hipStream_t s) {
    if (a.x_dtype == DT_F16) launch_gemm_prepare_frag<DT_F16>(a, s);
    else if (a.x_dtype == DT_BF16) launch_gemm_prepare_frag<DT_BF16>(a, s);
    else launch_gemm_prepare_frag<DT_F32>(a, s);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    // The ping-pong body once its 512-row tiles still give most CUs a workgroup (measured at C3's 4096 x 14336: 768 to
    // 4096 rows 13-24% faster than the 256-row decode-wave tile; at 512 rows, 112 workgroups, 18% slower, and with k in
    // halves, 224 workgroups, 3% faster).
    int arm = a.arm ? a.arm : gemm_default_arm(a.groups, a.rows, a.out);
    if constexpr (FAM == FAM_PAIR || FAM == FAM_MUL1) arm = 4;  // the ping-pong body serves the hash-product families
    if constexpr (N > 64) arm = 4;  // K = 5 .. 8 are built for the decode-wave tile only
    // n = 40's unaligned lane reader does not fit the 512-row tile's registers (it would spill): the 256-row one
    if constexpr (N == 40) arm = arm == 5 ? (a.arm ? 6 : 4) : arm;
    if (arm == 7 && (N == 40 || !a.kpart)) arm = 4;  // the split needs its partial region (the host sizes it)
    if constexpr (N <= 64) {
        if (arm == 5 || arm == 6 || arm == 7) {
            const int mt = arm == 6 ? 256 : 512;
            dim3 grid((unsigned)((a.out / 128) * ((a.rows + mt - 1) / mt) * (arm == 7 ? 2 : 1)), 1, (unsigned)a.groups);
            if constexpr (FAM != FAM_PAIR && FAM != FAM_MUL1) {
                if constexpr (N != 40) {
                    if (arm == 5) launch_gemm5<FAM, N, 512, 1, EPI>(a, e, grid, s);
                    if (arm == 7) launch_gemm5<FAM, N, 512, 2, EPI>(a, e, grid, s);
                }
                if (arm == 6) launch_gemm5<FAM, N, 256, 1, EPI>(a, e, grid, s);
            }
            return hipGetLastError();
        }
    }
    if constexpr (EPI) {
        if (e->split.part) {
            const GemmSplit &sp = e->split;
            const int tiles = (a.out / 128) * ((a.rows + sp.tile_rows - 1) / sp.tile_rows);
            hipLaunchKernelGGL((gemm4_split_kernel<FAM, N>), dim3((unsigned)(tiles * sp.splits)), dim3(G4_THREADS), 0, s, a, sp);
            const hipError_t launched = hipGetLastError();
            if (launched != hipSuccess) return launched;
            // four rows a wave once that leaves four waves a SIMD (200 rows of 2560 x 16384, two splits, gelu: 12.2 -> 9.5 us;
            // 600 rows of 2048 x 2048, 9600 rows of a block, 1 us more)
            const bool four = (long)a.rows * (a.out / 128) >= 16384;
            const dim3 fg((unsigned)(a.out / 128), (unsigned)((a.rows + (four ? 15 : 3)) / (four ? 16 : 4)));
            if (four) hipLaunchKernelGGL((gemm_split_finish_kernel<FAM, 4>), fg, dim3(256), 0, s, a, sp, e->args);
            else hipLaunchKernelGGL((gemm_split_finish_kernel<FAM, 1>), fg, dim3(256), 0, s, a, sp, e->args);
            return hipGetLastError();
        }
    }
    dim3 grid((unsigned)((a.out / 128) * ((a.rows + G2_MT - 1) / G2_MT)), 1, (unsigned)a.groups);
    if constexpr (EPI) hipLaunchKernelGGL((gemm4_epilogue_kernel<FAM, N>), grid, dim3(G4_THREADS), 0, s, a, e->args);
    else hipLaunchKernelGGL((gemm4_kernel<FAM, N>), grid, dim3(G4_THREADS), 0, s, a);
    return hipGetLastError();
}

template <int FAM, int N, bool EPI>
static hipError_t launch_gemm_n(const GemmArgs &a, const uint16_t *wt, const GemmEpilogue *e, hipStream_t s) {
    dim3 grid((unsigned)(a.out / 128), (unsigned)((a.rows + GM_MT - 1) / GM_MT), (unsigned)a.groups);
    if constexpr (EPI) hipLaunchKernelGGL((gemm_epilogue_kernel<FAM, N>), grid, dim3(GM_THREADS), 0, s, a, wt, e->args);
    else hipLaunchKernelGGL((gemm_kernel<FAM, N>), grid, dim3(GM_THREADS), 0, s, a, wt);
    return hipGetLastError();
}

template <int FAM, bool EPI>
static hipError_t launch_gemm_fam(const GemmArgs &a, const GemmEpilogue *e, hipStream_t s) {
    switch (a.n) {
    case 16: return launch_gemm_lane_n<FAM, 16, EPI>(a, e, s);
    case 24: return launch_gemm_lane_n<FAM, 24, EPI>(a, e, s);
    case 32: return launch_gemm_lane_n<FAM, 32, EPI>(a, e, s);
    case 40: return launch_gemm_lane_n<FAM, 40, EPI>(a, e, s);
    case 48: return launch_gemm_lane_n<FAM, 48, EPI>(a, e, s);
    case 64: return launch_gemm_lane_n<FAM, 64, EPI>(a, e, s);
    default: break;
    }
    // K = 5 .. 8 (PAIR1 has no rows there): the lane reader inside the tile, instead of a pass that writes the f16
    // weights and a body that reads them back.  MCG n = 96, 17 / 200 / 777 / 2048 rows: 2560 x 16384 139 / 169 / 243 /
    // 481 -> 37 / 53 / 119 / 234 us, 14336 x 4096 429 / 533 / 552 / 637 -> 118 / 189 / 211 / 287 us; MUL1 at 14336 x 4096
    // 440 / 545 / 561 / 646 -> 192 / 274 / 294 / 366 us.
    if constexpr (FAM != FAM_PAIR) {
        switch (a.n) {
        case 80: return launch_gemm_lane_n<FAM, 80, EPI>(a, e, s);
        case 96: return launch_gemm_lane_n<FAM, 96, EPI>(a, e, s);
        case 112: return launch_gemm_lane_n<FAM, 112, EPI>(a, e, s);
        case 128: return launch_gemm_lane_n<FAM, 128, EPI>(a, e, s);
        default: break;
        }
    }
    hipLaunchKernelGGL(gemm_prepare_kernel, dim3((unsigned)(a.in / 128), (unsigned)a.rows, (unsigned)a.groups),
                       dim3(64), 0, s, a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    // Any other rate: decode to a transposed f16 copy in workspace (held after xp), then the same MFMA body.
    uint16_t *wt = a.wt;
    hipLaunchKernelGGL(gemm_decode_transposed_kernel<FAM>,
                       dim3((unsigned)((a.in / 16) * (a.out / 16)), (unsigned)a.groups), dim3(128), 0, s, a, wt);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
    return launch_gemm_n<FAM, 0, EPI>(a, wt, e, s);
}

template <bool EPI>
static hipError_t launch_gemm(int fam, const GemmArgs &a, const GemmEpilogue *e, hipStream_t s) {
    switch (fam) {
    case FAM_MCG: return launch_gemm_fam<FAM_MCG, EPI>(a, e, s);
    case FAM_MUL1: return launch_gemm_fam<FAM_MUL1, EPI>(a, e, s);
    case FAM_HASH: return launch_gemm_fam<FAM_HASH, EPI>(a, e, s);
    case FAM_PAIR: return launch_gemm_fam<FAM_PAIR, EPI>(a, e, s);
    default: return launch_gemm_fam<FAM_3INST, EPI>(a, e, s);
    }
}

}  // namespace exl3
