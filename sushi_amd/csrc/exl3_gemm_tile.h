// The decode-wave GEMM tile: decode waves fill an LDS slab with a bank's weights while MFMA waves multiply it.  Shared by
// the dense and routed prefill GEMMs (exl3_gemm_body.h, exl3_moe_gemm.hip) and the product with the transposed
// bank (exl3_gradient.hip).
#pragma once
#include "exl3_kernels.h"
#include "exl3_lane_decode.h"
#include "exl3_tables.h"

namespace exl3 {

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// ---- the decode-once GEMM (integer and half-integer rates with a lane reader: n = 16, 24, 32, 40, 48, 64, 80, 96, 112, 128)
//
// A workgroup owns a 256-row x 128-column output tile (one Hadamard block wide, so the FWHT + svh finish runs in its
// epilogue) over all of k, in super-steps of 128 k (eight trellis k-tile rows), with the decode and the MFMAs on
// different waves.  The decoders (lane 8o + j: codewords 32j..32j+31 of tile o = columns j and j+8 over 16 k rows,
// the GEMV's lane decoder) fill a double-buffered LDS slab held column-major (B[col][k]), their tile words loaded a
// super-step ahead: waves 8-11, wave 8 + d decoding k-tile rows d and d + 4 of every super-step; when the live rows
// fit in 128 (MFMA waves 4-7 would have no rows), waves 4-7 decode too and each of the eight decoders takes one row
// (wave 8 + d row d, wave 4 + d row 4 + d), so a short window -- the common MoE window -- decodes on two waves per
// SIMD.  Waves 0-7 run the MFMAs: wave w owns rows 64 (w >> 1) .. + 63 and columns 64 (w & 1) .. + 63 as 4 x 4
// v_mfma_f32_16x16x32_f16 tiles per 32 k, with A fragments read from the prepared input in fragment order (one
// contiguous 1 KiB per load, a 64-k step ahead) and each 64-k step's B fragments read from the slab before its first
// MFMA.  One workgroup barrier per super-step hands the slab over: after barrier S + 1 the MFMA waves have finished
// reading slab S & 1 and the decoders have finished writing slab (S + 1) & 1.  Every weight is decoded once per
// 256-row tile.  Row groups wholly past the live rows leave before the first barrier.
constexpr int G2_MT = 256;   // rows per workgroup
constexpr int G2_BP = 72;    // LDS pitch (halves) of one ping-pong slab column: 64 k + 8 pad (16-byte aligned rows)
constexpr int G4_BP = 136;   // LDS pitch (halves) of one decode-wave-tile slab column: 128 k + 8 pad
constexpr int G4_HELP_ROWS = 128;  // live rows up to which MFMA waves 4-7 decode
constexpr int G2_EP = 129;   // epilogue staging pitch (floats)
constexpr int G4_STAGE_ALL = G2_MT * G2_EP * 4;  // bytes of a staged 256-row tile
constexpr int G4_WAVES = 12;
constexpr int G4_THREADS = 64 * G4_WAVES;

// Outputs at columns i and i + 64 of one row, in y's dtype.
__device__ __forceinline__ void store_y4(void *y, int dt, size_t i, float y0, float y1) {
    if (dt == DT_F16) {
        store_act<DT_F16>(y, i, y0);
        store_act<DT_F16>(y, i + 64, y1);
    } else if (dt == DT_BF16) {
        store_act<DT_BF16>(y, i, y0);
        store_act<DT_BF16>(y, i + 64, y1);
    } else {
        store_act<DT_F32>(y, i, y0);
        store_act<DT_F32>(y, i + 64, y1);
    }
}

// The MFMA waves' main loop of the decode-wave tile over the first NRB of the wave's four 16-row blocks (the rest of
// acc stays zero): instantiated per live-block count, so a short row group (a window of 65-85 rows leaves its second
// one or two) neither loads A nor issues MFMAs for its empty blocks, without a branch in the loop.  nks 64-k steps,
// two per super-step: 1 + nks / 2 barriers, as the decoders meet.
// TR: the slab is contracted over its columns (the product with the transposed bank): its columns are the k of the step,
// and each B fragment comes by transposing reads -- within 16 lanes, lane c hands in the address of four neighbouring
// k-tile rows of column k0 + c / 4 and receives row c of columns k0 .. k0 + 3.
typedef short s4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 read_transposed(const uint16_t *p) {
    typedef __attribute__((address_space(3))) s4_t lds_s4;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)const_cast<uint16_t *>(p)));
}
template <int NRB, bool TR = false>
__device__ __forceinline__ void gemm4_mfma_loop(const uint16_t *const (&xfrag)[4], int nks, int cb0, int c, int h,
                                                uint16_t (*Bs)[128 * G4_BP], f4_t (&acc)[4][4]) {
    // A fragments in two register sets, a full step apart: set X serves even steps and set Y odd ones; each set is
    // refilled for the step after next as soon as its MFMAs have issued, so a fragment has a whole step to arrive.
    uint4 AX[4][2], AY[4][2];
    auto load_a = [&](int ks, uint4 (&A)[4][2]) __attribute__((always_inline)) {
        const int kk = min(ks, nks - 1);
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int rb = 0; rb < NRB; rb++)
                A[rb][kb] = *reinterpret_cast<const uint4 *>(xfrag[rb] + (size_t)(kk * 2 + kb) * 512);
    };
    load_a(0, AX);
    load_a(1, AY);
    __syncthreads();  // barrier 0
    auto mstep = [&](int ks, uint4 (&A)[4][2]) __attribute__((always_inline)) {
        const uint16_t *slab = Bs[(ks >> 1) & 1] + (ks & 1) * (TR ? 64 * G4_BP : 64);  // super-step ks / 2, its k half ks & 1
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            uint4 bv[4];  // this half-step's B fragments (the A sets hold the registers a whole step of B would take)
#pragma unroll
            for (int cb = 0; cb < 4; cb++) {
                if constexpr (TR) {
                    const uint16_t *p = slab + (kb * 32 + 8 * h + (c >> 2)) * G4_BP + (cb0 + cb) * 16 + 4 * (c & 3);
                    const uint2 lo = read_transposed(p), hi = read_transposed(p + 4 * G4_BP);
                    bv[cb] = uint4{lo.x, lo.y, hi.x, hi.y};
                } else {
                    bv[cb] = *reinterpret_cast<const uint4 *>(slab + ((cb0 + cb) * 16 + c) * G4_BP + kb * 32 + 8 * h);
                }
            }
#pragma unroll
            for (int cb = 0; cb < 4; cb++) {
                const h8_t B8 = __builtin_bit_cast(h8_t, bv[cb]);
#pragma unroll
                for (int rb = 0; rb < NRB; rb++)
                    acc[rb][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, A[rb][kb]), B8,
                                                                         acc[rb][cb], 0, 0, 0);
            }
        }
        load_a(ks + 2, A);
    };
    for (int ks = 0; ks < nks; ks += 2) {  // nks is even: one super-step
        mstep(ks, AX);
        mstep(ks + 1, AY);
        __syncthreads();
    }
}

// ---- the decoders' readers: where a decoder finds k-tile row rs * i + r of its output group in its i-th load (the
// group's 8 tiles, lane 8 o + j reading chunk j of tile o; rs = 4 or 8 rows apart), and how a lane's chunk decodes.
// load(i) is called for i = 0, 1, 2, ... in order (past the last, nks - 1, it re-reads the last).
// One rate N for the bank: the row lies `kstep` halves further each load.
template <int FAM, int N>
struct RateReader {
    static constexpr int AW = LaneBits<N>::AW;
    const uint16_t *tb;  // the row in k-step 0
    size_t kstep;
    uint32_t lane_words;
    int j, nks;
    DecodeK k;
    __device__ __forceinline__ RateReader(const uint16_t *bank, int r, int rs, int OT, int og, int nks_, int lane,
                                          const DecodeK &k_)
        : tb(bank + ((size_t)r * OT + og * 8) * N), kstep((size_t)rs * OT * N),
          lane_words((uint32_t)((lane >> 3) * N) >> 1), j(lane & 7), nks(nks_), k(k_) {}
    __device__ __forceinline__ void load(int ks, uint32_t (&W)[AW]) {
        load_lane_words_u<N>(reinterpret_cast<const uint32_t *>(tb + (size_t)min(ks, nks - 1) * kstep), lane_words,
                             j, W);
    }
    __device__ __forceinline__ void decode(const uint32_t (&W)[AW], uint32_t (&w)[16]) const {
        if (k.wmask != 0xFFFFu) decode_weights<FAM, N, true>(W, k, w);
        else decode_weights<FAM, N, false>(W, k, w);
    }
};

// A per-tile-rate projection (a K1 / K2 mix): the row of load i is segment seg0 + i * seg_step, at the
// word offset and with the rate mask of the segment tables; lane 8 o + j's tile starts 16 o - 8 popcount(mask below o)
// words in, at TILED_NA when bit o is set.  The segment's offset and mask (scalar loads) are fetched two loads ahead,
// so a tile's vector loads never wait on them, also where a decoder issues two loads back to back.
template <int FAM>
struct TiledReader {
    static constexpr int AW = 4;  // the lane's three words and its tile's rate flag
    const uint32_t *words;        // the projection's whole trellis
    const uint32_t *seg_off;
    const uint8_t *seg_k1;
    size_t seg0, seg_step;
    int o, j, nks;
    DecodeK ka, kb;
    uint32_t n_off, n_m, f_off, f_m;  // offset and mask of the next load and of the one after it
    __device__ __forceinline__ TiledReader(const uint16_t *trellis, const uint32_t *off, const uint8_t *k1, int e,
                                           int r, int rs, int IT, int OT, int og, int nks_, int lane,
                                           const DecodeK &ka_, const DecodeK &kb_)
        : words(reinterpret_cast<const uint32_t *>(trellis)), seg_off(off), seg_k1(k1),
          seg0(((size_t)e * IT + r) * (size_t)(OT >> 3) + og), seg_step((size_t)rs * (OT >> 3)), o(lane >> 3),
          j(lane & 7), nks(nks_), ka(ka_), kb(kb_) {
        fetch(0, n_off, n_m);
        fetch(1, f_off, f_m);
    }
    __device__ __forceinline__ void fetch(int ks, uint32_t &off, uint32_t &m) const {
        const size_t seg = seg0 + (size_t)min(ks, nks - 1) * seg_step;
        m = seg_mask(seg_k1, seg);
        off = seg_off[seg];
    }
    __device__ __forceinline__ void load(int ks, uint32_t (&W)[AW]) {
        const uint32_t m = n_m, off = n_off;
        const bool k1 = ((m >> o) & 1u) != 0;
        const uint32_t lw = 16u * (uint32_t)o - 8u * (uint32_t)__builtin_popcount(m & ((1u << o) - 1u));
        uint32_t A[3];
        load_lane_words_tiled(words + off, lw, j, k1, A);
        W[0] = A[0];
        W[1] = A[1];
        W[2] = A[2];
        W[3] = k1 ? 1u : 0u;
        n_off = f_off;
        n_m = f_m;
        fetch(ks + 2, f_off, f_m);
    }
    __device__ __forceinline__ void decode(const uint32_t (&W)[AW], uint32_t (&w)[16]) const {
        const uint32_t A[3] = {W[0], W[1], W[2]};
        const bool k1 = W[3] != 0;
        if (kb.wmask != 0xFFFFu) decode_weights_tiled<FAM, true>(A, k1, ka, kb, w);
        else decode_weights_tiled<FAM, false>(A, k1, ka, kb, w);
    }
};

// The decoders of the decode-wave tile, D of them (4: waves 8-11; 8: waves 8-11 and 4-7), decoder d decoding rows
// d + 4 t (t < 8 / D) of each super-step into the slab the MFMA waves read after the super-step's barrier, the words
// of the next super-step in flight.  The reader takes row d every 8 / D loads apart (4 rows apart for D = 4, 8 for
// D = 8), nsup * 8 / D loads in all.  1 + nsup barriers.
template <int FAM, int D, class R>
__device__ __forceinline__ void gemm4_decode_waves(R &rd, int nsup, int d, int lane, uint16_t (*Bs)[128 * G4_BP]) {
    static_assert(D == 4 || D == 8, "four or eight decoders");
    constexpr int T = 8 / D;  // rows per decoder per super-step
    const int o = lane >> 3, j = lane & 7;
    auto decode_store = [&](const uint32_t (&W)[R::AW], uint16_t *slab, int row) __attribute__((always_inline)) {
        uint32_t w[16];
        rd.decode(W, w);
        uint16_t *cj = slab + (o * 16 + j) * G4_BP + row * 16;
        uint16_t *cj8 = cj + 8 * G4_BP;
        *reinterpret_cast<uint4 *>(cj) = uint4{w[0], w[4], w[8], w[12]};
        *reinterpret_cast<uint4 *>(cj + 8) = uint4{w[1], w[5], w[9], w[13]};
        *reinterpret_cast<uint4 *>(cj8) = uint4{w[2], w[6], w[10], w[14]};
        *reinterpret_cast<uint4 *>(cj8 + 8) = uint4{w[3], w[7], w[11], w[15]};
    };
    uint32_t P[T][R::AW], Q[T][R::AW];
#pragma unroll
    for (int t = 0; t < T; t++) rd.load(t, P[t]);
#pragma unroll
    for (int t = 0; t < T; t++) rd.load(T + t, Q[t]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < T; t++) decode_store(P[t], Bs[0], d + 4 * t);
    __syncthreads();  // barrier 0: slab 0 is ready
    // super-step S: the words of S + 2 into the set just decoded, S + 1's rows into slab (S + 1) & 1
    auto sstep = [&](int S, const uint32_t (&C)[T][R::AW], uint32_t (&Nx)[T][R::AW]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < T; t++) rd.load(T * (S + 2) + t, Nx[t]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < T; t++) decode_store(C[t], Bs[(S + 1) & 1], d + 4 * t);
        __syncthreads();
    };
    int S = 0;
    for (; S + 1 < nsup; S += 2) {
        sstep(S, Q, P);
        sstep(S + 1, P, Q);
    }
    if (S < nsup) sstep(S, Q, P);
}

// The MFMA waves (waves 0-7) of one workgroup's 256-row x 128-column output tile: prepared rows in fragment tiles from
// xfrag0 (row tile rt at xfrag0 + rt * (in / 32) * 512), of which the first `rows` (<= 256) are live.  The epilogue
// hands the raw inner products of rows m .. m + 3 to emit(m, live, v0[4], v1[4], lane, rid) (columns lane and
// lane + 64 of the group, m the row within the tile, the first `live` of them live); the caller applies the output
// transform (four rows at a time) or stores the raw values.  With row_ids, lane l of rid holds row_ids[m0 + l] for the
// wave's row group m0 .. m0 + 63 (loaded before the main loop, so the epilogue finds each row's id with a lane read
// instead of a memory round trip per row); without, rid is 0.
// nks: 64-k steps (even), xfrag0 at the first of them; TR as gemm4_mfma_loop.
// ALL: every row block is staged before the first is handed on (Bs then holds G4_STAGE_ALL bytes), so emit is one body in a
// loop: for an epilogue of some length, whose eight copies would not stay in the instruction cache.
template <bool TR = false, bool ALL = false, class Emit>
__device__ __forceinline__ void gemm4_mfma_waves(int in, int nks, const uint16_t *__restrict__ xfrag0, int rows,
                                                 const uint32_t *__restrict__ row_ids, uint16_t (*Bs)[128 * G4_BP],
                                                 Emit emit) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // A row group wholly past the live rows (a short window or row tail) has nothing to compute and leaves at once;
    // like the decode waves' exit, an ended wave no longer counts at the barriers.
    const int m0 = (wave >> 1) * 64, cb0 = (wave & 1) * 4;
    if (m0 >= rows) return;
    const uint32_t rid = row_ids ? row_ids[min(m0 + lane, rows - 1)] : 0u;
    const int c = lane & 15, h = lane >> 4;
    const int RT = (rows + 15) / 16;
    const uint16_t *xfrag[4];
#pragma unroll
    for (int rb = 0; rb < 4; rb++) {
        const int rt = min(m0 / 16 + rb, RT - 1);
        xfrag[rb] = xfrag0 + (size_t)rt * (size_t)(in / 32) * 512 + (size_t)lane * 8;
    }
    f4_t acc[4][4];
#pragma unroll
    for (int rb = 0; rb < 4; rb++)
#pragma unroll
        for (int cb = 0; cb < 4; cb++) acc[rb][cb] = f4_t{0.f, 0.f, 0.f, 0.f};
    switch (min(4, RT - m0 / 16)) {  // the wave's live 16-row blocks
    case 1: gemm4_mfma_loop<1, TR>(xfrag, nks, cb0, c, h, Bs, acc); break;
    case 2: gemm4_mfma_loop<2, TR>(xfrag, nks, cb0, c, h, Bs, acc); break;
    case 3: gemm4_mfma_loop<3, TR>(xfrag, nks, cb0, c, h, Bs, acc); break;
    default: gemm4_mfma_loop<4, TR>(xfrag, nks, cb0, c, h, Bs, acc); break;
    }

    // ---- epilogue (the decode waves have left, so the barriers below join the live MFMA waves): per 16-row block, the
    // two waves of a row group stage their column halves side by side in LDS, then each hands 8 of the rows on.
    if constexpr (ALL) {
        float *ep = reinterpret_cast<float *>(&Bs[0][0]) + (wave >> 1) * 64 * G2_EP;
#pragma unroll
        for (int rb = 0; rb < 4; rb++)
#pragma unroll
            for (int cb = 0; cb < 4; cb++)
#pragma unroll
                for (int i = 0; i < 4; i++) ep[(rb * 16 + 4 * h + i) * G2_EP + (cb0 + cb) * 16 + c] = acc[rb][cb][i];
        __syncthreads();
#pragma unroll 1
        for (int q = 0; q < 8; q++) {
            const int r = (q >> 1) * 16 + (wave & 1) * 8 + (q & 1) * 4, m = m0 + r;
            if (m >= rows) break;
            float v0[4], v1[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v0[i] = ep[(r + i) * G2_EP + lane];
                v1[i] = ep[(r + i) * G2_EP + lane + 64];
            }
            emit(m, min(4, rows - m), v0, v1, lane, rid);
        }
        return;
    }
    float *ep = reinterpret_cast<float *>(&Bs[0][0]) + (wave >> 1) * 16 * G2_EP;
#pragma unroll
    for (int rb = 0; rb < 4; rb++) {
#pragma unroll
        for (int cb = 0; cb < 4; cb++)
#pragma unroll
            for (int i = 0; i < 4; i++) ep[(4 * h + i) * G2_EP + (cb0 + cb) * 16 + c] = acc[rb][cb][i];
        __syncthreads();
#pragma unroll
        for (int r4 = 0; r4 < 8; r4 += 4) {
            const int r = (wave & 1) * 8 + r4, m = m0 + rb * 16 + r;
            if (m >= rows) break;
            float v0[4], v1[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v0[i] = ep[(r + i) * G2_EP + lane];
                v1[i] = ep[(r + i) * G2_EP + lane + 64];
            }
            emit(m, min(4, rows - m), v0, v1, lane, rid);
        }
        __syncthreads();
    }
}

// This wave's decoder index in the decode-wave tile, or -1 for an MFMA wave: waves 8-11 are decoders 0-3; with the
// live rows within G4_HELP_ROWS, waves 4-7 (whose row groups are empty) are decoders 4-7.
__device__ __forceinline__ int gemm4_decoder(int wave, int rows) {
    if (wave >= 8) return wave - 8;
    return (rows <= G4_HELP_ROWS && wave >= 4) ? wave : -1;
}

// Decoder d over the reader mk(r, rs, loads) makes (row r, rows rs apart, `loads` loads): eight decoders when `help`
// (the live rows within G4_HELP_ROWS), else four.
template <int FAM, class MakeReader>
__device__ __forceinline__ void gemm4_decode_role(bool help, int d, int nsup, int lane, uint16_t (*Bs)[128 * G4_BP],
                                                  MakeReader mk) {
    if (help) {
        auto rd = mk(d, 8, nsup);
        gemm4_decode_waves<FAM, 8>(rd, nsup, d, lane, Bs);
    } else {
        auto rd = mk(d, 4, 2 * nsup);
        gemm4_decode_waves<FAM, 4>(rd, nsup, d, lane, Bs);
    }
}

// One workgroup's 256-row x 128-column output tile of output group og of a bank at one rate N whose tiles start at
// `bank` ([in/16][out/16][N]): the decoders (gemm4_decoder) decode, the other waves multiply (gemm4_mfma_waves, whose
// `emit` receives the raw inner products).
template <int FAM, int N, bool ALL = false, class Emit>
__device__ __forceinline__ void gemm4_tile(int in, int out, int og, const uint16_t *__restrict__ bank,
                                           const uint16_t *__restrict__ xfrag0, int rows, const uint32_t *row_ids,
                                           const DecodeK &k, uint16_t (*Bs)[128 * G4_BP], Emit emit) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int d = gemm4_decoder(wave, rows);
    if (d >= 0) {
        gemm4_decode_role<FAM>(rows <= G4_HELP_ROWS, d, in >> 7, lane, Bs, [&](int r, int rs, int loads) {
            return RateReader<FAM, N>(bank, r, rs, out >> 4, og, loads, lane, k);
        });
        return;
    }
    gemm4_mfma_waves<false, ALL>(in, in >> 6, xfrag0, rows, row_ids, Bs, emit);  // in is a multiple of 128
}

}  // namespace exl3
