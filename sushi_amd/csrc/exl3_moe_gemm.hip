// The routed GEMM arm's kernels (moePrefill, beamivalice/sushi src/exl3/expert_exl3_kernels.zig:2861-2931): the prepare,
// the expert-window GEMM on the decode-wave tile (exl3_gemm_tile.h) and the mid.
#include "exl3_gemm_tile.h"

namespace exl3 {

// Expert index of a window (routed ones clamped below `experts`; with a shared expert, `experts` is it) and the token
// row of a slot (routed slot s is token s / topk, shared slot nslots + r is token r).
__device__ __forceinline__ int moe_expert(const MoeGemmArgs &a, uint32_t e) {
    return (int)min(e, (uint32_t)(a.experts - 1 + a.sh));
}
__device__ __forceinline__ uint32_t moe_token(const MoeGemmArgs &a, uint32_t slot) {
    return slot < (uint32_t)a.nslots ? slot / (uint32_t)a.topk : slot - (uint32_t)a.nslots;
}

// ---- the routed GEMM arm: workgroup (og, window w, projection p) runs the tile of window w's rows against its
// expert's bank and writes the raw inner products to planes[p][slot][out] (the mid / the reduce applies the output
// transform).  Windows past the count exit before any barrier.  Workgroups go out to the XCDs in turn (L & 7), so
// the out / 128 column groups of one window are numbered to land on one XCD one after another: they read the same
// prepared rows, which then come from that XCD's L2 after the first (numbered by the window, each group would pull
// them through its own XCD's L2).
// N > 0: a uniform bank at rate N.  N == -1: a ragged bank (`rate_groups.moePrefill`, rate_groups.zig:2039-2075):
// each workgroup reads its expert's rate and tile offset from the meta table and its decode waves take that rate's
// reader (one launch for every rate group; the MFMA waves are the same for all).  N == N_TILED: a per-tile-rate bank,
// the decode waves reading each k-step's segment offset and rate mask.  Either way a fused shared expert (expert
// `experts`) decodes at its own uniform rate sh_n.
template <int FAM>
__device__ __forceinline__ DecodeK rate_decode(const DecodeK &base, int table, int n) {
    DecodeK k = base;
    if constexpr (FAM == FAM_HASH || FAM == FAM_PAIR) table_row(table, n, k.mult, k.mask0, k.mask1, k.rot);
    return k;
}

// Decoder d at a rate known only at run time (a lane-reader rate; any other leaves the slab undecoded, which the
// host rules out).
template <int FAM>
__device__ __forceinline__ void gemm4_decode_waves_at(int n, const uint16_t *bank, int OT, int og, int nsup, int d,
                                                      bool help, int lane, const DecodeK &k,
                                                      uint16_t (*Bs)[128 * G4_BP]) {
    switch (n) {
#define EXL3_RATE_CASE(NN)                                                                                             \
    case NN:                                                                                                           \
        gemm4_decode_role<FAM>(help, d, nsup, lane, Bs, [&](int r, int rs, int loads) {                                \
            return RateReader<FAM, NN>(bank, r, rs, OT, og, loads, lane, k);                                           \
        });                                                                                                            \
        break;
        EXL3_RATE_CASE(16)
        EXL3_RATE_CASE(24)
        EXL3_RATE_CASE(32)
        EXL3_RATE_CASE(40)
        EXL3_RATE_CASE(48)
        EXL3_RATE_CASE(64)
#undef EXL3_RATE_CASE
    default: break;
    }
}

template <int FAM, int N>
__global__ __launch_bounds__(G4_THREADS) void moe_gemm4_kernel(MoeGemmArgs a) {
    const int nog = a.out / 128, L = blockIdx.x, q = L >> 3;
    const int og = q % nog, w = (q / nog) * 8 + (L & 7), p = blockIdx.y;
    if ((uint32_t)w >= *a.win.win_count) return;
    const int IT = a.in >> 4, OT = a.out >> 4;
    const int e = moe_expert(a, a.win.win_expert[w]);
    const int rows = (int)min(a.win.win_rows[w], (uint32_t)G2_MT);
    const uint32_t *slots = a.win.sorted + a.win.win_start[w];
    __shared__ __align__(16) uint16_t Bs[2][128 * G4_BP];
    const uint16_t *xfrag0 = a.xp[p] + (size_t)a.win.win_tile0[w] * (size_t)(a.in / 32) * 512;
    float *planes = a.planes[p];
    auto emit = [&](int m, int live, float (&v0)[4], float (&v1)[4], int ln, uint32_t rid)
                    __attribute__((always_inline)) {
        for (int i = 0; i < live; i++) {  // rid: the slot of row (m & ~63) + lane
            const uint32_t slot = (uint32_t)__builtin_amdgcn_readlane((int)rid, (m & 63) + i);
            float *row = planes + (size_t)slot * a.out + (size_t)og * 128;
            row[ln] = v0[i] * codebook_scale<FAM>();
            row[ln + 64] = v1[i] * codebook_scale<FAM>();
        }
    };
    if constexpr (N > 0) {
        const uint16_t *bank = e < a.experts ? a.trellis[p] + (size_t)e * IT * OT * N : a.sh_trellis[p];
        gemm4_tile<FAM, N>(a.in, a.out, og, bank, xfrag0, rows, slots, a.k, Bs, emit);
    } else {
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        const int d = gemm4_decoder(wave, rows);
        if (d < 0) {
            gemm4_mfma_waves(a.in, a.in >> 6, xfrag0, rows, slots, Bs, emit);
            return;
        }
        const int nsup = IT / 8;
        const bool help = rows <= G4_HELP_ROWS;
        if (e >= a.experts) {  // the shared expert: its own uniform bank
            gemm4_decode_waves_at<FAM>(a.sh_n, a.sh_trellis[p], OT, og, nsup, d, help, lane,
                                       rate_decode<FAM>(a.k, a.table, a.sh_n), Bs);
            return;
        }
        if constexpr (N == N_TILED) {
            const DecodeK ka = rate_decode<FAM>(a.k, a.table, TILED_NA), kb = rate_decode<FAM>(a.k, a.table, TILED_NB);
            gemm4_decode_role<FAM>(help, d, nsup, lane, Bs, [&](int r, int rs, int loads) {
                return TiledReader<FAM>(a.trellis[p], a.seg_off[p], a.seg_k1[p], e, r, rs, IT, OT, og, loads, lane, ka,
                                        kb);
            });
        } else {
            const uint32_t *m = a.meta + (size_t)e * 8;
            const int col = a.meta_col[p];
            const int n = (int)m[col];
            gemm4_decode_waves_at<FAM>(n, a.trellis[p] + 2 * (size_t)m[4 + col], OT, og, nsup, d, help, lane,
                                       rate_decode<FAM>(a.k, a.table, n), Bs);
        }
    }
}

// ---- the routed GEMM arm's inputs.  Tile t (16 sorted rows of one window, the window's tiles contiguous from
// win_tile0) is prepared into fragment order at xp + t * (in / 32) * 512, as gemm_prepare_frag_kernel does for dense
// rows; rows past the window's end are zeros.  Tiles past the count exit at once.
struct TileRows {
    bool live;
    int rows;             // live rows of the tile (16 unless the window's last)
    int e;                // the window's expert
    const uint32_t *slots;
};

__device__ __forceinline__ TileRows tile_rows(const MoeGemmArgs &a, int t) {
    TileRows r;
    const uint4 ti = a.win.tile_info[t];  // t < max_tiles (the grid); read beside the count, used only if live
    r.live = (uint32_t)t < *a.win.tile_count;
    if (!r.live) return r;
    r.rows = (int)ti.y;
    r.e = moe_expert(a, ti.x);
    r.slots = a.win.sorted + ti.z;
    return r;
}

// The 16 x 128 f16 tile in LDS to fragment order (one 16-byte store per thread).
__device__ __forceinline__ void tile_to_frag(const uint16_t (*tl)[128 + 8], uint16_t *xp, int t, int b, int in,
                                             int tid) {
    const int lane = tid & 63, kq = tid >> 6, c = lane & 15, h = lane >> 4;
    const uint4 v = *reinterpret_cast<const uint4 *>(&tl[c][kq * 32 + 8 * h]);
    *reinterpret_cast<uint4 *>(xp + ((size_t)t * (in / 32) + (size_t)b * 4 + kq) * 512 + (size_t)lane * 8) = v;
}

// prepareInput (expert_exl3.zig:490-501) of each row's token with its expert's suh, for gate and up from one load of
// the rows, over NB consecutive 128-column blocks of one tile.  Every load is in bounds (a row past the tile's end
// reads the tile's last live row and is zeroed after), so a wave's four rows of every block go out together with the
// suh loads, behind only the tile's table and slot reads; the transforms then run for both projections at once.
// (A workgroup per projection gathered each token row from memory once per projection: 95 us at 2048 tokens.)
template <int NB, int DT>
__global__ __launch_bounds__(256) void moe_gemm_prepare_kernel(MoeGemmArgs a) {
    const int b0 = blockIdx.x * NB, t = blockIdx.y;
    const TileRows tr = tile_rows(a, t);
    if (!tr.live) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ __align__(16) uint16_t tl[NB][2][16][128 + 8];
    const bool shx = tr.e >= a.experts;
    const size_t se = shx ? 0 : (size_t)tr.e * a.in;
    uint32_t sl[4];
#pragma unroll
    for (int rr = 0; rr < 4; rr++) sl[rr] = tr.slots[min(wave * 4 + rr, max(tr.rows - 1, 0))];
    size_t xr[4];
#pragma unroll
    for (int rr = 0; rr < 4; rr++) xr[rr] = (size_t)moe_token(a, __builtin_amdgcn_readfirstlane(sl[rr])) * a.in;
    float x0[NB][4], x1[NB][4], u0[NB][2], u1[NB][2];
#pragma unroll
    for (int rr = 0; rr < 4; rr++)
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const size_t xi = xr[rr] + (size_t)(b0 + nb) * 128;
            x0[nb][rr] = load_act<DT>(a.x, xi + lane);
            x1[nb][rr] = load_act<DT>(a.x, xi + lane + 64);
        }
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const uint16_t *su = shx ? a.sh_suh[q] : a.suh[q];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            const size_t si = se + (size_t)(b0 + nb) * 128;
            u0[nb][q] = h2f(su[si + lane]);
            u1[nb][q] = h2f(su[si + lane + 64]);
        }
    }
    const float sc = fwht_relaid_sign(lane) * HAD_SCALE;
    const int c0 = fwht_relaid_col(lane, 0), c1 = fwht_relaid_col(lane, 1);
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
        float v0[8], v1[8];  // [projection][row]; rows past the end are zeros
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const bool live = wave * 4 + rr < tr.rows;
            const float y0 = live ? f16r(x0[nb][rr]) : 0.f, y1 = live ? f16r(x1[nb][rr]) : 0.f;
#pragma unroll
            for (int q = 0; q < 2; q++) {
                v0[q * 4 + rr] = y0 * u0[nb][q];
                v1[q * 4 + rr] = y1 * u1[nb][q];
            }
        }
        fwht128_wave_rows_relaid<8>(v0, v1, lane);
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int rr = 0; rr < 4; rr++) {
                const int r = wave * 4 + rr;
                tl[nb][q][r][c0] = __half_as_ushort(__float2half_rn(v0[q * 4 + rr] * sc));
                tl[nb][q][r][c1] = __half_as_ushort(__float2half_rn(v1[q * 4 + rr] * sc));
            }
    }
    __syncthreads();
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int q = 0; q < 2; q++) tile_to_frag(tl[nb][q], a.xp[q], t, b0 + nb, a.in, tid);
}

// The SwiGLU mid of the routed GEMM arm (DOWN_FUSED_SOURCE's prologue, expert_exl3_kernels.zig:1838-1925; the
// decode chain's PRO_MID with one plane): gate and up = svh * H(raw inner), the clamps, SiLU(gate) * up * suh_down,
// H, f16 -- the down projection's prepared input, in fragment order at xp[0] (a.in = inter).
__global__ __launch_bounds__(256) void moe_gemm_mid_kernel(MoeGemmArgs a) {
    const int b = blockIdx.x, t = blockIdx.y;
    const TileRows tr = tile_rows(a, t);
    if (!tr.live) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ __align__(16) uint16_t tl[16][128 + 8];
    const bool shx = tr.e >= a.experts;  // the shared expert's rows: its own scales
    const size_t si = (shx ? 0 : (size_t)tr.e * a.in) + (size_t)b * 128;
    const uint16_t *svg = shx ? a.sh_mid_svh[0] : a.mid_svh[0], *svu = shx ? a.sh_mid_svh[1] : a.mid_svh[1];
    const uint16_t *sud = shx ? a.sh_down_suh : a.down_suh;
    // the gate / up transforms leave column fwht_relaid_col(lane, s) in slot s, so the scales are read there
    const int c0 = fwht_relaid_col(lane, 0), c1 = fwht_relaid_col(lane, 1);
    const float sg0 = h2f(svg[si + c0]), sg1 = h2f(svg[si + c1]);
    const float su0 = h2f(svu[si + c0]), su1 = h2f(svu[si + c1]);
    const float sd0 = h2f(sud[si + c0]), sd1 = h2f(sud[si + c1]);
    // the wave's four rows, both planes, all loads in bounds and out together (a row past the tile's end reads the
    // last live row and is zeroed after)
    uint32_t sl[4];
#pragma unroll
    for (int rr = 0; rr < 4; rr++) sl[rr] = tr.slots[min(wave * 4 + rr, max(tr.rows - 1, 0))];
    float w0[8], w1[8];  // [gate rows 0..3, up rows 0..3]
#pragma unroll
    for (int rr = 0; rr < 4; rr++) {
        const size_t pi = (size_t)__builtin_amdgcn_readfirstlane(sl[rr]) * a.in + (size_t)b * 128;
        w0[rr] = a.mid_planes[0][pi + lane];
        w1[rr] = a.mid_planes[0][pi + lane + 64];
        w0[4 + rr] = a.mid_planes[1][pi + lane];
        w1[4 + rr] = a.mid_planes[1][pi + lane + 64];
    }
#pragma unroll
    for (int rr = 0; rr < 4; rr++)
        if (wave * 4 + rr >= tr.rows) w0[rr] = w1[rr] = w0[4 + rr] = w1[4 + rr] = 0.f;
    fwht128_wave_rows_relaid<8>(w0, w1, lane);
    // the transforms' sign folded into the scales (exact: both factors change sign)
    const float sgn = fwht_relaid_sign(lane);
    const float kg0 = sgn * (HAD_SCALE * sg0), kg1 = sgn * (HAD_SCALE * sg1);
    const float ku0 = sgn * (HAD_SCALE * su0), ku1 = sgn * (HAD_SCALE * su1);
    float v0[4], v1[4];
#pragma unroll
    for (int rr = 0; rr < 4; rr++) {
        float a0 = w0[rr] * kg0, a1 = w1[rr] * kg1;
        float b0 = w0[4 + rr] * ku0, b1 = w1[4 + rr] * ku1;
        if (a.clamp_limit > 0.f) {
            a0 = fminf(a0, a.clamp_limit);
            a1 = fminf(a1, a.clamp_limit);
            b0 = fminf(fmaxf(b0, -a.clamp_limit), a.clamp_limit);
            b1 = fminf(fmaxf(b1, -a.clamp_limit), a.clamp_limit);
        }
        v0[rr] = silu(a0) * b0 * sd0;
        v1[rr] = silu(a1) * b1 * sd1;
    }
    fwht128_wave_rows_relaid<4, true>(v0, v1, lane);  // rows past the end: silu(0) * 0 = 0, zeros stay zeros
    const float sc = sgn * HAD_SCALE;
    const int d0 = fwht_relaid2_col(lane, 0), d1 = fwht_relaid2_col(lane, 1);
#pragma unroll
    for (int rr = 0; rr < 4; rr++) {
        const int r = wave * 4 + rr;
        tl[r][d0] = __half_as_ushort(__float2half_rn(v0[rr] * sc));
        tl[r][d1] = __half_as_ushort(__float2half_rn(v1[rr] * sc));
    }
    __syncthreads();
    tile_to_frag(tl, a.xp[0], t, b, a.in, tid);
}

template <int DT>
static void launch_moe_gemm_prepare(const MoeGemmArgs &a, hipStream_t s) {
    // two 128-column blocks a workgroup where they pair up (measured at 2048 tokens of 2048 x 768, top-8 of 256: 85 -> 79 us; four
    // blocks took 110)
    const int blocks = a.in / 128;
    if (blocks % 2 == 0)
        hipLaunchKernelGGL((moe_gemm_prepare_kernel<2, DT>), dim3((unsigned)(blocks / 2), (unsigned)a.max_tiles),
                           dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((moe_gemm_prepare_kernel<1, DT>), dim3((unsigned)blocks, (unsigned)a.max_tiles), dim3(256),
                           0, s, a);
}

hipError_t run_moe_gemm_prepare(const MoeGemmArgs &a, int nproj, hipStream_t s) {
    if (nproj != 2) return hipErrorInvalidValue;  // gate and up together
    if (a.x_dtype == DT_F16) launch_moe_gemm_prepare<DT_F16>(a, s);
    else if (a.x_dtype == DT_BF16) launch_moe_gemm_prepare<DT_BF16>(a, s);
    else launch_moe_gemm_prepare<DT_F32>(a, s);
    return hipGetLastError();
}

hipError_t run_moe_gemm_mid(const MoeGemmArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(moe_gemm_mid_kernel, dim3((unsigned)(a.in / 128), (unsigned)a.max_tiles), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int FAM>
static hipError_t launch_moe_gemm_fam(const MoeGemmArgs &a, int nproj, hipStream_t s) {
    // x: column group and window, the windows rounded up to whole rounds of the 8 XCDs (the extra ones exit)
    const dim3 grid((unsigned)(a.out / 128) * (unsigned)((a.max_windows + 7) / 8 * 8), (unsigned)nproj);
    if (a.seg_off[0]) {  // per-tile rates: the hash-product families
        if constexpr (FAM == FAM_PAIR || FAM == FAM_MUL1) return hipErrorInvalidValue;
        else hipLaunchKernelGGL((moe_gemm4_kernel<FAM, N_TILED>), grid, dim3(G4_THREADS), 0, s, a);
        return hipGetLastError();
    }
    if (a.meta) {
        hipLaunchKernelGGL((moe_gemm4_kernel<FAM, -1>), grid, dim3(G4_THREADS), 0, s, a);
        return hipGetLastError();
    }
    switch (a.n) {
    case 16: hipLaunchKernelGGL((moe_gemm4_kernel<FAM, 16>), grid, dim3(G4_THREADS), 0, s, a); break;
    case 24: hipLaunchKernelGGL((moe_gemm4_kernel<FAM, 24>), grid, dim3(G4_THREADS), 0, s, a); break;
    case 32: hipLaunchKernelGGL((moe_gemm4_kernel<FAM, 32>), grid, dim3(G4_THREADS), 0, s, a); break;
    case 40: hipLaunchKernelGGL((moe_gemm4_kernel<FAM, 40>), grid, dim3(G4_THREADS), 0, s, a); break;
    case 48: hipLaunchKernelGGL((moe_gemm4_kernel<FAM, 48>), grid, dim3(G4_THREADS), 0, s, a); break;
    case 64: hipLaunchKernelGGL((moe_gemm4_kernel<FAM, 64>), grid, dim3(G4_THREADS), 0, s, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t run_moe_gemm(int fam, const MoeGemmArgs &a, int nproj, hipStream_t s) {
    switch (fam) {
    case FAM_MCG: return launch_moe_gemm_fam<FAM_MCG>(a, nproj, s);
    case FAM_MUL1: return launch_moe_gemm_fam<FAM_MUL1>(a, nproj, s);
    case FAM_HASH: return launch_moe_gemm_fam<FAM_HASH>(a, nproj, s);
    case FAM_PAIR: return launch_moe_gemm_fam<FAM_PAIR>(a, nproj, s);
    default: return launch_moe_gemm_fam<FAM_3INST>(a, nproj, s);
    }
}

}  // namespace exl3
