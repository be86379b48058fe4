// The backward pass of a linear with an epilogue over a frozen trellis bank: with z = project(x) + bias and
// y = act(z) + residual,
//   dz = dy * act'(z),  dbias = sum over rows of dz,  dx = H(u W^T) * suh,  u = f16(H(dz * svh))
// (H: the orthonormal Hadamard transform of every 128; residual's gradient is dy itself).  u is rounded to f16 as the
// forward's prepared input is, under a power of two per row that brings the row's largest |dz * svh| to 2^10 .. 2^11:
// gradients lie far below f16's normal range, and |H v| <= sqrt(128) max |v| keeps the scaled values below 2^15.  (The largest
// |dy * svh| would spare the scan pre and the slopes, but a row whose activations are all saturated, or one large gradient on
// a dead unit, would then leave u in f16's subnormals: at pre = -7 +- 0.2 with gelu dx was off by 28 to 43% of its row's
// largest value, at -9, with gelu_tanh at -6.5 or silu at -30 all of it.)
//
//   grad_scan_kernel     reads dy and pre: each row's largest |dz * svh|
//   grad_prepare_kernel  reads dy and pre: u in MFMA A-fragment order, each row's scale, dbias's sums by row tile
//   grad_gemm_kernel     u W^T on the decode-wave tile (exl3_gemm_tile.h), the trellis decoded once per 256 rows into the
//                        same column-major slab as the forward's and read back transposed by the MFMA waves; with few
//                        row and column tiles the contraction is split
//   grad_finish_kernel   sums the splits' products in their order
// What bounds it and what it took (MI355X, medians of traced launches): 2048 rows of 4096 x 14336, n = 48, bf16,
// gelu_tanh: scan 28 us (117 MB and every slope; 12 us without an activation, dy alone at 4.8 TB/s), prepare 39 to 46 (176
// MB, 3.8 to 4.5 TB/s), dbias 5, product 241 to 269 (240 GFLOP, 0.89 to 1.00 PFLOP/s against 1.09 of a library product of
// f16 matrices, by the card's clock); 333 rows of 2560 x 16384, n = 96, gelu: 10 + 11 + 5, product 50 (its decode: 240
// workgroups, every weight decoded by each of two row tiles), finish 5; 5 rows of 4096 x 4096: 2.4 + 3.1 + 8.6 + 2.2 (each
// launch's floor about 2).
#include "exl3_gemm_tile.h"
#include "exl3_epilogue.h"

namespace exl3 {

// Eight consecutive values of a row, 8-byte aligned (the host checks; the 16-byte loads need 4).
template <int DT>
__device__ __forceinline__ void load8(const void *p, size_t i, float (&v)[8]) {
    if constexpr (DT == DT_F32) {
        typedef float f4a __attribute__((ext_vector_type(4), aligned(8)));
        const f4a a = *reinterpret_cast<const f4a *>(static_cast<const float *>(p) + i);
        const f4a b = *reinterpret_cast<const f4a *>(static_cast<const float *>(p) + i + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(8)));
        const u4a a = *reinterpret_cast<const u4a *>(static_cast<const uint16_t *>(p) + i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const uint32_t h = q & 1 ? w[q >> 1] >> 16 : w[q >> 1] & 0xFFFFu;
            v[q] = DT == DT_F16 ? h2f((uint16_t)h) : __uint_as_float(h << 16);
        }
    }
}

__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, xor_lane_row<1>(v));
    v = fmaxf(v, xor_lane_row<2>(v));
    v = fmaxf(v, xor_lane_row<4>(v));
    v = fmaxf(v, xor_lane_row<8>(v));
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// max |dz * svh| over eight columns of a row.  ACT: through an activation.
template <int DT, bool ACT>
__device__ __forceinline__ float max8(const GradArgs &a, int row, int c) {
    float d[8], m = 0.f;
    load8<DT>(a.dy, (size_t)row * a.out + c, d);
    const uint4 s = *reinterpret_cast<const uint4 *>(a.svh + c);
    if constexpr (ACT) {
        float z[8];
        load8<DT>(a.pre, (size_t)row * a.out + c, z);
        act_slopes<8>(a.act, z, d);
    }
    const uint32_t w[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int q = 0; q < 8; q++) m = fmaxf(m, fabsf(d[q] * h2f((uint16_t)(q & 1 ? w[q >> 1] >> 16 : w[q >> 1] & 0xFFFFu))));
    return m;
}

// One workgroup a row.  Through an activation its slopes are the time: they are evaluated here and again in the prepare (kept
// between them, dz would be four bytes an element to write and read in place of pre's two).
template <int DT, bool ACT>
__global__ __launch_bounds__(256) void grad_scan_kernel(GradArgs a) {
    __shared__ float part[4];
    float m = 0.f;
#pragma unroll ACT ? 1 : 4
    for (int c = threadIdx.x * 8; c < a.out; c += 2048) m = fmaxf(m, max8<DT, ACT>(a, blockIdx.x, c));
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) a.amax[blockIdx.x] = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}

// dbias from the row tiles' sums, in tile order (four interleaved shares of them, joined in order): 64 columns a
// workgroup.  A chunk of rows after the first adds to what the ones before it left.
__global__ __launch_bounds__(256) void grad_dbias_kernel(GradArgs a, int tiles) {
    __shared__ float part[4][64];
    const int lane = threadIdx.x & 63, q = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;  // out is a multiple of 128
    float s = 0.f;
#pragma unroll 8
    for (int t = q; t < tiles; t += 4) s += a.dbias_part[(size_t)t * a.out + c];
    part[q][lane] = s;
    __syncthreads();
    if (q == 0) {
        s = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
        a.dbias[c] = a.dbias_adds ? a.dbias[c] + s : s;
    }
}

// The power of two that brings m to 2^10 .. 2^11 (1 for zero and non-finite rows), and its inverse, both normal floats.
__device__ __forceinline__ int grad_exponent(float m) {
    if (!(m > 0.f) || m > 3.4028235e38f) return 0;
    const int e = (int)(__float_as_uint(m) >> 23) - 127;  // subnormals: -127, and the clamp below
    return min(max(10 - e, -126), 126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Two neighbouring values of a row.
template <int DT>
__device__ __forceinline__ void load2(const void *p, size_t i, float &x, float &y) {
    if constexpr (DT == DT_F32) {
        const float2 v = *reinterpret_cast<const float2 *>(static_cast<const float *>(p) + i);
        x = v.x, y = v.y;
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(p) + i);
        x = DT == DT_F16 ? h2f((uint16_t)w) : __uint_as_float(w << 16);
        y = DT == DT_F16 ? h2f((uint16_t)(w >> 16)) : __uint_as_float(w & 0xFFFF0000u);
    }
}

// u in A-fragment order (gemm_prepare_frag_kernel's): workgroup (128-block b, row tile) takes a.prep_tiles fragment tiles
// of 16 rows one after another, wave w their rows 4 w .. 4 w + 3, rows past the end as zeros; dbias_part[tile][col] = the
// tile's sum of dz (one row tile: dbias itself).  inv_scale is written by the workgroups of block 0.
// A lane holds columns 2 l and 2 l + 1 of a block (one load), which the transform takes as its values l and l + 64: the
// transform of any order of the index's bits is the same up to that order, so value i is column 2 (i % 64) + i / 64 on both
// of its sides.
template <int DT>
__global__ __launch_bounds__(256) void grad_prepare_kernel(GradArgs a) {
    const int b = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ __align__(16) uint16_t t[16][128 + 8];
    __shared__ float sums[4][128];
    const size_t col = (size_t)b * 128 + 2 * lane;
    const uint32_t sw = *reinterpret_cast<const uint32_t *>(a.svh + col);
    const float s0 = h2f((uint16_t)sw), s1 = h2f((uint16_t)(sw >> 16));
    const float sc = fwht_relaid_sign(lane) * HAD_SCALE;
    const int i0 = fwht_relaid_col(lane, 0), i1 = fwht_relaid_col(lane, 1);
    const int c0 = 2 * (i0 & 63) + (i0 >> 6), c1 = 2 * (i1 & 63) + (i1 >> 6);
    const int RT = (a.rows + 15) / 16, rt0 = blockIdx.y * a.prep_tiles, rt1 = min(rt0 + a.prep_tiles, RT);
    float b0 = 0.f, b1 = 0.f;
    for (int rt = rt0; rt < rt1; rt++) {
        const int m0 = rt * 16 + wave * 4;
        float v0[4], v1[4], m[4];
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const int row = min(m0 + rr, a.rows - 1);
            load2<DT>(a.dy, (size_t)row * a.out + col, v0[rr], v1[rr]);
            m[rr] = a.amax[row];
        }
        if (a.act != ACT_NONE) {
            float z0[4], z1[4];
#pragma unroll
            for (int rr = 0; rr < 4; rr++) load2<DT>(a.pre, (size_t)min(m0 + rr, a.rows - 1) * a.out + col, z0[rr], z1[rr]);
            act_slopes<4>(a.act, z0, v0);
            act_slopes<4>(a.act, z1, v1);
        }
        float two[4];
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const bool live = m0 + rr < a.rows;
            const int e = grad_exponent(m[rr]);
            two[rr] = pow2(e);
            if (b == 0 && lane == 0 && live) a.inv_scale[m0 + rr] = pow2(-e);
            v0[rr] = live ? v0[rr] : 0.f;
            v1[rr] = live ? v1[rr] : 0.f;
            b0 += v0[rr];
            b1 += v1[rr];
            v0[rr] *= s0;
            v1[rr] *= s1;
        }
        fwht128_wave_rows_relaid<4>(v0, v1, lane);
        if (rt > rt0) __syncthreads();  // the tile before has been read
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const int r = wave * 4 + rr;
            t[r][c0] = __half_as_ushort(__float2half_rn(v0[rr] * sc * two[rr]));
            t[r][c1] = __half_as_ushort(__float2half_rn(v1[rr] * sc * two[rr]));
        }
        __syncthreads();
        const int c = lane & 15, h = lane >> 4;  // 32-k block `wave` of the 128-block, fragment lane (c, h)
        const uint4 v = *reinterpret_cast<const uint4 *>(&t[c][wave * 32 + 8 * h]);
        *reinterpret_cast<uint4 *>(a.u + ((size_t)rt * (a.out / 32) + (size_t)b * 4 + wave) * 512 + (size_t)lane * 8) = v;
    }
    if (!a.dbias) return;
    sums[wave][2 * lane] = b0;
    sums[wave][2 * lane + 1] = b1;
    __syncthreads();
    if (tid < 128) {
        float *dst = a.dbias_part ? a.dbias_part + (size_t)blockIdx.y * a.out : a.dbias;
        dst[b * 128 + tid] = (sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid]);
    }
}

// The decoders' reader for the product with the transposed bank: the slab of super-step S is the input block's 8 k-tile
// rows of output group g0 + S, so load i of a decoder (rows r, r + rs, ... of a super-step) is row r + rs (i % (8 / rs)) of
// group g0 + i / (8 / rs).
template <int FAM, int N>
struct GradReader {
    static constexpr int AW = LaneBits<N>::AW;
    const uint16_t *tb;
    size_t row_step;
    uint32_t lane_words;
    int j, loads, per;
    DecodeK k;
    __device__ __forceinline__ GradReader(const uint16_t *bank, int ib, int r, int rs, int OT, int g0, int loads_, int,
                                          int lane, const DecodeK &k_)
        : tb(bank + (((size_t)ib * 8 + r) * OT + (size_t)g0 * 8) * N), row_step((size_t)rs * OT * N),
          lane_words((uint32_t)((lane >> 3) * N) >> 1), j(lane & 7), loads(loads_), per(8 / rs), k(k_) {}
    __device__ __forceinline__ void load(int i, uint32_t (&W)[AW]) {
        const int l = min(i, loads - 1);
        const uint16_t *p = tb + (size_t)(l % per) * row_step + (size_t)(l / per) * (8 * N);
        load_lane_words_u<N>(reinterpret_cast<const uint32_t *>(p), lane_words, j, W);
    }
    __device__ __forceinline__ void decode(const uint32_t (&W)[AW], uint32_t (&w)[16]) const {
        if (k.wmask != 0xFFFFu) decode_weights<FAM, N, true>(W, k, w);
        else decode_weights<FAM, N, false>(W, k, w);
    }
};

// Any other rate (N = 0): the loads only note where, and the decode reads each codeword's words.
template <int FAM>
struct GradReader<FAM, 0> {
    static constexpr int AW = 1;
    const uint16_t *tb;
    size_t row_step;
    int j, loads, per, n;
    DecodeK k;
    __device__ __forceinline__ GradReader(const uint16_t *bank, int ib, int r, int rs, int OT, int g0, int loads_, int n_,
                                          int lane, const DecodeK &k_)
        : tb(bank + (((size_t)ib * 8 + r) * OT + (size_t)g0 * 8 + (lane >> 3)) * n_), row_step((size_t)rs * OT * n_),
          j(lane & 7), loads(loads_), per(8 / rs), n(n_), k(k_) {}
    __device__ __forceinline__ void load(int i, uint32_t (&W)[AW]) { W[0] = (uint32_t)min(i, loads - 1); }
    __device__ __forceinline__ void decode(const uint32_t (&W)[AW], uint32_t (&w)[16]) const {
        const int l = (int)W[0];
#pragma unroll
        for (int q = 0; q < 16; q++) w[q] = 0u;
        const uint32_t *words =
            reinterpret_cast<const uint32_t *>(tb + (size_t)(l % per) * row_step + (size_t)(l / per) * (8 * n));
        // one pair at a time through w[15], the others shifted down: sixteen pairs' addresses would not fit the registers
#pragma unroll 1
        for (int i = 0; i < 16; i++) {
#pragma unroll
            for (int q = 0; q < 15; q++) w[q] = w[q + 1];
            w[15] = decode_pair_h2<FAM>(codeword_at(words, n, 32 * j + 2 * i), codeword_at(words, n, 32 * j + 2 * i + 1), k);
        }
    }
};

// Workgroup: a tile of dx of a.tile_rows rows (up to 256) x 128 columns (one input block ib) over the output groups of one
// split.
template <int FAM, int N>
__global__ __launch_bounds__(G4_THREADS) void grad_gemm_kernel(GradArgs a) {
    const int nib = a.in / 128, nm = (a.rows + a.tile_rows - 1) / a.tile_rows, nog = a.out / 128;
    const int sp = (int)blockIdx.x / (nib * nm), L = (int)blockIdx.x - sp * nib * nm;
    int ib, mt;
    if (nm <= 8 && 8 % nm == 0 && nib % (8 / nm) == 0) {  // a row tile's workgroups share an XCD (its u in one L2)
        const int xcd = L & 7, per = 8 / nm;
        mt = xcd / per;
        ib = (L >> 3) * per + xcd % per;
    } else {
        ib = L % nib;
        mt = L / nib;
    }
    const int g0 = (int)((long)nog * sp / a.splits), nsup = (int)((long)nog * (sp + 1) / a.splits) - g0;  // >= 1 each
    __shared__ __align__(16) uint16_t Bs[2][128 * G4_BP];
    const int rows = min(a.tile_rows, a.rows - mt * a.tile_rows);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int d = gemm4_decoder(wave, rows);
    if (d >= 0) {
        gemm4_decode_role<FAM>(rows <= G4_HELP_ROWS, d, nsup, lane, Bs, [&](int r, int rs, int loads) {
            return GradReader<FAM, N>(a.trellis, ib, r, rs, a.out >> 4, g0, loads, a.n, lane, a.k);
        });
        return;
    }
    const uint16_t *u0 = a.u + (size_t)mt * (a.tile_rows / 16) * (size_t)(a.out / 32) * 512 + (size_t)g0 * 4 * 512;
    gemm4_mfma_waves<true>(
        a.out, 2 * nsup, u0, rows, nullptr, Bs,
        [&](int m, int live, float (&v0)[4], float (&v1)[4], int ln, uint32_t) __attribute__((always_inline)) {
            const size_t row = (size_t)mt * a.tile_rows + m, col = (size_t)ib * 128 + ln;
            if (a.splits > 1) {  // the raw products, for grad_finish_kernel
                float *plane = a.part + ((size_t)sp * a.rows + row) * a.in + col;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (i < live) {
                        plane[(size_t)i * a.in] = v0[i];
                        plane[(size_t)i * a.in + 64] = v1[i];
                    }
                return;
            }
            // (the scales are fetched here: held through the main loop they would not fit its registers)
            const float s0 = h2f(a.suh[col]) * (codebook_scale<FAM>() * HAD_SCALE);
            const float s1 = h2f(a.suh[col + 64]) * (codebook_scale<FAM>() * HAD_SCALE);
            fwht128_wave_rows<4>(v0, v1, ln);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < live) {
                    const float inv = a.inv_scale[row + i];
                    store_y4(a.dx, a.dx_dtype, (row + i) * a.in + col, v0[i] * s0 * inv, v1[i] * s1 * inv);
                }
        });
}

// dx from the splits' raw products, in split order: a wave per (input block, row).  (The last split of a tile to arrive did
// this for its own rows at first: 0.9 us less for 1 row of 4096 x 4096, a launch being saved, and 0.5 to 1.3 us more for 5
// and 8 rows, the sums then being a few waves' instead of the whole GPU's.)
template <int FAM>
__global__ __launch_bounds__(256) void grad_finish_kernel(GradArgs a) {
    const int ib = blockIdx.x, row = blockIdx.y * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    const size_t col = (size_t)ib * 128 + lane;
    const float s0 = h2f(a.suh[col]), s1 = h2f(a.suh[col + 64]), inv = a.inv_scale[row];
    float v0, v1;
    sum_planes<false>(a.part + (size_t)row * a.in + (size_t)ib * 128, (size_t)a.rows * a.in, a.splits, lane, v0, v1);
    fwht128_wave(v0, v1, lane);
    const float sc = codebook_scale<FAM>() * HAD_SCALE;
    store_y4(a.dx, a.dx_dtype, (size_t)row * a.in + col, v0 * (s0 * sc) * inv, v1 * (s1 * sc) * inv);
}

template <int FAM, int N>
static hipError_t launch_grad(const GradArgs &a, hipStream_t s) {
    const unsigned wgs = (unsigned)(a.in / 128) * (unsigned)((a.rows + a.tile_rows - 1) / a.tile_rows) * (unsigned)a.splits;
    hipLaunchKernelGGL((grad_gemm_kernel<FAM, N>), dim3(wgs), dim3(G4_THREADS), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL(grad_finish_kernel<FAM>, dim3((unsigned)(a.in / 128), (unsigned)((a.rows + 3) / 4)), dim3(256), 0, s,
                       a);
    return hipGetLastError();
}

template <int FAM>
static hipError_t launch_grad_fam(const GradArgs &a, hipStream_t s) {
    switch (a.n) {
    case 16: return launch_grad<FAM, 16>(a, s);
    case 24: return launch_grad<FAM, 24>(a, s);
    case 32: return launch_grad<FAM, 32>(a, s);
    case 40: return launch_grad<FAM, 40>(a, s);
    case 48: return launch_grad<FAM, 48>(a, s);
    case 64: return launch_grad<FAM, 64>(a, s);
    default: break;
    }
    if constexpr (FAM != FAM_PAIR) {  // PAIR1 has no rows there
        switch (a.n) {
        case 80: return launch_grad<FAM, 80>(a, s);
        case 96: return launch_grad<FAM, 96>(a, s);
        case 112: return launch_grad<FAM, 112>(a, s);
        case 128: return launch_grad<FAM, 128>(a, s);
        default: break;
        }
    }
    return launch_grad<FAM, 0>(a, s);
}

template <int DT>
static hipError_t launch_grad_prepare(const GradArgs &a, hipStream_t s) {
    const int tiles = ((a.rows + 15) / 16 + a.prep_tiles - 1) / a.prep_tiles;
    const dim3 grid((unsigned)(a.out / 128), (unsigned)tiles);
    if (a.act == ACT_NONE) hipLaunchKernelGGL((grad_scan_kernel<DT, false>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((grad_scan_kernel<DT, true>), dim3((unsigned)a.rows), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((grad_prepare_kernel<DT>), grid, dim3(256), 0, s, a);
    e = hipGetLastError();
    if (e != hipSuccess || !a.dbias || !a.dbias_part) return e;
    hipLaunchKernelGGL(grad_dbias_kernel, dim3((unsigned)(a.out / 64)), dim3(256), 0, s, a, tiles);
    return hipGetLastError();
}

hipError_t run_gradient(int fam, const GradArgs &a, hipStream_t s) {
    const hipError_t e = a.dtype == DT_F16    ? launch_grad_prepare<DT_F16>(a, s)
                         : a.dtype == DT_BF16 ? launch_grad_prepare<DT_BF16>(a, s)
                                              : launch_grad_prepare<DT_F32>(a, s);
    if (e != hipSuccess) return e;
    switch (fam) {
    case FAM_MCG: return launch_grad_fam<FAM_MCG>(a, s);
    case FAM_MUL1: return launch_grad_fam<FAM_MUL1>(a, s);
    case FAM_HASH: return launch_grad_fam<FAM_HASH>(a, s);
    case FAM_PAIR: return launch_grad_fam<FAM_PAIR>(a, s);
    default: return launch_grad_fam<FAM_3INST>(a, s);
    }
}

}  // namespace exl3
