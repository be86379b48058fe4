// The backward pass of a linear with an epilogue over a frozen trellis bank: with z = project(x) + bias and
// y = act(z) + residual,
//   dz = dy * act'(z),  dbias = sum over rows of dz,  dx = H(u W^T) * suh,  u = f16(H(dz * svh))
// (H: the orthonormal Hadamard transform of every 128; residual's gradient is dy itself).  u is rounded to f16 as the
// forward's prepared input is, under a power of two per row that brings the row's largest |dz * svh| to 2^10 .. 2^11:
// gradients lie far below f16's normal range, and |H v| <= sqrt(128) max |v| keeps the scaled values below 2^15.
//
//   grad_scan_kernel     reads dy and pre once: the rows' largest values by column chunk, dbias's partial sums
//   grad_prepare_kernel  reads them again: u in MFMA A-fragment order, each row's scale
//   grad_gemm_kernel     u W^T on the decode-wave tile (exl3_gemm_tile.h), the trellis decoded once per 256 rows into the
//                        same column-major slab as the forward's and read back transposed by the MFMA waves; with few
//                        row and column tiles the contraction is split and grad_finish_kernel sums the splits in order
#include "exl3_gemm_tile.h"
#include "exl3_epilogue.h"

namespace exl3 {

constexpr int GS_COLS = GRAD_SCAN_COLS;  // 64 lanes x 8

// Eight consecutive values of a row (16-byte loads; the host checks the alignment).
template <int DT>
__device__ __forceinline__ void load8(const void *p, size_t i, float (&v)[8]) {
    if constexpr (DT == DT_F32) {
        const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
        const float4 b = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const uint32_t h = q & 1 ? w[q >> 1] >> 16 : w[q >> 1] & 0xFFFFu;
            v[q] = DT == DT_F16 ? h2f((uint16_t)h) : __uint_as_float(h << 16);
        }
    }
}

__device__ __forceinline__ float wave_max_abs(float v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

// Workgroup (column chunk, row tile of a.tile_rows rows): wave w takes the tile's rows w, w + 4, ..., lane l the chunk's
// columns 8 l .. 8 l + 7.  amax[row][chunk] = max |dz * svh|; dbias_part[tile][col] = sum of dz (one tile: dbias itself).
template <int DT>
__global__ __launch_bounds__(256) void grad_scan_kernel(GradArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * GS_COLS + lane * 8;
    const bool in = col < a.out;  // out is a multiple of 128, so a lane's eight columns are all in or all out
    const int c0 = in ? col : 0;
    float sv[8], sum[8] = {};
#pragma unroll
    for (int q = 0; q < 8; q++) sv[q] = in ? h2f(a.svh[c0 + q]) : 0.f;
    const int r0 = blockIdx.y * a.tile_rows, r1 = min(r0 + a.tile_rows, a.rows);
    for (int r = r0 + wave; r < r1; r += 4) {
        float d[8];
        load8<DT>(a.dy, (size_t)r * a.out + c0, d);
        if (a.act != ACT_NONE) {
            float z[8];
            load8<DT>(a.pre, (size_t)r * a.out + c0, z);
#pragma unroll
            for (int q = 0; q < 8; q++) d[q] *= act_slope(a.act, z[q]);
        }
        float m = 0.f;
#pragma unroll
        for (int q = 0; q < 8; q++) {
            m = fmaxf(m, fabsf(d[q] * sv[q]));  // columns past the end have sv = 0
            sum[q] += d[q];
        }
        m = wave_max_abs(m);
        if (lane == 0) a.amax[(size_t)r * a.chunks + blockIdx.x] = m;
    }
    if (!a.dbias) return;
    __shared__ float part[4][GS_COLS];
#pragma unroll
    for (int q = 0; q < 8; q++) part[wave][lane * 8 + q] = sum[q];
    __syncthreads();
    float *dst = gridDim.y == 1 ? a.dbias : a.dbias_part + (size_t)blockIdx.y * a.out;
    for (int i = threadIdx.x; i < GS_COLS; i += 256) {
        const int cc = blockIdx.x * GS_COLS + i;
        if (cc < a.out) dst[cc] = (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]);
    }
}

// dbias from the row tiles' sums, in tile order.
__global__ __launch_bounds__(256) void grad_dbias_kernel(GradArgs a, int tiles) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.out) return;
    float s = 0.f;
    for (int t = 0; t < tiles; t++) s += a.dbias_part[(size_t)t * a.out + c];
    a.dbias[c] = s;
}

// The power of two that brings m to 2^10 .. 2^11 (1 for zero and non-finite rows), and its inverse, both normal floats.
__device__ __forceinline__ int grad_exponent(float m) {
    if (!(m > 0.f) || m > 3.4028235e38f) return 0;
    const int e = (int)(__float_as_uint(m) >> 23) - 127;  // subnormals: -127, and the clamp below
    return min(max(10 - e, -126), 126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// u in A-fragment order (gemm_prepare_frag_kernel's), 16 rows x one 128-block of the gradient a workgroup: wave w takes
// rows 4 w .. 4 w + 3.  Rows past the end are zeros.  inv_scale[row] is written by the workgroups of block 0.
template <int DT>
__global__ __launch_bounds__(256) void grad_prepare_kernel(GradArgs a) {
    const int b = blockIdx.x, rt = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ __align__(16) uint16_t t[16][128 + 8];
    __shared__ int ex[16];
    const int m0 = rt * 16 + wave * 4;
    const size_t col = (size_t)b * 128 + lane;
    float v0[4], v1[4], z0[4], z1[4];
    const float s0 = h2f(a.svh[col]), s1 = h2f(a.svh[col + 64]);
#pragma unroll
    for (int rr = 0; rr < 4; rr++) {
        const size_t i = (size_t)min(m0 + rr, a.rows - 1) * a.out + col;
        v0[rr] = load_act<DT>(a.dy, i);
        v1[rr] = load_act<DT>(a.dy, i + 64);
    }
    if (a.act != ACT_NONE) {
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const size_t i = (size_t)min(m0 + rr, a.rows - 1) * a.out + col;
            z0[rr] = load_act<DT>(a.pre, i);
            z1[rr] = load_act<DT>(a.pre, i + 64);
        }
    }
    // the row's largest value over its chunks: 16 lanes a row
    {
        const int row = min(rt * 16 + (tid >> 4), a.rows - 1);
        float m = 0.f;
        for (int q = tid & 15; q < a.chunks; q += 16) m = fmaxf(m, a.amax[(size_t)row * a.chunks + q]);
#pragma unroll
        for (int k = 8; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
        if ((tid & 15) == 0) {
            const int e = grad_exponent(m);
            ex[tid >> 4] = e;
            if (b == 0 && rt * 16 + (tid >> 4) < a.rows) a.inv_scale[rt * 16 + (tid >> 4)] = pow2(-e);
        }
    }
    __syncthreads();
#pragma unroll
    for (int rr = 0; rr < 4; rr++) {
        if (a.act != ACT_NONE) {
            v0[rr] *= act_slope(a.act, z0[rr]);
            v1[rr] *= act_slope(a.act, z1[rr]);
        }
        const bool live = m0 + rr < a.rows;
        v0[rr] = live ? v0[rr] * s0 : 0.f;
        v1[rr] = live ? v1[rr] * s1 : 0.f;
    }
    fwht128_wave_rows_relaid<4>(v0, v1, lane);
    const float sc = fwht_relaid_sign(lane) * HAD_SCALE;
    const int c0 = fwht_relaid_col(lane, 0), c1 = fwht_relaid_col(lane, 1);
#pragma unroll
    for (int rr = 0; rr < 4; rr++) {
        const int r = wave * 4 + rr;
        const float two = pow2(ex[r]);
        t[r][c0] = __half_as_ushort(__float2half_rn(v0[rr] * sc * two));
        t[r][c1] = __half_as_ushort(__float2half_rn(v1[rr] * sc * two));
    }
    __syncthreads();
    const int kq = tid >> 6, c = lane & 15, h = lane >> 4;  // 32-k block kq of the 128-block, fragment lane (c, h)
    const uint4 v = *reinterpret_cast<const uint4 *>(&t[c][kq * 32 + 8 * h]);
    *reinterpret_cast<uint4 *>(a.u + ((size_t)rt * (a.out / 32) + (size_t)b * 4 + kq) * 512 + (size_t)lane * 8) = v;
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

// Workgroup: a 256-row x 128-column tile of dx (one input block ib) over the output groups of one split.
template <int FAM, int N>
__global__ __launch_bounds__(G4_THREADS) void grad_gemm_kernel(GradArgs a) {
    const int nib = a.in / 128, nm = (a.rows + G2_MT - 1) / G2_MT, nog = a.out / 128;
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
    const int rows = min(G2_MT, a.rows - mt * G2_MT);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int d = gemm4_decoder(wave, rows);
    if (d >= 0) {
        gemm4_decode_role<FAM>(rows <= G4_HELP_ROWS, d, nsup, lane, Bs, [&](int r, int rs, int loads) {
            return GradReader<FAM, N>(a.trellis, ib, r, rs, a.out >> 4, g0, loads, a.n, lane, a.k);
        });
        return;
    }
    const uint16_t *u0 = a.u + (size_t)mt * (G2_MT / 16) * (size_t)(a.out / 32) * 512 + (size_t)g0 * 4 * 512;
    gemm4_mfma_waves<true>(
        a.out, 2 * nsup, u0, rows, nullptr, Bs,
        [&](int m, int live, float (&v0)[4], float (&v1)[4], int ln, uint32_t) __attribute__((always_inline)) {
            const size_t row = (size_t)mt * G2_MT + m, col = (size_t)ib * 128 + ln;
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

// dx from the splits' raw products, in split order: a wave per (input block, row).
template <int FAM>
__global__ __launch_bounds__(256) void grad_finish_kernel(GradArgs a) {
    const int lane = threadIdx.x & 63, row = blockIdx.y * 4 + (int)(threadIdx.x >> 6);
    if (row >= a.rows) return;
    const size_t col = (size_t)blockIdx.x * 128 + lane;
    const float s0 = h2f(a.suh[col]), s1 = h2f(a.suh[col + 64]), inv = a.inv_scale[row];
    float v0, v1;
    sum_planes<false>(a.part + (size_t)row * a.in + (size_t)blockIdx.x * 128, (size_t)a.rows * a.in, a.splits, lane, v0, v1);
    fwht128_wave(v0, v1, lane);
    const float sc = codebook_scale<FAM>() * HAD_SCALE;
    store_y4(a.dx, a.dx_dtype, (size_t)row * a.in + col, v0 * (s0 * sc) * inv, v1 * (s1 * sc) * inv);
}

hipError_t run_grad_scan(const GradArgs &a, hipStream_t s) {
    const int tiles = (a.rows + a.tile_rows - 1) / a.tile_rows;
    const dim3 grid((unsigned)a.chunks, (unsigned)tiles);
    if (a.dtype == DT_F16) hipLaunchKernelGGL(grad_scan_kernel<DT_F16>, grid, dim3(256), 0, s, a);
    else if (a.dtype == DT_BF16) hipLaunchKernelGGL(grad_scan_kernel<DT_BF16>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(grad_scan_kernel<DT_F32>, grid, dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.dbias || tiles == 1) return e;
    hipLaunchKernelGGL(grad_dbias_kernel, dim3((unsigned)((a.out + 255) / 256)), dim3(256), 0, s, a, tiles);
    return hipGetLastError();
}

template <int FAM, int N>
static hipError_t launch_grad(const GradArgs &a, hipStream_t s) {
    const unsigned wgs = (unsigned)(a.in / 128) * (unsigned)((a.rows + G2_MT - 1) / G2_MT) * (unsigned)a.splits;
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

hipError_t run_grad_gemm(int fam, const GradArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)(a.out / 128), (unsigned)((a.rows + 15) / 16));
    if (a.dtype == DT_F16) hipLaunchKernelGGL(grad_prepare_kernel<DT_F16>, grid, dim3(256), 0, s, a);
    else if (a.dtype == DT_BF16) hipLaunchKernelGGL(grad_prepare_kernel<DT_BF16>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(grad_prepare_kernel<DT_F32>, grid, dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
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
