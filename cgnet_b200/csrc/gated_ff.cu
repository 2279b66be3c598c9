// Gated feed-forward block: both projections, the activation and the product in one kernel, and its backward pass.
//
//     g = x Wg^T,  u = x Wu^T,  h = act(g) * u                       x (rows, dim), Wg and Wu (hidden, dim), h (rows, hidden)
//     dg = dh * u * act'(g),  du = dh * act(g)
//     dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// A forward whose backward follows leaves g and u in float32: kept in 16 bits their rounding alone would add as much error to
// every gradient as the gradient's own rounding.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "ff_gemm.cuh"

namespace cgb200 {

struct FfArgs {
    const void *x, *wg, *wu;
    int64_t x_stride, wg_stride, wu_stride;    // values between rows
    int64_t rows;
    int dim, hidden, act;
    void* h;                                   // forward
    float* gu;                                 // [2][rows][gu_pitch]: g, u; null where no backward follows
    int64_t gu_pitch;                          // hidden rounded up to whole 16 bytes
    const void* dh;                            // backward
    int64_t dh_stride;
    void *dx, *dwg, *dwu;                      // each may be null
};

// ---- a few rows: one warp per hidden unit, bound by reading the weights ------------------------------------------------
constexpr int kFfFewRows = 4;

// Four chunks of either weight row are on their way at a time; tensor cores would have 1 row of 128 to work on.  1 x 4096 -> 8192
// bf16 (134 MB of weights) 23.8 us = 5.6 TB/s; 4 rows a quarter more.  EDGE: rows that do not start or end on 16-byte boundaries.
template <typename T, int M, bool EDGE>
__global__ void __launch_bounds__(128) ff_few_rows_kernel(FfArgs a) {
    constexpr int N = Chunk<T>::N, U = 4;
    const int lane = threadIdx.x & 31;
    const int64_t j = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (j >= a.hidden) return;
    const T* wg = (const T*)a.wg + j * a.wg_stride;
    const T* wu = (const T*)a.wu + j * a.wu_stride;
    const int pg = EDGE ? row_phase(wg) : 0, pu = EDGE ? row_phase(wu) : 0;
    float g[M], u[M];
#pragma unroll
    for (int m = 0; m < M; ++m) g[m] = u[m] = 0.f;
    auto multiply = [&](const uint4& rg, const uint4& ru, int k, bool inside) {
        float vg[N], vu[N];
        unpack16(rg, vg, (const T*)nullptr);
        unpack16(ru, vu, (const T*)nullptr);
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const T* x = (const T*)a.x + m * a.x_stride;
            float vx[N];
            const uint4 rx = !EDGE ? *reinterpret_cast<const uint4*>(x + k * N) : inside ? load_inside(x, row_phase(x), k) : load_at(x, row_phase(x), k, a.dim);
            unpack16(rx, vx, (const T*)nullptr);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                g[m] = fmaf(vg[i], vx[i], g[m]);
                u[m] = fmaf(vu[i], vx[i], u[m]);
            }
        }
    };
    const int chunks = (a.dim + N - 1) / N;
    int k = lane;
    if (!EDGE) {
        for (; k + (U - 1) * 32 < chunks; k += U * 32) {
            uint4 rg[U], ru[U];
#pragma unroll
            for (int c = 0; c < U; ++c) {
                rg[c] = __ldcs(reinterpret_cast<const uint4*>(wg) + k + c * 32);
                ru[c] = __ldcs(reinterpret_cast<const uint4*>(wu) + k + c * 32);
            }
#pragma unroll
            for (int c = 0; c < U; ++c) multiply(rg[c], ru[c], k + c * 32, true);
        }
    } else {
        // behind the first 32 chunks, and with a whole group behind the last of a step, no group leaves the row
        if (k < chunks) multiply(load_at(wg, pg, k, a.dim), load_at(wu, pu, k, a.dim), k, false);
        for (k += 32; (k - lane + 2 * 32 + 1) * N <= a.dim; k += 2 * 32) {
            uint4 rg[2], ru[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) rg[c] = load_inside(wg, pg, k + c * 32), ru[c] = load_inside(wu, pu, k + c * 32);
#pragma unroll
            for (int c = 0; c < 2; ++c) multiply(rg[c], ru[c], k + c * 32, true);
        }
    }
    for (; k < chunks; k += 32) multiply(load_at(wg, pg, k, a.dim), load_at(wu, pu, k, a.dim), k, false);
#pragma unroll
    for (int m = 0; m < M; ++m) {
        g[m] = warp_sum(g[m]);
        u[m] = warp_sum(u[m]);
        if (lane == 0) {
            ((T*)a.h)[m * (int64_t)a.hidden + j] = from_f32<T>(activate<false>(a.act, g[m]).x * u[m]);
            if (a.gu != nullptr) {
                a.gu[m * a.gu_pitch + j] = g[m];
                a.gu[(a.rows + m) * a.gu_pitch + j] = u[m];
            }
        }
    }
}

// ---- CUDA-core tiles: small products, where the time is one chain of loads ----------------------------------------------
// A block has 32 x 32 outputs.  Its warps share the contraction: each takes a part of it, in slabs of eight terms that it fetches while it
// multiplies the slab before and keeps in shared memory of its own, so no barrier stands between them; their sums are added in a fixed
// order at the end, by all threads.  Lane (ly, lx) has outputs 8 ly .. 8 ly + 7 x 4 lx .. 4 lx + 3 of its warp's sums.  Operands
// of any alignment.  The code is kept short: run once by a few blocks, it is bound by fetching its instructions (unrolled
// to 16 terms, with the results written by one warp, 52 -> 256 at 100 rows took 12 + 38 us; now 10 + 23 between events).
constexpr int kFfTile = 32, kFfSlab = 8, kFfPitch = kFfTile + 4, kFfFwdWarps = 8, kFfBwdWarps = 16;
constexpr int kFfSumPitch = kFfTile + 1, kFfSums = kFfFwdWarps * kFfTile * kFfSumPitch;      // floats of eight warps' sums

// acc += slab
__device__ __forceinline__ void ff_slab(const float (*a)[kFfPitch], const float (*b)[kFfPitch], int ly, int lx, float (&acc)[8][4]) {
#pragma unroll 4
    for (int k = 0; k < kFfSlab; ++k) {
        const float4 a0 = *(const float4*)&a[k][ly * 8], a1 = *(const float4*)&a[k][ly * 8 + 4], b0 = *(const float4*)&b[k][lx * 4];
        const float av[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w}, bv[4] = {b0.x, b0.y, b0.z, b0.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
    }
}
__device__ __forceinline__ void ff_leave(const float (&acc)[8][4], float* buf, int slot, int ly, int lx) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) buf[(slot * kFfTile + ly * 8 + i) * kFfSumPitch + lx * 4 + j] = acc[i][j];
}
// Sum of eight warps' values of output (row, col)
__device__ __forceinline__ float ff_sum(const float* buf, int row, int col) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += buf[(w * kFfTile + row) * kFfSumPitch + col];
    return s;
}

template <typename T>
__global__ void __launch_bounds__(kFfFwdWarps * 32) ff_tile_fwd_kernel(FfArgs a) {
    __shared__ __align__(16) float sums[kFfSums];                         // the slabs lie in the same memory
    static_assert(kFfSums >= kFfFwdWarps * 3 * kFfSlab * kFfPitch, "the slabs must fit");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ly = lane >> 3, lx = lane & 7;
    float (*sm)[kFfSlab][kFfPitch] = (float (*)[kFfSlab][kFfPitch])(sums + warp * 3 * kFfSlab * kFfPitch);
    const int64_t m0 = (int64_t)blockIdx.x * kFfTile;
    const int j0 = blockIdx.y * kFfTile;
    const int per = (a.dim + kFfFwdWarps - 1) / kFfFwdWarps, k_lo = warp * per, k_hi = min(a.dim, k_lo + per);
    const int lk = lane & 7, li = lane >> 3;          // 8 terms x 4 rows a load
    const T* px = (const T*)a.x + (m0 + li) * a.x_stride + lk;
    const T* pg = (const T*)a.wg + (int64_t)(j0 + li) * a.wg_stride + lk;
    const T* pu = (const T*)a.wu + (int64_t)(j0 + li) * a.wu_stride + lk;
    float x[8], wg[8], wu[8];
    auto fetch = [&](int k0) {
        const bool in = k0 + lk < k_hi;
        const int nx = in ? (int)min((int64_t)kFfTile, a.rows - m0) : 0, nj = in ? min(kFfTile, a.hidden - j0) : 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int i = li + 4 * r;
            x[r] = i < nx ? to_f32(px[4 * r * a.x_stride + k0]) : 0.f;
            wg[r] = i < nj ? to_f32(pg[4 * r * a.wg_stride + k0]) : 0.f;
            wu[r] = i < nj ? to_f32(pu[4 * r * a.wu_stride + k0]) : 0.f;
        }
    };
    float g[8][4] = {}, u[8][4] = {};
    fetch(k_lo);
    for (int k0 = k_lo; k0 < k_hi; k0 += kFfSlab) {
        __syncwarp();
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int i = li + 4 * r;
            sm[0][lk][i] = x[r], sm[1][lk][i] = wg[r], sm[2][lk][i] = wu[r];
        }
        __syncwarp();
        if (k0 + kFfSlab < k_hi) fetch(k0 + kFfSlab);
        ff_slab(sm[0], sm[1], ly, lx, g);
        ff_slab(sm[0], sm[2], ly, lx, u);
    }
    // row `warp` + 8 i and column `lane` of the tile, i = 0 .. 3
    float gs[4];
    __syncthreads();
    ff_leave(g, sums, warp, ly, lx);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) gs[i] = ff_sum(sums, warp + 8 * i, lane);
    __syncthreads();
    ff_leave(u, sums, warp, ly, lx);
    __syncthreads();
    const int c = j0 + lane;
    if (c >= a.hidden) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + warp + 8 * i, at = m * a.hidden + c;
        if (m >= a.rows) break;
        const float us = ff_sum(sums, warp + 8 * i, lane);
        ((T*)a.h)[at] = from_f32<T>(activate_shared(a.act, gs[i]).x * us);
        if (a.gu != nullptr) a.gu[m * a.gu_pitch + c] = gs[i], a.gu[(a.rows + m) * a.gu_pitch + c] = us;
    }
}

// One launch for all gradients: the first `nx` blocks hold tiles of dx, the others tiles of [dWg; dWu].
template <typename T>
__global__ void __launch_bounds__(kFfBwdWarps * 32) ff_tile_bwd_kernel(FfArgs a, int nx, int tiles_d) {
    __shared__ __align__(16) float sums[kFfBwdWarps * 2 * kFfSlab * kFfPitch];       // slabs, then the sums of half of the warps
    static_assert(sizeof(sums) >= kFfSums * sizeof(float), "the sums must fit");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ly = lane >> 3, lx = lane & 7;
    float (*sm)[kFfSlab][kFfPitch] = (float (*)[kFfSlab][kFfPitch])(sums + warp * 2 * kFfSlab * kFfPitch);
    const bool dx = (int)blockIdx.x < nx;
    const int tile = dx ? blockIdx.x : blockIdx.x - nx;
    const int64_t i0 = (int64_t)(tile / tiles_d) * kFfTile;      // row of the output: sample, or hidden unit (g, then u)
    const int d0 = (tile % tiles_d) * kFfTile;
    const int64_t n_i = dx ? a.rows : 2 * (int64_t)a.hidden, n_k = dx ? 2 * (int64_t)a.hidden : a.rows;
    const int64_t per = (n_k + kFfBwdWarps - 1) / kFfBwdWarps, k_lo = warp * per, k_hi = min(n_k, k_lo + per);
    // dx reads dgu along its rows (8 terms x 4 rows a load), dW down its columns: neighbouring lanes take neighbouring addresses
    const int la = dx ? lane >> 3 : 0, step = dx ? 4 : 1;
    float gv[8], uv[8], dv[8], bv[8];
    bool up = false;
    auto fetch = [&](int64_t k0) {
        const int64_t unit = dx ? k0 + (lane & 7) : i0 + lane, row = dx ? i0 + la : k0;      // of dgu
        up = unit >= a.hidden;
        const int64_t j = up ? unit - a.hidden : unit;
        const int n = (int)min((int64_t)kFfTile, dx ? (unit < k_hi ? n_i - row : 0) : (unit < n_i ? k_hi - row : 0));
        const float* g = a.gu + row * a.gu_pitch + j;
        const float* u = g + a.rows * a.gu_pitch;
        const T* h = (const T*)a.dh + row * a.dh_stride + j;
        const int nb = d0 + lane < a.dim ? (int)min((int64_t)kFfSlab, k_hi - k0) : 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int q = step * r;
            const bool in = q < n;
            gv[r] = in ? g[q * a.gu_pitch] : 0.f;
            uv[r] = in && !up ? u[q * a.gu_pitch] : 1.f;
            dv[r] = in ? to_f32(h[q * a.dh_stride]) : 0.f;
            const int64_t k = k0 + r;
            const T* b = !dx ? (const T*)a.x + k * a.x_stride : k < a.hidden ? (const T*)a.wg + k * a.wg_stride : (const T*)a.wu + (k - a.hidden) * a.wu_stride;
            bv[r] = r < nb ? to_f32(b[d0 + lane]) : 0.f;
        }
    };
    float acc[8][4] = {};
    fetch(k_lo);
    for (int64_t k0 = k_lo; k0 < k_hi; k0 += kFfSlab) {
        __syncwarp();
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const float2 f = activate_shared(a.act, gv[r]);
            float* s = dx ? &sm[0][lane & 7][la + 4 * r] : &sm[0][r][lane];
            *s = dv[r] * (up ? f.x : uv[r] * f.y);
            sm[1][r][lane] = bv[r];
        }
        __syncwarp();
        if (k0 + kFfSlab < k_hi) fetch(k0 + kFfSlab);
        ff_slab(sm[0], sm[1], ly, lx, acc);
    }
    // the upper half of the warps hands its sums to the lower half, which then adds up as in the forward
    __syncthreads();
    if (warp >= 8) ff_leave(acc, sums, warp - 8, ly, lx);
    __syncthreads();
    if (warp < 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] += sums[(warp * kFfTile + ly * 8 + i) * kFfSumPitch + lx * 4 + j];
    }
    __syncthreads();
    if (warp < 8) ff_leave(acc, sums, warp, ly, lx);
    __syncthreads();
    const int d = d0 + lane;
    if (d >= a.dim) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t r = i0 + warp + 16 * i;
        if (r >= n_i) break;
        T* out = dx ? (T*)a.dx + r * a.dim : r < a.hidden ? (T*)a.dwg : (T*)a.dwu;
        if (out == nullptr) continue;
        if (!dx && r >= a.hidden) out += (r - a.hidden) * a.dim;
        else if (!dx) out += r * a.dim;
        out[d] = from_f32<T>(ff_sum(sums, warp + 16 * i, lane));
    }
}

// ---- operands of the tensor-core products ------------------------------------------------------------------------------
// The tiled copies want rows on 16-byte boundaries and 16-bit values.  A 16-bit matrix that lies so is read where it is; other
// ones are copied into the workspace first, float32 ones as three bfloat16 planes whose sum is the value.
struct FfPackOp {
    const void* src;
    int64_t stride, rows;
    int cols;
    void* dst;             // [planes][rows][pitch]
    int64_t pitch;
};
struct FfPackArgs {
    FfPackOp op[3];
};
__device__ __forceinline__ void split3(float x, float& hi, float& mid, float& lo) {
    hi = __bfloat162float(__float2bfloat16_rn(x));
    if (isinf(hi) && !isinf(x)) hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);       // the largest values: rounded towards 0
    const bool fine = fabsf(hi) < INFINITY;            // an infinity or NaN is its own first part
    const float r = x - hi;
    mid = fine ? __bfloat162float(__float2bfloat16_rn(r)) : 0.f;
    lo = fine ? r - mid : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_operand(T* dst, int64_t plane, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(dst) = pack16(v, (const T*)nullptr);
}
// float32: dst holds bfloat16 planes
template <>
__device__ __forceinline__ void store_operand<float>(float* dst, int64_t plane, const float (&v)[8]) {
    __nv_bfloat16* d = (__nv_bfloat16*)dst;
    float hi[8], mid[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) split3(v[i], hi[i], mid[i], lo[i]);
    *reinterpret_cast<uint4*>(d) = pack16(hi, (const __nv_bfloat16*)nullptr);
    *reinterpret_cast<uint4*>(d + plane) = pack16(mid, (const __nv_bfloat16*)nullptr);
    *reinterpret_cast<uint4*>(d + 2 * plane) = pack16(lo, (const __nv_bfloat16*)nullptr);
}
// 2-byte slot `i` of an operand buffer, as the pointer type store_operand takes
template <typename T>
__device__ __forceinline__ T* operand_at(void* dst, int64_t i) {
    return (T*)((uint16_t*)dst + i);
}

// Copies of operands that tiled bulk copies cannot read: rows that do not start on 16-byte boundaries, and float32 as three planes
// (bound by HBM: 4 bytes in, 6 out).
template <typename T>
__global__ void __launch_bounds__(256) ff_pack_kernel(FfPackArgs a) {
    const FfPackOp& o = a.op[blockIdx.y];
    const int64_t chunks = o.pitch / 8, n = o.rows * chunks;
    for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < n; c += (int64_t)gridDim.x * 256) {
        const int64_t r = c / chunks;
        const int e0 = (int)(c - r * chunks) * 8;
        float v[8];
        load_params<T, 8>((const T*)o.src + r * o.stride, e0, o.cols, v);
        store_operand<T>(operand_at<T>(o.dst, r * o.pitch + e0), o.rows * o.pitch, v);
    }
}

// dg and du, as operands of the products behind them, in the type of x (half precision: ff_range_kernel).  In bfloat16 that rounding adds
// as much error to the gradients as their own: 1.4 times the error of one rounding (relative, 8192 rows, 2048 -> 5120: 2.34e-3 against
// 1.66e-3); a second plane of each would double the products (456 us).  At the HBM roof: 8192 x 5120 bf16 (419 MB read, 132 written) 83 us.
template <typename T>
__global__ void __launch_bounds__(256) ff_dgu_kernel(FfArgs a, void* dg, void* du, int64_t pitch) {
    const int64_t chunks = pitch / 8, n = a.rows * chunks;
    const float* g = a.gu;
    const float* u = a.gu + a.rows * a.gu_pitch;
    for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < n; c += (int64_t)gridDim.x * 256) {
        const int64_t r = c / chunks;
        const int e0 = (int)(c - r * chunks) * 8;
        float gv[8], uv[8], dv[8];
        load_params<float, 8>(g + r * a.gu_pitch, e0, a.hidden, gv);
        load_params<float, 8>(u + r * a.gu_pitch, e0, a.hidden, uv);
        load_params<T, 8>((const T*)a.dh + r * a.dh_stride, e0, a.hidden, dv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = activate<true>(a.act, gv[i]);
            gv[i] = dv[i] * uv[i] * f.y;
            uv[i] = dv[i] * f.x;
        }
        store_operand<T>(operand_at<T>(dg, r * pitch + e0), a.rows * pitch, gv);
        store_operand<T>(operand_at<T>(du, r * pitch + e0), a.rows * pitch, uv);
    }
}

// Half precision's dg and du may leave its range, on either side, where the gradients behind them do not.  The largest finite value of
// each row and each hidden unit is found as they are written.  Where one is out of range (fits_half), its tile of 128 rows, for
// dx, or of 128 units, for the weights' gradients, is written once more, each row or unit scaled by a power of two of its own,
// which costs no digits; the products read that copy instead and their epilogue scales back.  (By rows and by units, because a factor
// may not change along a contraction, and so that a large row or unit costs no other one its small values.)
struct FfRange {
    uint32_t *rows, *cols;              // largest |dg|, |du| of a row, [rows]; of a unit, [2][pitch]; bits of a float32; null where not wanted
    uint32_t *row_flag, *col_flag;      // per tile, [row tiles], [2][unit tiles]
    int64_t pitch;
    int w, steps;                       // lanes side by side (a power of two from 2 to 32), rows of a thread in the first kernel
    __half *dg, *du;                    // [rows][pitch]
    __half *dg_rows, *du_rows, *dg_cols, *du_cols;
};
constexpr int kFfRangeSteps = 8;

// dg and du of eight units of a row
template <int ACT>
__device__ __forceinline__ void turn_gradients(float (&g)[8], float (&u)[8], const float (&dh)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = activate_as<ACT, true>(g[i]);
        g[i] = dh[i] * u[i] * f.y;
        u[i] = dh[i] * f.x;
    }
}
__device__ __forceinline__ void load_gradients(const FfArgs& a, int64_t r, int64_t e0, float (&dg)[8], float (&du)[8]) {
    float dh[8];
    load_params<float, 8>(a.gu + r * a.gu_pitch, e0, a.hidden, dg);
    load_params<float, 8>(a.gu + (a.rows + r) * a.gu_pitch, e0, a.hidden, du);
    load_params<__half, 8>((const __half*)a.dh + r * a.dh_stride, e0, a.hidden, dh);
    if (a.act == CGB200_ACT_RELU) turn_gradients<CGB200_ACT_RELU>(dg, du, dh);
    else if (a.act == CGB200_ACT_SILU) turn_gradients<CGB200_ACT_SILU>(dg, du, dh);
    else turn_gradients<CGB200_ACT_GELU>(dg, du, dh);
}
// A block has `w` lanes of eight units side by side and `steps` rows for each of the others: eight where the rows keep the SMs busy, so that
// few blocks meet at one unit's largest value, fewer where they do not (256 x 1024: 17 us with eight, 6 with one).
// 8192 x 5120 112 us (551 MB, 4.9 TB/s; 83 without the maxima); the kernel behind it 5 where nothing is out of range, 147 where everything is.
__global__ void __launch_bounds__(256, 4) ff_range_kernel(FfArgs a, FfRange q) {
    __shared__ uint32_t most[8 * 16 * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = q.w, at = (int)threadIdx.x & (w - 1);
    const int64_t e0 = ((int64_t)blockIdx.y * w + at) * 8, row0 = (int64_t)blockIdx.x * (256 / w) * q.steps + threadIdx.x / w;
    uint32_t top[16];           // of this thread's units
#pragma unroll
    for (int i = 0; i < 16; ++i) top[i] = 0;
#pragma unroll 2
    for (int s = 0; s < q.steps; ++s) {
        const int64_t r = row0 + (int64_t)s * (256 / w);
        uint32_t big = 0;
        if (r < a.rows && e0 < q.pitch) {
            float dg[8], du[8];
            load_gradients(a, r, e0, dg, du);
            *reinterpret_cast<uint4*>(q.dg + r * q.pitch + e0) = pack16(dg, (const __half*)nullptr);
            *reinterpret_cast<uint4*>(q.du + r * q.pitch + e0) = pack16(du, (const __half*)nullptr);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // an infinity or NaN spoils its own row and unit, but is no measure for them
                uint32_t bg = __float_as_uint(fabsf(dg[i])), bu = __float_as_uint(fabsf(du[i]));
                bg = bg < 0x7f800000u ? bg : 0u, bu = bu < 0x7f800000u ? bu : 0u;
                top[i] = max(top[i], bg), top[8 + i] = max(top[8 + i], bu);
                big = max(big, max(bg, bu));
            }
        }
        if (q.rows != nullptr) {
            if (w == 32) {
                big = __reduce_max_sync(0xffffffffu, big);
            } else {
                for (int o = w / 2; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
            }
            if (at == 0 && r < a.rows && big != 0) atomicMax(q.rows + r, big);
        }
    }
    if (q.cols == nullptr) return;
    // the rows of a warp, then its block's warps
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        for (int o = 16; o >= w; o >>= 1) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
        most[(warp * 16 + i) * 32 + lane] = top[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < w * 16; i += 256) {
        const int unit = i / 16, side = i % 16 / 8, j = i % 8;
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = max(m, most[(k * 16 + side * 8 + j) * 32 + unit]);
        const int64_t col = ((int64_t)blockIdx.y * w + unit) * 8 + j;
        if (m != 0 && col < q.pitch) atomicMax(q.cols + side * q.pitch + col, m);
    }
}
// The scaled copies of the tiles that need one, and the flags of all: a block has 128 rows and 8 w units, which are one or two tiles.
__global__ void __launch_bounds__(256) ff_rescale_kernel(FfArgs a, FfRange q) {
    __shared__ uint32_t flags;        // 1: the rows; 2, 4: the first and second tile of units in dg; 8, 16: in du
    const int w = q.w, at = (int)threadIdx.x & (w - 1), t = (int)threadIdx.x;
    const int64_t r0 = (int64_t)blockIdx.x * kFfBM, u0 = (int64_t)blockIdx.y * w * 8, e0 = u0 + at * 8;
    if (t == 0) flags = 0;
    __syncthreads();
    uint32_t mine = 0;
    if (q.rows != nullptr && t < kFfBM && r0 + t < a.rows && !fits_half(q.rows[r0 + t])) mine = 1;
    if (q.cols != nullptr && t < w * 8 && u0 + t < q.pitch) {
        if (!fits_half(q.cols[u0 + t])) mine |= 2u << (t / kFfBM);
        if (!fits_half(q.cols[q.pitch + u0 + t])) mine |= 8u << (t / kFfBM);
    }
    mine = __reduce_or_sync(0xffffffffu, mine);
    if ((t & 31) == 0 && mine != 0) atomicOr(&flags, mine);
    __syncthreads();
    mine = flags;
    if (t == 0 && blockIdx.y == 0 && q.rows != nullptr) q.row_flag[blockIdx.x] = mine & 1;
    const int64_t tiles = (q.pitch + kFfBM - 1) / kFfBM, tile = u0 / kFfBM + t / 2;
    if (t < 4 && blockIdx.x == 0 && q.cols != nullptr && tile < tiles) q.col_flag[t % 2 * tiles + tile] = mine >> (1 + t % 2 * 2 + t / 2) & 1;
    if (mine == 0 || e0 >= q.pitch) return;
    const bool by_rows = mine & 1, dg_cols = mine >> (1 + at * 8 / kFfBM) & 1, du_cols = mine >> (3 + at * 8 / kFfBM) & 1;
    if (!by_rows && !dg_cols && !du_cols) return;
    float sg[8], su[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sg[i] = dg_cols ? scale_of(q.cols[e0 + i]) : 1.f, su[i] = du_cols ? scale_of(q.cols[q.pitch + e0 + i]) : 1.f;
    for (int64_t r = r0 + t / w; r < min(a.rows, r0 + kFfBM); r += 256 / w) {
        float dg[8], du[8], x[8];
        load_gradients(a, r, e0, dg, du);
        const float sr = by_rows ? scale_of(q.rows[r]) : 1.f;
        auto leave = [&](__half* out, const float (&v)[8], const float* each) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = v[i] * (each != nullptr ? each[i] : sr);
            *reinterpret_cast<uint4*>(out + r * q.pitch + e0) = pack16(x, (const __half*)nullptr);
        };
        if (by_rows) leave(q.dg_rows, dg, nullptr), leave(q.du_rows, du, nullptr);
        if (dg_cols) leave(q.dg_cols, dg, sg);
        if (du_cols) leave(q.du_cols, du, su);
    }
}

// Parts of a split contraction (few tiles, long k: one tile's time would be the launch's), added in order: out[i] = sum over s of part[s][i].
struct FfReduceArgs {
    const float* part[2];
    int splits[2], sets[2];
    int64_t n[2];                 // values of a set
    void* out[2][2];
};
template <typename T>
__global__ void __launch_bounds__(256) ff_reduce_kernel(FfReduceArgs a) {
    const int p = blockIdx.y >> 1, set = blockIdx.y & 1;
    if (a.splits[p] <= 1 || set >= a.sets[p] || a.out[p][set] == nullptr) return;
    const float* src = a.part[p] + set * a.n[p];
    const int64_t step = a.sets[p] * a.n[p];
    T* out = (T*)a.out[p][set];
    const int splits = a.splits[p];
    const int64_t n = a.n[p];
    if (n % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {      // the parts start on 16-byte boundaries then
        for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
            float4 s = *(const float4*)(src + i);
#pragma unroll 4
            for (int k = 1; k < splits; ++k) {
                const float4 v = *(const float4*)(src + k * step + i);
                s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
            }
            T r[4] = {from_f32<T>(s.x), from_f32<T>(s.y), from_f32<T>(s.z), from_f32<T>(s.w)};
            if constexpr (sizeof(T) == 2) {
                uint2 u;
                memcpy(&u, r, 8);
                *(uint2*)(out + i) = u;
            } else {
                *(float4*)(out + i) = make_float4(r[0], r[1], r[2], r[3]);
            }
        }
        return;
    }
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = src[i];
#pragma unroll 4
        for (int k = 1; k < splits; ++k) s += src[k * step + i];
        out[i] = from_f32<T>(s);
    }
}

// The forward with a split contraction: the parts of g and u, added in order, and what is made of them.
template <typename T>
__global__ void __launch_bounds__(256) ff_join_kernel(FfArgs a, const float* g_part, const float* u_part, int splits) {
    const int64_t n = a.rows * a.hidden;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float g = g_part[i], u = u_part[i];
#pragma unroll 4
        for (int k = 1; k < splits; ++k) g += g_part[k * n + i], u += u_part[k * n + i];
        ((T*)a.h)[i] = from_f32<T>(activate<false>(a.act, g).x * u);
        if (a.gu != nullptr) {
            const int64_t m = i / a.hidden, j = i - m * a.hidden;
            a.gu[m * a.gu_pitch + j] = g;
            a.gu[(a.rows + m) * a.gu_pitch + j] = u;
        }
    }
}

// ---- which path, and what it needs -------------------------------------------------------------------------------------
// The tensor cores are used from this length of the longest contraction on (forward: dim; backward: rows or 2 hidden), or from this
// much work (rows x dim x hidden).  CUDA cores / tensor cores, us, launches of a graph: 16 bits, forward 16 x 64 -> 64 5.0 / 6.3,
// 16 x 128 -> 256 6.8 / 6.4, 10 x 976 -> 104 36 / 8.0; backward 7.0 / 7.2, 19 / 8.7, 11 / 7.8.  float32 (three planes, a copy in
// front), forward 100 x 256 -> 256 8.8 / 12.1, 100 x 512 -> 256 14.6 / 13.5, 32 x 640 -> 128 17.1 / 14.5; backward 16 / 19, 1000 x 48 -> 48 28 / 21.
struct FfLimits {
    int forward, backward;
    int64_t work;
};
static FfLimits ff_limits(int dtype) { return dtype == CGB200_F32 ? FfLimits{512, 640, 16 << 20} : FfLimits{128, 160, 8 << 20}; }

constexpr int kFfOutputStages = 8;
// Stages of 16-bit operands that one accumulator takes: the tensor core truncates each of its additions, four a stage, so a long sum of one
// sign comes out low, by 1.7e-4 after 512 stages, 8e-4 after 2048 (measured; half a step of bfloat16 is 3.9e-3, of float16 4.9e-4).
// Longer contractions go in parts that are added, rounded, in float32.  (float32 operands are flushed every kFfFlush stages.)
static int ff_longest(int dtype) { return dtype == CGB200_F32 ? 1 << 30 : dtype == CGB200_BF16 ? 512 : 256; }
// A forward whose tiles keep at most half of the SMs busy is split along dim from this many stages on.  Whole / split, us, launches of a
// graph: bf16 16 x 1024 -> 1000 9.1 / 8.0, 16 x 4096 -> 1000 19.3 / 9.7, 500 x 2048 -> 1000 13.3 / 13.1, 156 x 3330 -> 342 30.8 / 15.7;
// float32 300 x 640 -> 500 19.9 / 16.4, 156 x 3330 -> 342 78.8 / 22.5.
static int ff_split_stages(int dtype) { return dtype == CGB200_F32 ? 8 : 16; }

struct FfPlan {
    bool tensor;
    bool joined;                          // the forward's contraction is split: g and u are products of their own, joined afterwards
    int planes, bn;
    bool pack[3];                         // x, Wg, Wu
    int64_t pitch_d, pitch_h;             // of packed operands (dim columns) and of dg, du (hidden columns)
    int64_t off_pack[3], off_dg, off_du, off_rows, off_cols, off_amax, off_part[2], bytes;      // off_rows, off_cols: scaled copies of dg, du
    int64_t d_bytes;                      // of dg or du
    int n_problems;
    FfProblem problem[2];
};

static int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
static bool lies_aligned(const void* p, int64_t stride, int64_t rows, int cols) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows <= 1 ? true : stride >= cols && stride % 8 == 0 && rows * stride * 2 < (1ll << 39));
}

// `grads`: 0 for the forward, else the sum of 1 (dx), 2 (dWg), 4 (dWu).
static FfPlan ff_plan(const FfArgs& a, int dtype, int grads) {
    FfPlan q{};
    const bool fwd = grads == 0;
    const int64_t work = a.rows * a.dim * (int64_t)a.hidden;
    const FfLimits limit = ff_limits(dtype);
    const bool longer = fwd ? a.dim >= limit.forward : std::max<int64_t>(a.rows, 2 * (int64_t)a.hidden) >= limit.backward;
    q.tensor = a.rows > 0 && (longer || work >= limit.work) && !(fwd && a.rows <= kFfFewRows);
    if (!q.tensor) return q;
    q.planes = dtype == CGB200_F32 ? 3 : 1;
    const bool need[3] = {true, fwd || (grads & 1), fwd || (grads & 1)};
    const void* src[3] = {a.x, a.wg, a.wu};
    const int64_t stride[3] = {a.x_stride, a.wg_stride, a.wu_stride}, rows[3] = {a.rows, a.hidden, a.hidden};
    q.pitch_d = up(a.dim, 8), q.pitch_h = up(a.hidden, 8);
    int64_t at = 0;
    for (int i = 0; i < 3; ++i) {
        q.pack[i] = need[i] && (i > 0 || fwd || (grads & 6)) && (q.planes == 3 || !lies_aligned(src[i], stride[i], rows[i], a.dim));
        q.off_pack[i] = at;
        if (q.pack[i]) at += up(q.planes * rows[i] * q.pitch_d * 2, 256);
    }
    q.d_bytes = up(q.planes * a.rows * q.pitch_h * 2, 256);
    if (!fwd) q.off_dg = at, q.off_du = at + q.d_bytes, at += 2 * q.d_bytes;
    if (!fwd && dtype == CGB200_F16) {
        if (grads & 1) q.off_rows = at, at += 2 * q.d_bytes;
        if (grads & 6) q.off_cols = at, at += 2 * q.d_bytes;
        q.off_amax = at, at += up((a.rows + 2 * q.pitch_h + (a.rows + kFfBM - 1) / kFfBM + 2 * ((q.pitch_h + kFfBM - 1) / kFfBM)) * 4, 256);
    }
    const int64_t ti = (a.rows + kFfBM - 1) / kFfBM;
    const int hk = (a.hidden + kFfBK - 1) / kFfBK, dk = (a.dim + kFfBK - 1) / kFfBK;
    const int mk = (int)((a.rows + kFfBK - 1) / kFfBK), th = (a.hidden + kFfBM - 1) / kFfBM;
    const int w_sets = ((grads & 2) ? 1 : 0) + ((grads & 4) ? 1 : 0);
    auto units_at = [&](int bn) -> int64_t {
        if (fwd) return ti * ((a.hidden + bn / 2 - 1) / (bn / 2));
        const int64_t tj = (a.dim + bn - 1) / bn;
        return ((grads & 1) ? ti * tj : 0) + (int64_t)w_sets * th * tj;
    };
    // wide tiles move less through shared memory; narrow ones fill the SMs where the wide ones do not
    q.bn = q.planes == 3 || units_at(256) < kNumSM ? 128 : 256;
    const int longest = ff_longest(dtype);
    q.joined = fwd && ((2 * units_at(128) <= kNumSM && dk >= ff_split_stages(dtype)) || dk > longest);
    if (q.joined) {
        for (int i = 0; i < 2; ++i) {
            FfProblem& p = q.problem[q.n_problems++];
            p.a_map[0] = kMapX, p.b_map[0] = kMapWg + i;
            p.sources = 1, p.kblk = dk, p.sets = 1;
            p.tiles_i = (int)ti, p.tiles_j = (a.hidden + q.bn - 1) / q.bn;
            p.n_i = a.rows, p.n_j = a.hidden;
        }
    } else if (fwd) {
        FfProblem& p = q.problem[q.n_problems++];
        p.a_map[0] = kMapX, p.b_map[0] = kMapWg, p.b_map[1] = kMapWu;
        p.sources = 1, p.kblk = dk, p.sets = 1;
        p.tiles_i = (int)ti, p.tiles_j = (a.hidden + q.bn / 2 - 1) / (q.bn / 2);
        p.n_i = a.rows, p.n_j = a.hidden;
    }
    if (grads & 1) {
        FfProblem& p = q.problem[q.n_problems++];
        p.a_map[0] = kMapDg, p.a_map[1] = kMapDu, p.a_scaled[0] = kMapDgRows, p.a_scaled[1] = kMapDuRows, p.b_map[0] = kMapWg, p.b_map[1] = kMapWu, p.b_mn = 1;
        p.sources = 2, p.kblk = hk, p.sets = 1;
        p.tiles_i = (int)ti, p.tiles_j = (a.dim + q.bn - 1) / q.bn;
        p.n_i = a.rows, p.n_j = a.dim;
        p.out[0] = a.dx;
    }
    if (w_sets > 0) {
        FfProblem& p = q.problem[q.n_problems++];
        p.a_map[0] = (grads & 2) ? kMapDg : kMapDu, p.a_map[1] = kMapDu, p.b_map[0] = kMapX, p.a_mn = p.b_mn = 1;
        p.a_scaled[0] = (grads & 2) ? kMapDgCols : kMapDuCols, p.a_scaled[1] = kMapDuCols;
        p.sources = 1, p.kblk = mk, p.sets = w_sets;
        p.tiles_i = th, p.tiles_j = (a.dim + q.bn - 1) / q.bn;
        p.n_i = a.hidden, p.n_j = a.dim;
        p.out[0] = (grads & 2) ? a.dwg : a.dwu, p.out[1] = a.dwu;
    }
    // Units of very different length, or fewer than SMs: a long contraction goes in parts that are added in order afterwards.  A unit's
    // length is its stages and, for its output, about eight more; one much beyond an SM's share of all would be waited for.
    int64_t total = 0;
    for (int i = 0; i < q.n_problems; ++i) {
        const FfProblem& p = q.problem[i];
        total += (int64_t)p.sets * p.tiles_i * p.tiles_j * (p.sources * p.kblk + kFfOutputStages);
    }
    const double share = (double)total / kNumSM;
    for (int i = 0; i < q.n_problems; ++i) {
        FfProblem& p = q.problem[i];
        const int stages = p.sources * p.kblk, length = stages + kFfOutputStages;
        int splits = q.joined                          ? (int)std::max<int64_t>(2, kNumSM / (2 * ti * p.tiles_j))
                     : fwd || length <= 1.5 * share ? 1
                                                    : (int)std::min(8.0, length / std::max(0.5 * share, 2.0 * kFfOutputStages) + 0.999);
        splits = std::max(std::max(1, std::min(splits, stages / 4)), stages / longest + (stages % longest != 0));
        p.kper = (stages + splits - 1) / splits;
        p.splits = (stages + p.kper - 1) / p.kper;
    }
    if (q.n_problems == 2 && q.problem[1].kper > q.problem[0].kper) std::swap(q.problem[0], q.problem[1]);      // long units first
    int64_t unit = 0;
    for (int i = 0; i < q.n_problems; ++i) {
        FfProblem& p = q.problem[i];
        p.unit0 = (int)unit;
        unit += (int64_t)p.sets * p.tiles_i * p.tiles_j * p.splits;
        q.off_part[i] = at;
        if (p.splits > 1) at += up((int64_t)p.splits * p.sets * p.n_i * p.n_j * 4, 256);
    }
    q.bytes = at;
    return q;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
    static std::atomic<void*> fn{nullptr};
    void* f = fn.load();
    if (f == nullptr) {
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            return nullptr;
        fn.store(f);
    }
    return (EncodeTiled)f;
}
static bool encode(CUtensorMap* m, EncodeTiled enc, CUtensorMapDataType type, int size, const void* p, int64_t pitch, int64_t rows, int cols,
                   int planes, cuuint32_t box_cols, cuuint32_t box_rows, cuuint32_t box_planes, CUtensorMapSwizzle swizzle) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)(pitch * size), (cuuint64_t)((planes > 1 ? rows * pitch : pitch) * size)};
    const cuuint32_t box[3] = {box_cols, box_rows, box_planes}, step[3] = {1, 1, 1};
    return enc(m, type, 3, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// [planes][rows][pitch] of 16-bit values, read in boxes of 64 rows x 64 columns; what lies outside reads as zero
static bool ff_map(CUtensorMap* m, EncodeTiled enc, const void* p, int64_t pitch, int64_t rows, int cols, int planes, bool half) {
    return encode(m, enc, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p, pitch, rows, cols, planes, 64, 64, 1,
                  CU_TENSOR_MAP_SWIZZLE_128B);
}
// An output, written in boxes of 32 rows x 64 bytes; g and u together
template <typename T>
static bool ff_out_map(CUtensorMap* m, EncodeTiled enc, const void* p, int64_t pitch, int64_t rows, int cols, int planes) {
    const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : sizeof(T) == 2               ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    return encode(m, enc, type, (int)sizeof(T), p, pitch, rows, cols, planes, 64 / sizeof(T), 32, planes, CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int PLANES, int BN, typename T, bool FWD>
static int ff_gemm_launch(const FfGemmArgs& g, int kid, cudaStream_t st) {
    auto kern = ff_gemm_kernel<PLANES, BN, T, FWD>;
    CGB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFfSmem));
    launch_begin(kid, st);
    kern<<<(unsigned)std::min(g.units, kNumSM), kFfThreads, kFfSmem, st>>>(g);
    launch_end(kid, st);
    CGB_CUDA(cudaGetLastError());
    return CGB200_OK;
}

// The tensor-core path of the forward (grads = 0) and of the backward.
template <typename T>
static int ff_tensor(const FfArgs& a, const FfPlan& q, int grads, char* ws, cudaStream_t st) {
    constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
    const bool fwd = grads == 0;
    // a thread that has made no CUDA call yet (autograd's, in its first backward) has no context, and the driver refuses to encode
    int device;
    CGB_CUDA(cudaGetDevice(&device));
    CGB_CUDA(cudaSetDevice(device));
    EncodeTiled enc = encode_tiled();
    if (enc == nullptr) {
        set_error("the driver has no cuTensorMapEncodeTiled");
        return CGB200_ERR_CUDA;
    }
    const int kid = fwd ? K_FF_FWD : K_FF_BWD;
    const void* src[3] = {a.x, a.wg, a.wu};
    int64_t stride[3] = {a.x_stride, a.wg_stride, a.wu_stride};
    const int64_t rows[3] = {a.rows, a.hidden, a.hidden};
    FfPackArgs pack{};
    int n_pack = 0;
    int64_t most = 0;
    for (int i = 0; i < 3; ++i) {
        if (!q.pack[i]) {
            if (rows[i] == 1) stride[i] = up(a.dim, 8);       // one row: any distance to the next
            continue;
        }
        pack.op[n_pack++] = FfPackOp{src[i], stride[i], rows[i], a.dim, ws + q.off_pack[i], q.pitch_d};
        src[i] = ws + q.off_pack[i], stride[i] = q.pitch_d;
        most = std::max(most, rows[i] * q.pitch_d / 8);
    }
    if (n_pack > 0) {
        launch_begin(kid, st);
        ff_pack_kernel<T><<<dim3((unsigned)std::min<int64_t>((most + 255) / 256, kNumSM * 16), n_pack), 256, 0, st>>>(pack);
        launch_end(kid, st);
        CGB_CUDA(cudaGetLastError());
    }
    FfGemmArgs g{};
    bool ok = true;
    constexpr bool half = std::is_same<T, __half>::value;
    FfRange range{};
    for (int i = 0; i < 3; ++i) {
        const bool used = fwd || (i == 0 ? (grads & 6) != 0 : (grads & 1) != 0);
        if (used) ok = ok && ff_map(&g.map[kMapX + i], enc, src[i], stride[i], rows[i], a.dim, PLANES, half);
    }
    if (!fwd) {
        void *dg = ws + q.off_dg, *du = ws + q.off_du;
        if constexpr (half) {
            range.pitch = q.pitch_h, range.w = 2;
            range.dg = (__half*)dg, range.du = (__half*)du;
            uint32_t* words = (uint32_t*)(ws + q.off_amax);
            if (grads & 1) range.rows = words, range.dg_rows = (__half*)(ws + q.off_rows), range.du_rows = (__half*)(ws + q.off_rows + q.d_bytes);
            if (grads & 6) range.cols = words + a.rows, range.dg_cols = (__half*)(ws + q.off_cols), range.du_cols = (__half*)(ws + q.off_cols + q.d_bytes);
            words += a.rows + 2 * q.pitch_h;
            range.row_flag = words, range.col_flag = words + (a.rows + kFfBM - 1) / kFfBM;
            while (range.w < 32 && range.w < q.pitch_h / 8) range.w *= 2;
            const int64_t side = (q.pitch_h / 8 + range.w - 1) / range.w, one = (a.rows * range.w + 255) / 256;      // blocks; of one row a thread
            range.steps = (int)std::max<int64_t>(1, std::min<int64_t>(kFfRangeSteps, one * side / (kNumSM * 8)));
            CGB_CUDA(cudaMemsetAsync(ws + q.off_amax, 0, (a.rows + 2 * q.pitch_h) * 4, st));
            launch_begin(kid, st);
            ff_range_kernel<<<dim3((unsigned)((one + range.steps - 1) / range.steps), (unsigned)side), 256, 0, st>>>(a, range);
            launch_end(kid, st);
            CGB_CUDA(cudaGetLastError());
            launch_begin(kid, st);
            ff_rescale_kernel<<<dim3((unsigned)((a.rows + kFfBM - 1) / kFfBM), (unsigned)side), 256, 0, st>>>(a, range);
            launch_end(kid, st);
            CGB_CUDA(cudaGetLastError());
            void* copies[4] = {range.dg_rows, range.du_rows, range.dg_cols, range.du_cols};
            for (int i = 0; i < 4; ++i)
                if (copies[i] != nullptr) ok = ok && ff_map(&g.map[kMapDgRows + i], enc, copies[i], q.pitch_h, a.rows, a.hidden, PLANES, half);
        } else {
            launch_begin(kid, st);
            ff_dgu_kernel<T><<<(unsigned)std::min<int64_t>((a.rows * q.pitch_h / 8 + 255) / 256, kNumSM * 16), 256, 0, st>>>(a, dg, du, q.pitch_h);
            launch_end(kid, st);
            CGB_CUDA(cudaGetLastError());
        }
        ok = ok && ff_map(&g.map[kMapDg], enc, dg, q.pitch_h, a.rows, a.hidden, PLANES, half);
        ok = ok && ff_map(&g.map[kMapDu], enc, du, q.pitch_h, a.rows, a.hidden, PLANES, half);
    }
    if (!ok) {
        set_error("gated feed-forward: an operand's layout was refused by the driver");
        return CGB200_ERR_CUDA;
    }
    g.problems = q.n_problems;
    for (int i = 0; i < q.n_problems; ++i) {
        g.p[i] = q.problem[i];
        g.p[i].part = (float*)(ws + q.off_part[i]);
        g.units += g.p[i].sets * g.p[i].tiles_i * g.p[i].tiles_j * g.p[i].splits;
    }
    auto at16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    for (int i = 0; i < q.n_problems; ++i) {
        FfProblem& p = g.p[i];
        p.out_map[0] = p.out_map[1] = -1;
        if (q.joined) continue;               // parts only
        if (fwd) {
            p.out[0] = a.h;
            p.h_aligned = at16(a.h) && a.hidden % Chunk<T>::N == 0;
            if (a.gu != nullptr) {
                p.out_map[0] = kMapOut;
                ok = ok && ff_out_map<float>(&g.map[kMapOut], enc, a.gu, a.gu_pitch, a.rows, a.hidden, 2);
            }
            continue;
        }
        for (int k = 0; half && k < p.sets; ++k) {
            const bool du = p.a_map[k] == kMapDu;
            p.amax[k] = !p.a_mn ? range.rows : range.cols + (du ? q.pitch_h : 0);
            p.flag[k] = !p.a_mn ? range.row_flag : range.col_flag + (du ? (q.pitch_h + kFfBM - 1) / kFfBM : 0);
        }
        for (int k = 0; k < p.sets; ++k)
            if (p.splits == 1 && p.out[k] != nullptr && at16(p.out[k]) && a.dim % Chunk<T>::N == 0) {
                const int m = p.a_mn ? kMapOutWg + k : kMapOut;
                p.out_map[k] = m;
                ok = ok && ff_out_map<T>(&g.map[m], enc, p.out[k], a.dim, p.n_i, a.dim, 1);
            }
    }
    if (!ok) {
        set_error("gated feed-forward: an output's layout was refused by the driver");
        return CGB200_ERR_CUDA;
    }
    g.idesc_type = half ? 0u : (1u << 7) | (1u << 10);
    g.act = a.act, g.polls = kDefaultWaitPolls;
    const bool fused = fwd && !q.joined;
    int rc;
    if constexpr (PLANES == 3) rc = fused ? ff_gemm_launch<3, 128, T, true>(g, kid, st) : ff_gemm_launch<3, 128, T, false>(g, kid, st);
    else if (q.bn == 256) rc = fused ? ff_gemm_launch<1, 256, T, true>(g, kid, st) : ff_gemm_launch<1, 256, T, false>(g, kid, st);
    else rc = fused ? ff_gemm_launch<1, 128, T, true>(g, kid, st) : ff_gemm_launch<1, 128, T, false>(g, kid, st);
    if (rc != CGB200_OK) return rc;
    if (q.joined) {
        const int64_t n = a.rows * a.hidden;
        launch_begin(kid, st);
        ff_join_kernel<T><<<(unsigned)std::min<int64_t>((n + 255) / 256, kNumSM * 16), 256, 0, st>>>(a, g.p[0].part, g.p[1].part, g.p[0].splits);
        launch_end(kid, st);
        CGB_CUDA(cudaGetLastError());
        return CGB200_OK;
    }
    FfReduceArgs r{};
    bool any = false;
    int64_t n = 0;
    for (int i = 0; i < g.problems; ++i) {
        const FfProblem& p = g.p[i];
        r.part[i] = p.part, r.splits[i] = p.splits, r.sets[i] = p.sets, r.n[i] = p.n_i * p.n_j;
        r.out[i][0] = p.out[0], r.out[i][1] = p.out[1];
        if (p.splits > 1) any = true, n = std::max(n, r.n[i]);
    }
    if (any && !fwd) {
        launch_begin(kid, st);
        ff_reduce_kernel<T><<<dim3((unsigned)std::min<int64_t>((n + 1023) / 1024, kNumSM * 8), 2 * g.problems), 256, 0, st>>>(r);
        launch_end(kid, st);
        CGB_CUDA(cudaGetLastError());
    }
    return CGB200_OK;
}

template <typename T>
static int ff_fwd(const FfArgs& a, const FfPlan& q, char* ws, cudaStream_t st) {
    if (q.tensor) return ff_tensor<T>(a, q, 0, ws, st);
    launch_begin(K_FF_FWD, st);
    if (a.rows <= kFfFewRows) {
        const unsigned grid = (unsigned)((a.hidden + 3) / 4);
        constexpr int N = Chunk<T>::N;
        const bool edge = a.dim % N != 0 || a.x_stride % N != 0 || a.wg_stride % N != 0 || a.wu_stride % N != 0 ||
                          ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.wg) | reinterpret_cast<uintptr_t>(a.wu)) & 15) != 0;
#define CGB_FEW(M_)                                                             \
    if (edge) ff_few_rows_kernel<T, M_, true><<<grid, 128, 0, st>>>(a);         \
    else ff_few_rows_kernel<T, M_, false><<<grid, 128, 0, st>>>(a);             \
    break
        switch (a.rows) {
            case 1: CGB_FEW(1);
            case 2: CGB_FEW(2);
            case 3: CGB_FEW(3);
            default: CGB_FEW(4);
        }
#undef CGB_FEW
    } else {
        ff_tile_fwd_kernel<T><<<dim3((unsigned)((a.rows + kFfTile - 1) / kFfTile), (a.hidden + kFfTile - 1) / kFfTile), kFfFwdWarps * 32, 0, st>>>(a);
    }
    launch_end(K_FF_FWD, st);
    CGB_CUDA(cudaGetLastError());
    return CGB200_OK;
}

template <typename T>
static int ff_bwd(const FfArgs& a, const FfPlan& q, int grads, char* ws, cudaStream_t st) {
    if (q.tensor) return ff_tensor<T>(a, q, grads, ws, st);
    const int tiles_d = (a.dim + kFfTile - 1) / kFfTile;
    const int64_t nx = a.dx != nullptr ? (a.rows + kFfTile - 1) / kFfTile * tiles_d : 0;
    const int64_t nw = a.dwg != nullptr || a.dwu != nullptr ? (2 * (int64_t)a.hidden + kFfTile - 1) / kFfTile * tiles_d : 0;
    if (nx + nw == 0) return CGB200_OK;
    CGB_REQUIRE(nx + nw <= 0x7fffffff, "gated feed-forward: too many tiles for one launch");
    launch_begin(K_FF_BWD, st);
    ff_tile_bwd_kernel<T><<<(unsigned)(nx + nw), kFfBwdWarps * 32, 0, st>>>(a, (int)nx, tiles_d);
    launch_end(K_FF_BWD, st);
    CGB_CUDA(cudaGetLastError());
    return CGB200_OK;
}

static int ff_check(const FfArgs& a, int64_t rows, int64_t dim, int64_t hidden, int act, int dtype) {
    CGB_REQUIRE(rows >= 0 && rows <= (1ll << 24) && dim > 0 && dim <= (1 << 20) && hidden > 0 && hidden <= (1 << 20),
                "gated feed-forward: sizes out of range");
    CGB_REQUIRE(rows * std::max(dim, hidden) <= (1ll << 38), "gated feed-forward: sizes out of range");      // the tile counts are int
    CGB_REQUIRE(dtype >= CGB200_F32 && dtype <= CGB200_F16, "gated feed-forward: unknown type");
    CGB_REQUIRE(act >= CGB200_ACT_SILU && act <= CGB200_ACT_RELU, "gated feed-forward: unknown activation");
    CGB_REQUIRE(a.wg != nullptr && a.wu != nullptr && (rows == 0 || a.x != nullptr), "gated feed-forward: null buffer");
    CGB_REQUIRE(a.x_stride >= 0 && a.x_stride <= (1ll << 32) && a.wg_stride >= 0 && a.wg_stride <= (1ll << 32) && a.wu_stride >= 0 &&
                    a.wu_stride <= (1ll << 32), "gated feed-forward: row stride out of range");
    return CGB200_OK;
}

static int ff_workspace(const FfPlan& q, const void* ws, int64_t bytes) {
    if (q.bytes > 0 && (ws == nullptr || bytes < q.bytes)) {
        set_error("workspace too small: need " + std::to_string(q.bytes) + " bytes");
        return CGB200_ERR_WORKSPACE;
    }
    CGB_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255) == 0, "workspace must be 256-byte aligned");
    return CGB200_OK;
}

}  // namespace cgb200

using namespace cgb200;

extern "C" {

int64_t cgb200_gated_ff_workspace_bytes(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride, const void* w_up,
                                        int64_t w_up_stride, int64_t rows, int64_t dim, int64_t hidden, int dtype, int gradients) {
    FfArgs a{};
    a.x = x, a.wg = w_gate, a.wu = w_up, a.x_stride = x_stride, a.wg_stride = w_gate_stride, a.wu_stride = w_up_stride;
    a.rows = rows, a.dim = (int)dim, a.hidden = (int)hidden;
    if (ff_check(a, rows, dim, hidden, CGB200_ACT_SILU, dtype) != CGB200_OK) return -1;
    return ff_plan(a, dtype, gradients & 7).bytes;
}

int cgb200_gated_ff_fwd(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride, const void* w_up, int64_t w_up_stride,
                        int activation, void* h, float* gate_up, int64_t rows, int64_t dim, int64_t hidden, int dtype, void* workspace,
                        int64_t workspace_bytes, void* stream) {
    FfArgs a{};
    a.x = x, a.wg = w_gate, a.wu = w_up, a.x_stride = x_stride, a.wg_stride = w_gate_stride, a.wu_stride = w_up_stride;
    a.rows = rows, a.dim = (int)dim, a.hidden = (int)hidden, a.act = activation, a.h = h, a.gu = gate_up;
    a.gu_pitch = up(hidden, 4);
    if (int rc = ff_check(a, rows, dim, hidden, activation, dtype)) return rc;
    if (rows == 0) return CGB200_OK;
    CGB_REQUIRE(h != nullptr, "gated feed-forward: null buffer");
    CGB_REQUIRE((reinterpret_cast<uintptr_t>(gate_up) & 15) == 0, "gated feed-forward: gate_up must be 16-byte aligned");
    const FfPlan q = ff_plan(a, dtype, 0);
    if (int rc = ff_workspace(q, workspace, workspace_bytes)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    char* ws = (char*)workspace;
    return dtype == CGB200_F32 ? ff_fwd<float>(a, q, ws, st) : dtype == CGB200_BF16 ? ff_fwd<__nv_bfloat16>(a, q, ws, st) : ff_fwd<__half>(a, q, ws, st);
}

int cgb200_gated_ff_bwd(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride, const void* w_up, int64_t w_up_stride,
                        int activation, const float* gate_up, const void* dh, int64_t dh_stride, void* dx, void* dw_gate, void* dw_up,
                        int64_t rows, int64_t dim, int64_t hidden, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    FfArgs a{};
    a.x = x, a.wg = w_gate, a.wu = w_up, a.x_stride = x_stride, a.wg_stride = w_gate_stride, a.wu_stride = w_up_stride;
    a.rows = rows, a.dim = (int)dim, a.hidden = (int)hidden, a.act = activation, a.gu = const_cast<float*>(gate_up);
    a.gu_pitch = up(hidden, 4);
    a.dh = dh, a.dh_stride = dh_stride, a.dx = dx, a.dwg = dw_gate, a.dwu = dw_up;
    if (int rc = ff_check(a, rows, dim, hidden, activation, dtype)) return rc;
    CGB_REQUIRE(rows == 0 || (gate_up != nullptr && dh != nullptr), "gated feed-forward: null buffer");
    CGB_REQUIRE(dh_stride >= 0 && dh_stride <= (1ll << 32), "gated feed-forward: row stride out of range");
    const int grads = (dx != nullptr && rows > 0 ? 1 : 0) | (dw_gate != nullptr ? 2 : 0) | (dw_up != nullptr ? 4 : 0);
    if (grads == 0) return CGB200_OK;
    const FfPlan q = ff_plan(a, dtype, grads);
    if (int rc = ff_workspace(q, workspace, workspace_bytes)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    char* ws = (char*)workspace;
    return dtype == CGB200_F32 ? ff_bwd<float>(a, q, grads, ws, st) : dtype == CGB200_BF16 ? ff_bwd<__nv_bfloat16>(a, q, grads, ws, st)
                                                                                         : ff_bwd<__half>(a, q, grads, ws, st);
}

}  // extern "C"
