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

#include "row_ops.cuh"

namespace cgb200 {

struct FfArgs {
    const void *x, *wg, *wu;
    int64_t x_stride, wg_stride, wu_stride;    // values between rows
    int64_t rows;
    int dim, hidden, act;
    void* h;                                   // forward
    float* gu;                                 // [2][rows][hidden]: g, u; null where no backward follows
    const void* dh;                            // backward
    int64_t dh_stride;
    void *dx, *dwg, *dwu;                      // each may be null
};

// act(g) and its derivative
template <bool GRAD>
__device__ __forceinline__ float2 activate(int act, float g) {
    if (act == CGB200_ACT_RELU) return g > 0.f ? make_float2(g, 1.f) : make_float2(g != g ? g : 0.f, 0.f);
    if (act == CGB200_ACT_SILU) {
        const float s = 1.f / (1.f + __expf(-g));
        // where s is 0, g may be -inf
        return s == 0.f ? make_float2(0.f, 0.f) : make_float2(g * s, GRAD ? s * (1.f + g * (1.f - s)) : 0.f);
    }
    const float c = 0.5f * erfcf(-0.70710678118654752f * g);
    return make_float2(c == 0.f ? 0.f : g * c, GRAD ? c + (fabsf(g) > 20.f ? 0.f : g * __expf(-0.5f * g * g) * 0.39894228040143268f) : 0.f);
}

// ---- a few rows: one warp per hidden unit, bound by reading the weights ------------------------------------------------
constexpr int kFfFewRows = 4;

template <typename T, int M>
__global__ void __launch_bounds__(256) ff_few_rows_kernel(FfArgs a) {
    constexpr int N = Chunk<T>::N;
    const int lane = threadIdx.x & 31;
    const int64_t j = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (j >= a.hidden) return;
    const T* wg = (const T*)a.wg + j * a.wg_stride;
    const T* wu = (const T*)a.wu + j * a.wu_stride;
    const int ph = row_phase(wg);
    float g[M], u[M];
#pragma unroll
    for (int m = 0; m < M; ++m) g[m] = u[m] = 0.f;
#pragma unroll 4
    for (int e0 = lane * N - ph; e0 < a.dim; e0 += 32 * N) {
        float vg[N], vu[N];
        load_chunk(wg, e0, a.dim, 0.f, vg);
        load_chunk(wu, e0, a.dim, 0.f, vu);
#pragma unroll
        for (int m = 0; m < M; ++m) {
            float vx[N];
            load_chunk((const T*)a.x + m * a.x_stride, e0, a.dim, 0.f, vx);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                g[m] = fmaf(vg[i], vx[i], g[m]);
                u[m] = fmaf(vu[i], vx[i], u[m]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
        g[m] = warp_sum(g[m]);
        u[m] = warp_sum(u[m]);
        if (lane == 0) {
            ((T*)a.h)[m * (int64_t)a.hidden + j] = from_f32<T>(activate<false>(a.act, g[m]).x * u[m]);
            if (a.gu != nullptr) {
                a.gu[m * (int64_t)a.hidden + j] = g[m];
                a.gu[(a.rows + m) * (int64_t)a.hidden + j] = u[m];
            }
        }
    }
}

// ---- CUDA-core tiles ---------------------------------------------------------------------------------------------------
// 64 x 64 outputs per block, 16 terms of the contraction at a time, 4 x 4 outputs per thread; operands of any alignment.
constexpr int kFfTile = 64, kFfK = 16;

template <typename T>
__global__ void __launch_bounds__(256) ff_tile_fwd_kernel(FfArgs a) {
    __shared__ float sx[kFfK][kFfTile + 4], sg[kFfK][kFfTile + 4], su[kFfK][kFfTile + 4];
    const int64_t m0 = (int64_t)blockIdx.x * kFfTile;
    const int j0 = blockIdx.y * kFfTile;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float g[4][4] = {}, u[4][4] = {};
    for (int k0 = 0; k0 < a.dim; k0 += kFfK) {
        const int k = threadIdx.x & 15;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = (threadIdx.x >> 4) + 16 * r;
            const bool kin = k0 + k < a.dim;
            sx[k][i] = kin && m0 + i < a.rows ? to_f32(((const T*)a.x)[(m0 + i) * a.x_stride + k0 + k]) : 0.f;
            const bool jin = kin && j0 + i < a.hidden;
            sg[k][i] = jin ? to_f32(((const T*)a.wg)[(int64_t)(j0 + i) * a.wg_stride + k0 + k]) : 0.f;
            su[k][i] = jin ? to_f32(((const T*)a.wu)[(int64_t)(j0 + i) * a.wu_stride + k0 + k]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kFfK; ++kk) {
            const float4 x = *(const float4*)&sx[kk][ty * 4], wg = *(const float4*)&sg[kk][tx * 4], wu = *(const float4*)&su[kk][tx * 4];
            const float xv[4] = {x.x, x.y, x.z, x.w}, gv[4] = {wg.x, wg.y, wg.z, wg.w}, uv[4] = {wu.x, wu.y, wu.z, wu.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    g[i][j] = fmaf(xv[i], gv[j], g[i][j]);
                    u[i][j] = fmaf(xv[i], uv[j], u[i][j]);
                }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty * 4 + i;
            const int c = j0 + tx * 4 + j;
            if (m >= a.rows || c >= a.hidden) continue;
            const int64_t at = m * a.hidden + c;
            ((T*)a.h)[at] = from_f32<T>(activate<false>(a.act, g[i][j]).x * u[i][j]);
            if (a.gu != nullptr) a.gu[at] = g[i][j], a.gu[a.rows * a.hidden + at] = u[i][j];
        }
}

// Value (m, c) of dg (c < hidden) or du (c >= hidden) from what the forward kept.
template <typename T>
__device__ __forceinline__ float ff_dgu(const FfArgs& a, int64_t m, int c) {
    const bool up = c >= a.hidden;
    const int j = up ? c - a.hidden : c;
    const int64_t at = m * a.hidden + j;
    const float dh = to_f32(((const T*)a.dh)[m * a.dh_stride + j]);
    const float2 f = activate<true>(a.act, a.gu[at]);
    return up ? dh * f.x : dh * a.gu[a.rows * a.hidden + at] * f.y;
}

// One launch for all gradients: the first `nx` blocks hold tiles of dx, the others tiles of [dWg; dWu].
template <typename T>
__global__ void __launch_bounds__(256) ff_tile_bwd_kernel(FfArgs a, int nx, int tiles_d) {
    __shared__ float sa[kFfK][kFfTile + 4], sb[kFfK][kFfTile + 4];
    const bool is_dx = (int)blockIdx.x < nx;
    const int tile = is_dx ? blockIdx.x : blockIdx.x - nx;
    const int64_t i0 = (int64_t)(tile / tiles_d) * kFfTile;      // row of the output: sample, or hidden unit (g, then u)
    const int d0 = (tile % tiles_d) * kFfTile;
    const int64_t n_i = is_dx ? a.rows : 2 * (int64_t)a.hidden, n_k = is_dx ? 2 * (int64_t)a.hidden : a.rows;
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < n_k; k0 += kFfK) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            {
                // dx reads dgu along its rows, dW down its columns: neighbouring threads take neighbouring addresses in both
                const int k = is_dx ? (threadIdx.x & 15) : (threadIdx.x >> 6) + 4 * r;
                const int i = is_dx ? (threadIdx.x >> 4) + 16 * r : (threadIdx.x & 63);
                float v = 0.f;
                if (k0 + k < n_k && i0 + i < n_i)
                    v = is_dx ? ff_dgu<T>(a, i0 + i, (int)(k0 + k)) : ff_dgu<T>(a, k0 + k, (int)(i0 + i));
                sa[k][i] = v;
            }
            const int k = (threadIdx.x >> 6) + 4 * r, d = threadIdx.x & 63;
            float v = 0.f;
            if (k0 + k < n_k && d0 + d < a.dim) {
                if (!is_dx) v = to_f32(((const T*)a.x)[(k0 + k) * a.x_stride + d0 + d]);
                else if (k0 + k < a.hidden) v = to_f32(((const T*)a.wg)[(k0 + k) * a.wg_stride + d0 + d]);
                else v = to_f32(((const T*)a.wu)[(k0 + k - a.hidden) * a.wu_stride + d0 + d]);
            }
            sb[k][d] = v;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kFfK; ++kk) {
            const float4 x = *(const float4*)&sa[kk][ty * 4], w = *(const float4*)&sb[kk][tx * 4];
            const float xv[4] = {x.x, x.y, x.z, x.w}, wv[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xv[i], wv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t r = i0 + ty * 4 + i;
            const int d = d0 + tx * 4 + j;
            if (r >= n_i || d >= a.dim) continue;
            T* out = is_dx ? (T*)a.dx + r * a.dim : r < a.hidden ? (T*)a.dwg : (T*)a.dwu;
            if (out == nullptr) continue;
            if (!is_dx) out += (r < a.hidden ? r : r - a.hidden) * a.dim;
            out[d] = from_f32<T>(acc[i][j]);
        }
}

template <typename T>
static int ff_fwd(const FfArgs& a, cudaStream_t st) {
    launch_begin(K_FF_FWD, st);
    if (a.rows <= kFfFewRows) {
        const unsigned grid = (unsigned)((a.hidden + 7) / 8);
        switch (a.rows) {
            case 1: ff_few_rows_kernel<T, 1><<<grid, 256, 0, st>>>(a); break;
            case 2: ff_few_rows_kernel<T, 2><<<grid, 256, 0, st>>>(a); break;
            case 3: ff_few_rows_kernel<T, 3><<<grid, 256, 0, st>>>(a); break;
            default: ff_few_rows_kernel<T, 4><<<grid, 256, 0, st>>>(a); break;
        }
    } else {
        ff_tile_fwd_kernel<T><<<dim3((unsigned)((a.rows + kFfTile - 1) / kFfTile), (a.hidden + kFfTile - 1) / kFfTile), 256, 0, st>>>(a);
    }
    launch_end(K_FF_FWD, st);
    CGB_CUDA(cudaGetLastError());
    return CGB200_OK;
}

template <typename T>
static int ff_bwd(const FfArgs& a, cudaStream_t st) {
    const int tiles_d = (a.dim + kFfTile - 1) / kFfTile;
    const int64_t nx = a.dx != nullptr ? (a.rows + kFfTile - 1) / kFfTile * tiles_d : 0;
    const int64_t nw = a.dwg != nullptr || a.dwu != nullptr ? (2 * (int64_t)a.hidden + kFfTile - 1) / kFfTile * tiles_d : 0;
    if (nx + nw == 0) return CGB200_OK;
    CGB_REQUIRE(nx + nw <= 0x7fffffff, "gated feed-forward: too many tiles for one launch");
    launch_begin(K_FF_BWD, st);
    ff_tile_bwd_kernel<T><<<(unsigned)(nx + nw), 256, 0, st>>>(a, (int)nx, tiles_d);
    launch_end(K_FF_BWD, st);
    CGB_CUDA(cudaGetLastError());
    return CGB200_OK;
}

static int ff_check(const FfArgs& a, int64_t rows, int64_t dim, int64_t hidden, int act, int dtype) {
    CGB_REQUIRE(rows >= 0 && rows <= (1ll << 24) && dim > 0 && dim <= (1 << 20) && hidden > 0 && hidden <= (1 << 20),
                "gated feed-forward: sizes out of range");
    CGB_REQUIRE(dtype >= CGB200_F32 && dtype <= CGB200_F16, "gated feed-forward: unknown type");
    CGB_REQUIRE(act >= CGB200_ACT_SILU && act <= CGB200_ACT_RELU, "gated feed-forward: unknown activation");
    CGB_REQUIRE(a.wg != nullptr && a.wu != nullptr && (rows == 0 || a.x != nullptr), "gated feed-forward: null buffer");
    CGB_REQUIRE(a.x_stride >= 0 && a.x_stride <= (1ll << 32) && a.wg_stride >= 0 && a.wg_stride <= (1ll << 32) && a.wu_stride >= 0 &&
                    a.wu_stride <= (1ll << 32), "gated feed-forward: row stride out of range");
    return CGB200_OK;
}

}  // namespace cgb200

using namespace cgb200;

extern "C" {

int64_t cgb200_gated_ff_workspace_bytes(int64_t rows, int64_t dim, int64_t hidden, int dtype, int backward) {
    (void)rows, (void)dim, (void)hidden, (void)dtype, (void)backward;
    return 0;
}

int cgb200_gated_ff_fwd(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride, const void* w_up, int64_t w_up_stride,
                        int activation, void* h, float* gate_up, int64_t rows, int64_t dim, int64_t hidden, int dtype, void* workspace,
                        int64_t workspace_bytes, void* stream) {
    (void)workspace, (void)workspace_bytes;
    FfArgs a{};
    a.x = x, a.wg = w_gate, a.wu = w_up, a.x_stride = x_stride, a.wg_stride = w_gate_stride, a.wu_stride = w_up_stride;
    a.rows = rows, a.dim = (int)dim, a.hidden = (int)hidden, a.act = activation, a.h = h, a.gu = gate_up;
    if (int rc = ff_check(a, rows, dim, hidden, activation, dtype)) return rc;
    if (rows == 0) return CGB200_OK;
    CGB_REQUIRE(h != nullptr, "gated feed-forward: null buffer");
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == CGB200_F32 ? ff_fwd<float>(a, st) : dtype == CGB200_BF16 ? ff_fwd<__nv_bfloat16>(a, st) : ff_fwd<__half>(a, st);
}

int cgb200_gated_ff_bwd(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride, const void* w_up, int64_t w_up_stride,
                        int activation, const float* gate_up, const void* dh, int64_t dh_stride, void* dx, void* dw_gate, void* dw_up,
                        int64_t rows, int64_t dim, int64_t hidden, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    (void)workspace, (void)workspace_bytes;
    FfArgs a{};
    a.x = x, a.wg = w_gate, a.wu = w_up, a.x_stride = x_stride, a.wg_stride = w_gate_stride, a.wu_stride = w_up_stride;
    a.rows = rows, a.dim = (int)dim, a.hidden = (int)hidden, a.act = activation, a.gu = const_cast<float*>(gate_up);
    a.dh = dh, a.dh_stride = dh_stride, a.dx = dx, a.dwg = dw_gate, a.dwu = dw_up;
    if (int rc = ff_check(a, rows, dim, hidden, activation, dtype)) return rc;
    CGB_REQUIRE(rows == 0 || (gate_up != nullptr && dh != nullptr), "gated feed-forward: null buffer");
    CGB_REQUIRE(dh_stride >= 0 && dh_stride <= (1ll << 32), "gated feed-forward: row stride out of range");
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == CGB200_F32 ? ff_bwd<float>(a, st) : dtype == CGB200_BF16 ? ff_bwd<__nv_bfloat16>(a, st) : ff_bwd<__half>(a, st);
}

}  // extern "C"
