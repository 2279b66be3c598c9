// Layer norm over the last axis, forward and backward, with the gradients of weight and bias.
//
//   y  = (x - mean) * rstd * w + b,    rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd * (w dy - mean(w dy) - xh * mean(w dy * xh)),   xh = (x - mean) * rstd
//   dw = sum over rows of dy * xh,     db = sum over rows of dy
//
// Everything is held in float32 between the loads and the one rounding of each result.  The variance is taken over centred
// values that stay in registers (not as a difference of moments), so a large common offset of a row costs it no digits; the mean's own
// rounding, a few units of 2^-24 of it, stays in y.
#include <cooperative_groups.h>

#include <algorithm>

#include "row_ops.cuh"
#include "tc_ptx.cuh"

namespace cgb200 {

namespace cg = cooperative_groups;

constexpr int kLnMaxChunks = 4;        // chunks of a row a thread of the forward kernel holds in registers
constexpr int kLnBwdValues = 16;       // values of a row a thread of the backward kernel holds
constexpr int kLnBwdMaxThreads = 512;
constexpr int kLnCluster = 8;          // blocks of 16 warps that add up the parameters' gradients in one launch
constexpr int64_t kLnClusterRows = 8 * 16 * kLnCluster;

struct LnArgs {
    const void* x;
    int64_t x_stride;       // values between rows
    const void* w;          // may be null: 1
    const void* b;          // may be null: 0
    float eps;
    int64_t rows, dim;
};

// Sum over the threads that share a row: a warp, or the whole block.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* buf) {
    return WARP ? warp_sum(v) : block_sum(v, buf);
}

// One row per warp (WARP) or per block; its values stay in registers between the three steps, so x is read once.  A warp has weight
// and bias on their way before the first value is waited for; a block fetches them chunk by chunk at the end (with all of them in
// registers 8192 x 4096 bf16 took 27 instead of 25 us, and 81 instead of 33 with float32 weights, which spilled).  EDGE: rows (or
// weight and bias) that do not start on 16-byte boundaries or do not end on them; without it every chunk is inside the row or
// behind it.
// Bound by the one read and the one write: 8192 x 4096 bf16 (134 MB) 25 us in a row of calls = 5.3 TB/s.  Rows that start anywhere
// take twice the instructions, for shifting the groups: 3001 x 1023 fp16 6.7 us against 3.6 at 1024 columns.
template <typename T, typename P, int CH, bool WARP, bool EDGE>
__global__ void __launch_bounds__(WARP ? 128 : 1024) ln_fwd_kernel(LnArgs a, float inv_n, T* __restrict__ y, float2* __restrict__ stats) {
    constexpr int N = Chunk<T>::N;
    __shared__ float red[2][32];
    __shared__ uint4 last[EDGE && !WARP ? 32 : 1];     // each warp's last chunk, for the next warp
    const int lane = threadIdx.x & 31, warp = (int)(threadIdx.x >> 5), n = (int)a.dim;
    const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : (int64_t)blockIdx.x;
    if (row >= a.rows) return;               // whole warps or whole blocks leave
    const T* xr = (const T*)a.x + row * a.x_stride;
    T* yr = y + row * a.dim;
    const int k0 = WARP ? 0 : warp * 32 * CH, k = k0 + lane;       // this thread's first chunk, the next ones are 32 further
    const bool before = EDGE && row > 0 && a.x_stride >= n && n >= N, behind = EDGE && row + 1 < a.rows && a.x_stride >= n && n >= N;
    uint4 raw[CH];
    Params<P, N> w[CH], b[CH];
    const bool whole = EDGE && aligned16(a.w) && aligned16(a.b);
    const int end = n / N * N;           // where a chunk begins that the row does not fill
    P w_end = from_f32<P>(0.f), b_end = w_end;
    auto load_wb = [&](int from, int to) {
        if (from == 0 && whole && lane < n - end) {
            if (a.w != nullptr) w_end = ((const P*)a.w)[end + lane];
            if (a.b != nullptr) b_end = ((const P*)a.b)[end + lane];
        }
#pragma unroll
        for (int c = from; c < to; ++c) {
            const int e0 = (k + 32 * c) * N;
            if (whole) {
                if (a.w != nullptr) w[c].load_whole((const P*)a.w, e0, n);
                if (a.b != nullptr) b[c].load_whole((const P*)a.b, e0, n);
            } else if (EDGE) {
                if (a.w != nullptr) w[c].load((const P*)a.w, e0, n);
                if (a.b != nullptr) b[c].load((const P*)a.b, e0, n);
            } else if (e0 < n) {
                if (a.w != nullptr) w[c].load_aligned((const P*)a.w + e0);
                if (a.b != nullptr) b[c].load_aligned((const P*)a.b + e0);
            }
        }
    };
    if (EDGE && !(before && behind)) {
#pragma unroll
        for (int c = 0; c < CH; ++c) raw[c] = load_at(xr, row_phase(xr), k + 32 * c, n, before, behind);
    } else if (EDGE) {
        const int ph = row_phase(xr);
        uint4 next[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (k + 32 * c) * N - ph;
            raw[c] = e0 < n ? *reinterpret_cast<const uint4*>(xr + e0) : make_uint4(0, 0, 0, 0);
            next[c] = ph != 0 && e0 + N < n ? *reinterpret_cast<const uint4*>(xr + e0 + N) : make_uint4(0, 0, 0, 0);
        }
        if (ph != 0) {
#pragma unroll
            for (int c = 0; c < CH; ++c) raw[c] = shifted(raw[c], next[c], ph * (int)sizeof(T));
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (k + 32 * c) * N;
            raw[c] = e0 < n ? *reinterpret_cast<const uint4*>(xr + e0) : make_uint4(0, 0, 0, 0);
        }
    }
    if (WARP) load_wb(0, CH);
    uint64_t v[CH][N / 2];              // pairs of columns
    // what lies behind the row's end counts for nothing; only a warp that reaches it has to look
    auto cut = [&](int c) {
        if ((k0 + 32 * c + 32) * N <= n) return;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const int e = (k + 32 * c) * N + (EDGE ? i : 0);
            const float2 d = unpair(v[c][i / 2]);
            v[c][i / 2] = pair(e < n ? d.x : 0.f, (EDGE ? e + 1 : e) < n ? d.y : 0.f);
        }
    };
    uint64_t s2 = pair(0.f, 0.f), q2 = s2;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float t[N];
        unpack16(raw[c], t, (const T*)nullptr);
#pragma unroll
        for (int i = 0; i < N; i += 2) v[c][i / 2] = pair(t[i], t[i + 1]);
        if (EDGE) cut(c);               // values of the next row
#pragma unroll
        for (int i = 0; i < N / 2; ++i) s2 = add2(s2, v[c][i]);
    }
    const float2 s = unpair(s2);
    const float mean = row_sum<WARP>(s.x + s.y, red[0]) * inv_n;
    const uint64_t mean2 = pair(-mean, -mean);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[c][i] = add2(v[c][i], mean2);
        cut(c);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) q2 = fma2(v[c][i], v[c][i], q2);
    }
    const float2 q = unpair(q2);
    const float rstd = 1.f / sqrtf(row_sum<WARP>(q.x + q.y, red[1]) * inv_n + a.eps);
    const uint64_t rstd2 = pair(rstd, rstd);
    if (stats != nullptr && (WARP ? lane : (int)threadIdx.x) == 0) stats[row] = make_float2(mean, rstd);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e0 = (k + 32 * c) * N;
        float t[N];
        if (!WARP) load_wb(c, c + 1);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[c][i] = mul2(v[c][i], rstd2);
        if (whole && end != n && end >= e0 - lane * N && end < e0 + (32 - lane) * N) {       // the same in the whole warp
            w[c].place_end(w_end, e0, n);
            b[c].place_end(b_end, e0, n);
        }
        if (a.w != nullptr) {
            w[c].get(t);
#pragma unroll
            for (int i = 0; i < N; i += 2) v[c][i / 2] = mul2(v[c][i / 2], pair(t[i], t[i + 1]));
        }
        if (a.b != nullptr) {
            b[c].get(t);
#pragma unroll
            for (int i = 0; i < N; i += 2) v[c][i / 2] = add2(v[c][i / 2], pair(t[i], t[i + 1]));
        }
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 d = unpair(v[c][i / 2]);
            t[i] = d.x, t[i + 1] = d.y;
        }
        raw[c] = pack16(t, (const T*)nullptr);
        if (!EDGE && e0 < n) *reinterpret_cast<uint4*>(yr + e0) = raw[c];
    }
    if (EDGE) {
        uint4 before = raw[0];
        if (!WARP) {
            if (lane == 31) last[warp] = raw[CH - 1];
            __syncthreads();
            if (warp > 0) before = last[warp - 1];
        }
        store_groups<T, CH>(yr, row_phase(yr), k0, n, raw, before);
        // the row's last values, where they are this warp's last chunk's and the group behind it is no one's
        if (lane == 31 && (WARP || warp == (int)(blockDim.x >> 5) - 1)) {
            const int tail = (k0 + 32 * CH) * N - row_phase(yr);
            if (tail < n) store_pieces(yr, tail, n, shifted(raw[CH - 1], raw[CH - 1], (N - row_phase(yr)) * (int)sizeof(T)));
        }
    }
}

// Rows too long for registers: one block per row, three passes over it (the second and third from L2).  512 x 65536 bf16 76 us:
// a row that stayed in a cluster's shared memory would need one pass, but such rows are rare behind an embedding.
template <typename T, typename P>
__global__ void ln_fwd_long_kernel(LnArgs a, T* __restrict__ y, float2* __restrict__ stats) {
    constexpr int N = Chunk<T>::N;
    __shared__ float red[2][32];
    const int64_t row = blockIdx.x;
    const T* xr = (const T*)a.x + row * a.x_stride;
    T* yr = y + row * a.dim;
    const int ph = row_phase(xr);
    float v[N];
    float s = 0.f;
    for (int64_t e0 = (int64_t)threadIdx.x * N - ph; e0 < a.dim; e0 += (int64_t)blockDim.x * N) {
        load_chunk(xr, e0, a.dim, 0.f, v);
#pragma unroll
        for (int i = 0; i < N; ++i) s += v[i];
    }
    const float mean = block_sum(s, red[0]) / (float)a.dim;
    float q = 0.f;
    for (int64_t e0 = (int64_t)threadIdx.x * N - ph; e0 < a.dim; e0 += (int64_t)blockDim.x * N) {
        load_chunk(xr, e0, a.dim, mean, v);
#pragma unroll
        for (int i = 0; i < N; ++i) q += (v[i] - mean) * (v[i] - mean);
    }
    const float rstd = 1.f / sqrtf(block_sum(q, red[1]) / (float)a.dim + a.eps);
    if (stats != nullptr && threadIdx.x == 0) stats[row] = make_float2(mean, rstd);
    for (int64_t e0 = (int64_t)threadIdx.x * N - ph; e0 < a.dim; e0 += (int64_t)blockDim.x * N) {
        load_chunk(xr, e0, a.dim, 0.f, v);
        float w[N], b[N];
        if (a.w != nullptr) load_params((const P*)a.w, e0, a.dim, w);
        if (a.b != nullptr) load_params((const P*)a.b, e0, a.dim, b);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float o = (v[i] - mean) * rstd;
            if (a.w != nullptr) o *= w[i];
            if (a.b != nullptr) o += b[i];
            v[i] = o;
        }
        store_chunk(yr, e0, a.dim, v);
    }
}

struct LnBwdArgs {
    const void* x;
    int64_t x_stride;
    const void* dy;
    int64_t dy_stride;
    const void* w;
    const float2* stats;
    void* dx;               // may be null: only the parameters' gradients are wanted
    float* part;            // [gridDim.x][2][dim]; null: the parameters' gradients are not wanted, or are joined by the cluster
    void *dw, *db;          // where the blocks are one cluster, which adds up its sums itself (each may be null)
    int64_t rows, dim;
};

template <typename T, int VE>
__device__ __forceinline__ void load_values(const T* p, int64_t e0, int64_t n, float (&v)[VE]) {
    if (VE > 1) {
        if (e0 < n) {
            float t[Chunk<T>::N];
            unpack16(*reinterpret_cast<const uint4*>(p + e0), t, (const T*)nullptr);
#pragma unroll
            for (int i = 0; i < VE; ++i) v[i] = t[i % Chunk<T>::N];
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) v[i] = 0.f;
        }
    } else {
        v[0] = e0 < n ? to_f32(p[e0]) : 0.f;
    }
}
template <typename T, int VE>
__device__ __forceinline__ void store_values(T* p, int64_t e0, int64_t n, const float (&v)[VE]) {
    if (e0 >= n) return;
    if (VE > 1) {
        float t[Chunk<T>::N];
#pragma unroll
        for (int i = 0; i < Chunk<T>::N; ++i) t[i] = v[i % VE];
        *reinterpret_cast<uint4*>(p + e0) = pack16(t, (const T*)nullptr);
    } else {
        p[e0] = from_f32<T>(v[0]);
    }
}

// A lane owns the same columns of every row its warp visits, so the sums over rows stay in registers until the end: x and dy are
// read once for all three gradients.  VE values per access (16 bytes, or one value where rows do not start on 16-byte
// boundaries), NC accesses.  Each block leaves one partial sum per column; ln_param_reduce_kernel adds them, so the result does
// not depend on timing.  Up to kLnClusterRows rows are one cluster whose blocks add their sums through each other's shared memory:
// such a call is latency alone, and a second launch would be half of it (100 x 52 fp32: 10.8 us cold, all three gradients).
template <typename T, typename P, int VE, int NC>
__global__ void __launch_bounds__(kLnBwdMaxThreads) ln_bwd_kernel(LnBwdArgs a) {
    extern __shared__ float sm[];
    const int t = (int)(threadIdx.x & 31), warp = threadIdx.x >> 5, nwarps = (int)(blockDim.x >> 5);
    const float inv_n = 1.f / (float)a.dim;
    float w[NC][VE], dw[NC][VE], db[NC][VE];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int64_t e0 = (int64_t)(t + c * 32) * VE;
        if (a.w != nullptr) {
            load_params<P, VE>((const P*)a.w, e0, a.dim, w[c]);
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) w[c][i] = 1.f;
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) dw[c][i] = db[c][i] = 0.f;
    }
    for (int64_t row = (int64_t)blockIdx.x * nwarps + warp; row < a.rows; row += (int64_t)gridDim.x * nwarps) {
        const T* xr = (const T*)a.x + row * a.x_stride;
        const T* gr = (const T*)a.dy + row * a.dy_stride;
        const float2 st = a.stats[row];
        float xh[NC][VE], g[NC][VE];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int64_t e0 = (int64_t)(t + c * 32) * VE;
            load_values<T, VE>(xr, e0, a.dim, xh[c]);
            load_values<T, VE>(gr, e0, a.dim, g[c]);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                xh[c][i] = (xh[c][i] - st.x) * st.y;     // beyond the row g is 0, so xh there counts for nothing
                dw[c][i] = fmaf(g[c][i], xh[c][i], dw[c][i]);
                db[c][i] += g[c][i];
                g[c][i] *= w[c][i];
                s1 += g[c][i];
                s2 = fmaf(g[c][i], xh[c][i], s2);
            }
        }
        if (a.dx != nullptr) {
            const float m1 = warp_sum(s1) * inv_n, m2 = warp_sum(s2) * inv_n;
            T* dxr = (T*)a.dx + row * a.dim;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float o[VE];
#pragma unroll
                for (int i = 0; i < VE; ++i) o[i] = st.y * (g[c][i] - m1 - xh[c][i] * m2);
                store_values<T, VE>(dxr, (int64_t)(t + c * 32) * VE, a.dim, o);
            }
        }
    }
    if (a.part == nullptr && a.dw == nullptr && a.db == nullptr) return;
    // the block's warps, in order
    const int n = (int)a.dim, n2 = 2 * n;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const int e = (t + c * 32) * VE + i;
            if (e < n) sm[warp * n2 + e] = dw[c][i], sm[warp * n2 + n + e] = db[c][i];
        }
    __syncthreads();
    for (int e = threadIdx.x; e < n2; e += blockDim.x) {
        float s = 0.f;
        for (int k = 0; k < nwarps; ++k) s += sm[k * n2 + e];
        if (a.part != nullptr) a.part[(int64_t)blockIdx.x * n2 + e] = s;
        else sm[e] = s;                  // only this thread has read column e of warp 0
    }
    if (a.part != nullptr) return;
    // and the cluster's blocks, in order: each block adds up its share of the columns
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int e = (int)(blockIdx.x * blockDim.x + threadIdx.x); e < n2; e += (int)(gridDim.x * blockDim.x)) {
        float s = 0.f;
        for (int k = 0; k < (int)gridDim.x; ++k) s += cluster.map_shared_rank(sm, k)[e];
        P* out = (P*)(e < n ? a.dw : a.db);
        if (out != nullptr) out[e < n ? e : e - n] = from_f32<P>(s);
    }
    cluster.sync();                      // no block leaves while its sums are read
}

// The same for rows of a block, which come through shared memory: a ring of `stages` rows of x and dy, filled by the bulk copies of
// one thread, keeps reads in flight across the barriers of a row.  Bulk copies move whole 16-byte groups.  EDGE: rows start
// anywhere; a copy then takes the groups the row lies in, with values of its neighbours at both ends, except for the matrix's
// first and last row (and rows that overlap), where the groups at the ends are read value by value.
constexpr size_t kLnRingBytes = 200 * 1024;     // of the blocks of an SM together
constexpr int kLnRingStages = 8;
constexpr int kLnBwdThreadsPerSM = 512;         // of these kernels: 128 registers a thread

// Groups a row of n values can touch, wherever it starts
template <typename T>
static __host__ __device__ int ring_groups(int64_t n, bool edge) {
    constexpr int N = Chunk<T>::N;
    return (int)((n + (edge ? N - 1 : 0) + N - 1) / N);
}
// What the ring holds of a row, and where: groups [g0, g1) of those that start `ph` values before it.
struct RingRow {
    int ph, g0, g1;
};
template <typename T, bool EDGE>
__device__ __forceinline__ RingRow ring_row(const T* r, int64_t row, int64_t rows, int64_t stride, int n) {
    constexpr int N = Chunk<T>::N;
    if (!EDGE) return RingRow{0, 0, n / N};
    const int ph = row_phase(r);
    return RingRow{ph, ph > 0 && (row == 0 || stride < n) ? 1 : 0, row == rows - 1 || stride < n ? (ph + n) / N : (ph + n + N - 1) / N};
}
template <typename T, bool EDGE>
__device__ __forceinline__ uint4 ring_at(const uint4* slot, const RingRow& q, const T* r, int k, int n, bool whole) {
    if (!EDGE) return slot[k];
    if (whole) return q.ph == 0 ? slot[k] : shifted(slot[k], slot[min(k + 1, q.g1 - 1)], q.ph * (int)sizeof(T));
    const uint4 lo = k >= q.g0 && k < q.g1 ? slot[k] : load_group(r, q.ph, k, n);
    if (q.ph == 0) return lo;
    const int j = k + 1;
    const uint4 hi = j >= q.g0 && j < q.g1 ? slot[j] : load_group(r, q.ph, j, n);
    return shifted(lo, hi, q.ph * (int)sizeof(T));
}

template <typename T, typename P, int NC, bool EDGE>
__global__ void __launch_bounds__(kLnBwdMaxThreads) ln_bwd_ring_kernel(LnBwdArgs a, int stages, uint32_t polls) {
    constexpr int VE = Chunk<T>::N;
    extern __shared__ __align__(128) char ring[];
    __shared__ float red[4][32];
    __shared__ uint4 last[EDGE ? kLnBwdMaxThreads / 32 : 1];
    __shared__ uint64_t full[kLnRingStages];
    __shared__ int failed_flag;
    volatile int* failed = &failed_flag;
    const int t = (int)threadIdx.x, warp = t >> 5, lane = t & 31, nwarps = (int)(blockDim.x >> 5), n = (int)a.dim;
    const int k0 = warp * 32 * NC, k = k0 + lane;          // this thread's first chunk, the next ones are 32 further
    const int slot = ring_groups<T>(a.dim, EDGE);           // groups of a row in the ring
    const float inv_n = 1.f / (float)a.dim;
    const int64_t n_here = (a.rows - blockIdx.x + gridDim.x - 1) / gridDim.x;      // rows blockIdx.x, + gridDim.x, ...
    auto place = [&](int s) { return (uint4*)ring + (size_t)s * 2 * slot; };
    auto fetch = [&](int64_t i, int s) {
        const int64_t row = blockIdx.x + i * gridDim.x;
        const T* xr = (const T*)a.x + row * a.x_stride;
        const T* gr = (const T*)a.dy + row * a.dy_stride;
        const RingRow qx = ring_row<T, EDGE>(xr, row, a.rows, a.x_stride, n), qg = ring_row<T, EDGE>(gr, row, a.rows, a.dy_stride, n);
        const uint32_t bx = (uint32_t)max(0, qx.g1 - qx.g0) * 16, bg = (uint32_t)max(0, qg.g1 - qg.g0) * 16;
        mbar_arrive_expect_tx(&full[s], bx + bg);
        if (bx > 0) bulk_g2s(place(s) + qx.g0, xr + (qx.g0 * VE - qx.ph), bx, &full[s]);
        if (bg > 0) bulk_g2s(place(s) + slot + qg.g0, gr + (qg.g0 * VE - qg.ph), bg, &full[s]);
    };
    if (t == 0) {
        failed_flag = 0;
        for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
        for (int s = 0; s < stages && s < n_here; ++s) fetch(s, s);
    }
    uint64_t w[NC][VE / 2], dw[NC][VE / 2], db[NC][VE / 2];      // pairs of columns
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float wv[VE];
        if (a.w != nullptr) {
            load_params<P, VE>((const P*)a.w, (k + 32 * c) * VE, a.dim, wv);
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) wv[i] = 1.f;
        }
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) w[c][i] = pair(wv[2 * i], wv[2 * i + 1]), dw[c][i] = db[c][i] = pair(0.f, 0.f);
    }
    __syncthreads();
    int s = 0, flip = 0;
    uint32_t phase = 0;
    float2 st = a.stats[blockIdx.x];
    for (int64_t i = 0; i < n_here; ++i) {
        const int64_t row = blockIdx.x + i * gridDim.x;
        const float2 now = st;
        if (i + 1 < n_here) st = a.stats[row + gridDim.x];
        // a wait that ran out (it cannot, short of a broken copy) makes this row and the sums NaN and goes on
        const float ok = mbar_wait(&full[s], phase, failed, polls) ? 0.f : __uint_as_float(kNaNBits);
        const T* xr = (const T*)a.x + row * a.x_stride;
        const T* gr = (const T*)a.dy + row * a.dy_stride;
        const RingRow qx = ring_row<T, EDGE>(xr, row, a.rows, a.x_stride, n), qg = ring_row<T, EDGE>(gr, row, a.rows, a.dy_stride, n);
        uint64_t xh[NC][VE / 2], g[NC][VE / 2];
        // every group of both rows is in the ring
        const bool whole = EDGE && qx.g0 == 0 && qg.g0 == 0 && qx.g1 * VE >= qx.ph + n && qg.g1 * VE >= qg.ph + n;
        uint64_t p1 = pair(ok, ok), p2 = p1;
        const uint64_t mean2 = pair(-now.x, -now.x), rstd2 = pair(now.y, now.y), ok2 = p1;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int at = k + 32 * c;
            float xv[VE], gv[VE];
            if (at * VE < n) {
                unpack16(ring_at<T, EDGE>(place(s), qx, xr, at, n, whole), xv, (const T*)nullptr);
                unpack16(ring_at<T, EDGE>(place(s) + slot, qg, gr, at, n, whole), gv, (const T*)nullptr);
                if (EDGE && (at + 1) * VE > n) {
#pragma unroll
                    for (int j = 0; j < VE; ++j)
                        if (at * VE + j >= n) xv[j] = gv[j] = 0.f;
                }
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j) xv[j] = gv[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < VE / 2; ++j) {
                const uint64_t x2 = mul2(add2(pair(xv[2 * j], xv[2 * j + 1]), mean2), rstd2);     // beyond the row g is 0, so it counts for nothing
                const uint64_t g2 = pair(gv[2 * j], gv[2 * j + 1]), wg = mul2(g2, w[c][j]);
                dw[c][j] = fma2(g2, x2, dw[c][j]);
                db[c][j] = add2(db[c][j], g2);
                p1 = add2(p1, wg);
                p2 = fma2(wg, x2, p2);
                xh[c][j] = x2, g[c][j] = wg;
            }
            dw[c][0] = add2(dw[c][0], ok2), db[c][0] = add2(db[c][0], ok2);
        }
        const float2 h1 = unpair(p1), h2 = unpair(p2);
        const float s1 = warp_sum(h1.x + h1.y), s2 = warp_sum(h2.x + h2.y);
        float *r1 = red[flip], *r2 = red[flip + 2];
        flip ^= 1;
        if (lane == 0) r1[warp] = s1, r2[warp] = s2;
        __syncthreads();
        // every thread has this stage in registers
        if (t == 0 && i + stages < n_here) fetch(i + stages, s);
        const float m1 = warp_sum(lane < nwarps ? r1[lane] : 0.f) * inv_n, m2 = warp_sum(lane < nwarps ? r2[lane] : 0.f) * inv_n;
        if (a.dx != nullptr) {
            const uint64_t m1n = pair(-m1, -m1), m2n = pair(-m2, -m2);
            T* dxr = (T*)a.dx + row * a.dim;
            uint4 out[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float o[VE];
#pragma unroll
                for (int j = 0; j < VE / 2; ++j) {
                    const float2 d = unpair(mul2(rstd2, fma2(xh[c][j], m2n, add2(g[c][j], m1n))));
                    o[2 * j] = d.x, o[2 * j + 1] = d.y;
                }
                out[c] = pack16(o, (const T*)nullptr);
                if (!EDGE && (k + 32 * c) * VE < n) *reinterpret_cast<uint4*>(dxr + (k + 32 * c) * VE) = out[c];
            }
            if (EDGE) {
                const int ph = row_phase(dxr);
                if (lane == 31) last[warp] = out[NC - 1];
                __syncthreads();          // before the next row's barrier, behind which `last` is written again
                store_groups<T, NC>(dxr, ph, k0, n, out, warp > 0 ? last[warp - 1] : out[0]);
                const int tail = (k0 + 32 * NC) * VE - ph;
                if (lane == 31 && warp == nwarps - 1 && tail < n) store_pieces(dxr, tail, n, shifted(out[NC - 1], out[NC - 1], (VE - ph) * (int)sizeof(T)));
            }
        }
        if (++s == stages) s = 0, phase ^= 1;
    }
    if (failed_flag && t == 0) {
        // let the copies still on their way land before the block gives up its shared memory
        for (int64_t i = max((int64_t)0, n_here - stages); i < n_here; ++i) mbar_drain(&full[i % stages], (uint32_t)(i / stages) & 1, polls);
    }
    if (a.part == nullptr) return;
    // through the ring's memory, which no thread reads any more, so that neighbours write side by side: straight from the threads, a
    // block's sums took as long as four of its rows
    float* sums = (float*)ring;
    const int pitch = (n + VE - 1) / VE * VE;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int e0 = (k + 32 * c) * VE;
        if (e0 >= n) continue;
#pragma unroll
        for (int j = 0; j < VE; j += 4) {
            const float2 v0 = unpair(dw[c][j / 2]), v1 = unpair(dw[c][j / 2 + 1]), u0 = unpair(db[c][j / 2]), u1 = unpair(db[c][j / 2 + 1]);
            *(float4*)(sums + e0 + j) = make_float4(v0.x, v0.y, v1.x, v1.y);
            *(float4*)(sums + pitch + e0 + j) = make_float4(u0.x, u0.y, u1.x, u1.y);
        }
    }
    __syncthreads();
    float* out = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    for (int e = t; e < n; e += (int)blockDim.x) out[e] = sums[e], out[a.dim + e] = sums[pitch + e];
}

// Rows too long for registers: dx alone, one block per row, and x and dy again from L2 for the columns' sums below (512 x 65536 bf16,
// 268 MB of HBM traffic at least: 131 us with them, 2 TB/s).
template <typename T, typename P>
__global__ void ln_bwd_long_kernel(LnBwdArgs a) {
    constexpr int N = Chunk<T>::N;
    __shared__ float red[2][32];
    const int64_t row = blockIdx.x;
    const T* xr = (const T*)a.x + row * a.x_stride;
    const T* gr = (const T*)a.dy + row * a.dy_stride;
    T* dxr = (T*)a.dx + row * a.dim;
    const int ph = row_phase(xr);
    const float2 st = a.stats[row];
    float s1 = 0.f, s2 = 0.f;
    float x[N], g[N], w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 1.f;
    for (int64_t e0 = (int64_t)threadIdx.x * N - ph; e0 < a.dim; e0 += (int64_t)blockDim.x * N) {
        load_chunk(xr, e0, a.dim, st.x, x);
        load_chunk(gr, e0, a.dim, 0.f, g);
        if (a.w != nullptr) load_params((const P*)a.w, e0, a.dim, w);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s1 += g[i] * w[i];
            s2 += g[i] * w[i] * ((x[i] - st.x) * st.y);
        }
    }
    const float m1 = block_sum(s1, red[0]) / (float)a.dim, m2 = block_sum(s2, red[1]) / (float)a.dim;
    for (int64_t e0 = (int64_t)threadIdx.x * N - ph; e0 < a.dim; e0 += (int64_t)blockDim.x * N) {
        load_chunk(xr, e0, a.dim, st.x, x);
        load_chunk(gr, e0, a.dim, 0.f, g);
        if (a.w != nullptr) load_params((const P*)a.w, e0, a.dim, w);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = st.y * (g[i] * w[i] - m1 - (x[i] - st.x) * st.y * m2);
        store_chunk(dxr, e0, a.dim, x);
    }
}

// The parameters' gradients for such rows: thread = column, blockIdx.y = one run of rows.
template <typename T>
__global__ void ln_bwd_cols_kernel(LnBwdArgs a, int64_t rows_per_part) {
    const int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (e >= a.dim) return;
    const int64_t r0 = (int64_t)blockIdx.y * rows_per_part, r1 = min(a.rows, r0 + rows_per_part);
    float dw = 0.f, db = 0.f;
    for (int64_t r = r0; r < r1; ++r) {
        const float2 st = a.stats[r];
        const float g = to_f32(((const T*)a.dy)[r * a.dy_stride + e]);
        dw += g * ((to_f32(((const T*)a.x)[r * a.x_stride + e]) - st.x) * st.y);
        db += g;
    }
    a.part[(int64_t)blockIdx.y * 2 * a.dim + e] = dw;
    a.part[(int64_t)blockIdx.y * 2 * a.dim + a.dim + e] = db;
}

// Partial sums [parts][2][dim] -> dw, db: 32 columns per block, thread row y adds parts y, y + 32, ... and the sums of the thread
// rows are added by a tree.  296 parts of 4096 columns: 6.8 us.
template <typename P>
__global__ void __launch_bounds__(1024) ln_param_reduce_kernel(const float* __restrict__ part, int parts, int64_t dim, P* __restrict__ dw,
                                                               P* __restrict__ db) {
    __shared__ float sm[32][33];
    const int64_t e = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (e < 2 * dim) {
        const float* src = part + e;
        const int64_t step = 2 * dim;
        int p = threadIdx.y;
        for (; p + 96 < parts; p += 128) {
            const float a = src[p * step], b = src[(p + 32) * step], c = src[(p + 64) * step], d = src[(p + 96) * step];
            s += a, s += b, s += c, s += d;
        }
        for (; p < parts; p += 32) s += src[p * step];
    }
    sm[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    // thread row y has column y of the 32 x 32 sums, one per lane
    s = warp_sum(sm[threadIdx.x][threadIdx.y]);
    const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && col < 2 * dim) {
        if (col < dim) {
            if (dw != nullptr) dw[col] = from_f32<P>(s);
        } else if (db != nullptr) {
            db[col - dim] = from_f32<P>(s);
        }
    }
}

// ---- launches ------------------------------------------------------------------------------------------------------
template <typename T, typename P, bool WARP, bool EDGE>
static void ln_fwd_launch(int ch, unsigned grid, int threads, const LnArgs& a, T* y, float2* stats, cudaStream_t st) {
    const float inv_n = 1.f / (float)a.dim;
    if constexpr (WARP) {
        if (ch == 1) { ln_fwd_kernel<T, P, 1, WARP, EDGE><<<grid, threads, 0, st>>>(a, inv_n, y, stats); return; }
        if (ch == 2) { ln_fwd_kernel<T, P, 2, WARP, EDGE><<<grid, threads, 0, st>>>(a, inv_n, y, stats); return; }
    }
    ln_fwd_kernel<T, P, kLnMaxChunks, WARP, EDGE><<<grid, threads, 0, st>>>(a, inv_n, y, stats);
}
static int pow2_at_least(int64_t n) {
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

template <typename T, typename P>
static int ln_fwd(const LnArgs& a, void* y, float2* stats, cudaStream_t st) {
    constexpr int N = Chunk<T>::N;
    auto at16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const bool edge = a.dim % N != 0 || a.x_stride % N != 0 || !at16(a.x) || !at16(y) || !at16(a.w) || !at16(a.b);
    const int64_t chunks = (a.dim + N - 1) / N;
    launch_begin(K_LN_FWD, st);
    if (chunks <= 32 * kLnMaxChunks) {
        const int ch = pow2_at_least((chunks + 31) / 32);
        const unsigned grid = (unsigned)((a.rows + 3) / 4);
        if (edge) ln_fwd_launch<T, P, true, true>(ch, grid, 128, a, (T*)y, stats, st);
        else ln_fwd_launch<T, P, true, false>(ch, grid, 128, a, (T*)y, stats, st);
    } else if (chunks <= 1024 * kLnMaxChunks) {
        // four chunks a thread; two and twice the threads took 39 instead of 31 us at 8192 x 4096 bf16
        const int ch = kLnMaxChunks, threads = (int)((chunks + 32 * ch - 1) / (32 * ch)) * 32;
        if (edge) ln_fwd_launch<T, P, false, true>(ch, (unsigned)a.rows, threads, a, (T*)y, stats, st);
        else ln_fwd_launch<T, P, false, false>(ch, (unsigned)a.rows, threads, a, (T*)y, stats, st);
    } else {
        ln_fwd_long_kernel<T, P><<<(unsigned)a.rows, 1024, 0, st>>>(a, (T*)y, stats);
    }
    launch_end(K_LN_FWD, st);
    CGB_CUDA(cudaGetLastError());
    return CGB200_OK;
}

// Blocks of the backward kernel (= partial sums) for rows a thread can hold, and threads per block.
struct LnBwdShape {
    bool fits, warp, cluster;
    int nc, threads, grid;
};
// N: values of a 16-byte group; vec: rows start and end on those
static LnBwdShape ln_bwd_shape(int64_t rows, int64_t dim, int N, bool vec) {
    LnBwdShape s{};
    const int64_t chunks = (dim + N - 1) / N;
    s.fits = chunks <= (int64_t)kLnBwdValues / N * kLnBwdMaxThreads;
    s.warp = dim <= 32 * kLnBwdValues;
    if (!s.fits) {
        // column kernel: runs of rows such that about 2048 threads per SM are busy
        const int64_t cols = (dim + 255) / 256;
        s.grid = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(rows, 256), (kNumSM * 8 + cols - 1) / cols));
    } else if (s.warp) {
        s.nc = pow2_at_least(((vec ? chunks : dim) + 31) / 32);
        // up to eight rows a warp of one cluster: a second launch for the sums would take longer than they do
        s.cluster = rows > 0 && rows <= kLnClusterRows;
        s.threads = s.cluster ? 512 : 256;
        s.grid = s.cluster ? (int)std::min<int64_t>(kLnCluster, pow2_at_least((rows + 15) / 16))
                           : (int)std::max<int64_t>(1, std::min<int64_t>((rows + 7) / 8, kNumSM * 4));
    } else {
        s.threads = (int)((chunks + 32 * (kLnBwdValues / N) - 1) / (32 * (kLnBwdValues / N))) * 32;
        const int per_sm = std::max(1, kLnBwdThreadsPerSM / s.threads);
        // a block has eight rows or more, so that its partial sums are a small part of its traffic
        s.grid = (int)std::max<int64_t>(std::min<int64_t>(rows, kNumSM), std::min<int64_t>((rows + 7) / 8, (int64_t)kNumSM * per_sm));
        s.grid = std::max(1, s.grid);
    }
    return s;
}
template <typename T, typename P, int VE, int NC>
static int ln_bwd_launch_nc(const LnBwdShape& s, const LnBwdArgs& a, cudaStream_t st) {
    const size_t smem = (size_t)(s.threads / 32) * 2 * a.dim * sizeof(float);
    auto kern = ln_bwd_kernel<T, P, VE, NC>;
    if (smem > 48 * 1024) CGB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (!s.cluster) {
        kern<<<s.grid, s.threads, smem, st>>>(a);
        return CGB200_OK;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)s.grid);
    cfg.blockDim = dim3((unsigned)s.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)s.grid;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CGB_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
    return CGB200_OK;
}
template <typename T, typename P, int VE>
static int ln_bwd_launch(const LnBwdShape& s, const LnBwdArgs& a, cudaStream_t st) {
#define CGB_LN_BWD(NC_) \
    if constexpr (NC_ * VE <= kLnBwdValues) return ln_bwd_launch_nc<T, P, VE, NC_>(s, a, st);
    switch (s.nc) {
        case 1: CGB_LN_BWD(1) break;
        case 2: CGB_LN_BWD(2) break;
        case 4: CGB_LN_BWD(4) break;
        case 8: CGB_LN_BWD(8) break;
        default: CGB_LN_BWD(16) break;
    }
#undef CGB_LN_BWD
    set_error("internal: layer norm asked for an unsupported row length");
    return CGB200_ERR_UNSUPPORTED;
}

template <typename T, typename P, bool EDGE>
static int ln_bwd_ring(const LnBwdShape& s, const LnBwdArgs& a, cudaStream_t st) {
    constexpr int NC = kLnBwdValues / Chunk<T>::N;
    const size_t slots = (size_t)2 * ring_groups<T>(a.dim, EDGE) * 16;
    const int per_sm = std::max(1, kLnBwdThreadsPerSM / s.threads);
    const int stages = (int)std::max<size_t>(2, std::min<size_t>(kLnRingStages, kLnRingBytes / per_sm / slots));
    const size_t smem = stages * slots;      // two stages hold a block's sums: 8 bytes a column
    auto kern = ln_bwd_ring_kernel<T, P, NC, EDGE>;
    CGB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kern<<<s.grid, s.threads, smem, st>>>(a, stages, kDefaultWaitPolls);
    return CGB200_OK;
}

template <typename T, typename P>
static int ln_bwd(LnBwdArgs a, void* dw, void* db, cudaStream_t st) {
    constexpr int N = Chunk<T>::N;
    auto at16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const bool vec = a.dim % N == 0 && a.x_stride % N == 0 && a.dy_stride % N == 0 && at16(a.x) && at16(a.dy) && at16(a.dx);
    const LnBwdShape s = ln_bwd_shape(a.rows, a.dim, N, vec);
    if (a.rows > 0) {
        if (s.fits) {
            int rc = CGB200_OK;
            if (s.cluster) a.dw = dw, a.db = db, a.part = nullptr;
            launch_begin(K_LN_BWD, st);
            if (vec && s.warp) rc = ln_bwd_launch<T, P, N>(s, a, st);
            else if (s.warp) rc = ln_bwd_launch<T, P, 1>(s, a, st);
            else if (vec) rc = ln_bwd_ring<T, P, false>(s, a, st);
            else rc = ln_bwd_ring<T, P, true>(s, a, st);
            launch_end(K_LN_BWD, st);
            if (rc != CGB200_OK) return rc;
        } else {
            if (a.dx != nullptr) {
                launch_begin(K_LN_BWD, st);
                ln_bwd_long_kernel<T, P><<<(unsigned)a.rows, 1024, 0, st>>>(a);
                launch_end(K_LN_BWD, st);
            }
            if (a.part != nullptr) {
                launch_begin(K_LN_BWD, st);
                ln_bwd_cols_kernel<T><<<dim3((unsigned)((a.dim + 255) / 256), s.grid), 256, 0, st>>>(a, (a.rows + s.grid - 1) / s.grid);
                launch_end(K_LN_BWD, st);
            }
        }
        CGB_CUDA(cudaGetLastError());
    }
    if (a.part != nullptr) {
        launch_begin(K_LN_REDUCE, st);
        ln_param_reduce_kernel<P><<<(unsigned)((2 * a.dim + 31) / 32), dim3(32, 32), 0, st>>>(a.part, a.rows > 0 ? s.grid : 0, a.dim, (P*)dw, (P*)db);
        launch_end(K_LN_REDUCE, st);
        CGB_CUDA(cudaGetLastError());
    }
    return CGB200_OK;
}

}  // namespace cgb200

using namespace cgb200;

#define CGB_LN_TYPES(CALL_)                                                                    \
    do {                                                                                       \
        if (dtype == CGB200_F32) return CALL_(float, float);                                   \
        if (dtype == CGB200_BF16 && param_dtype == CGB200_F32) return CALL_(__nv_bfloat16, float);   \
        if (dtype == CGB200_BF16) return CALL_(__nv_bfloat16, __nv_bfloat16);                  \
        if (param_dtype == CGB200_F32) return CALL_(__half, float);                            \
        return CALL_(__half, __half);                                                          \
    } while (0)

static int ln_check(int64_t rows, int64_t dim, int dtype, int param_dtype) {
    CGB_REQUIRE(rows >= 0 && rows <= 0x7fffffff && dim > 0 && dim <= (1ll << 30), "layer norm: sizes out of range");
    CGB_REQUIRE(dtype >= CGB200_F32 && dtype <= CGB200_F16, "layer norm: unknown type");
    CGB_REQUIRE(param_dtype == dtype || param_dtype == CGB200_F32, "layer norm: weight and bias have the type of x or float32");
    return CGB200_OK;
}

extern "C" {

int cgb200_layer_norm_fwd(const void* x, int64_t x_stride, const void* weight, const void* bias, float eps, void* y, float* stats,
                          int64_t rows, int64_t dim, int dtype, int param_dtype, void* stream) {
    if (int rc = ln_check(rows, dim, dtype, param_dtype)) return rc;
    if (rows == 0) return CGB200_OK;
    CGB_REQUIRE(x != nullptr && y != nullptr, "layer norm: null buffer");
    CGB_REQUIRE(x_stride >= 0 && x_stride <= (1ll << 40), "layer norm: row stride out of range");
    CGB_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0, "layer norm: stats must be 8-byte aligned");
    const LnArgs a{x, x_stride, weight, bias, eps, rows, dim};
    cudaStream_t st = (cudaStream_t)stream;
#define CGB_CALL(T_, P_) ln_fwd<T_, P_>(a, y, (float2*)stats, st)
    CGB_LN_TYPES(CGB_CALL);
#undef CGB_CALL
}

int64_t cgb200_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t dim, int dtype) {
    if (ln_check(rows, dim, dtype, dtype) != CGB200_OK) return -1;
    const int n = dtype == CGB200_F32 ? 4 : 8;
    const LnBwdShape s = ln_bwd_shape(rows, dim, n, false);
    const int parts = s.cluster ? 0 : s.grid;
    return (int64_t)parts * 2 * dim * (int64_t)sizeof(float);
}

int cgb200_layer_norm_bwd(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight, const float* stats,
                          void* dx, void* dweight, void* dbias, int64_t rows, int64_t dim, int dtype, int param_dtype, void* workspace,
                          int64_t workspace_bytes, void* stream) {
    if (int rc = ln_check(rows, dim, dtype, param_dtype)) return rc;
    const bool params = dweight != nullptr || dbias != nullptr;
    if (!params && (dx == nullptr || rows == 0)) return CGB200_OK;
    CGB_REQUIRE(rows == 0 || (x != nullptr && dy != nullptr && stats != nullptr), "layer norm: null buffer");
    CGB_REQUIRE(x_stride >= 0 && x_stride <= (1ll << 40) && dy_stride >= 0 && dy_stride <= (1ll << 40), "layer norm: row stride out of range");
    CGB_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0, "layer norm: stats must be 8-byte aligned");
    if (params) {
        const int64_t need = cgb200_layer_norm_bwd_workspace_bytes(rows, dim, dtype);
        if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
            set_error("workspace too small: need " + std::to_string(need) + " bytes");
            return CGB200_ERR_WORKSPACE;
        }
        CGB_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "workspace must be 16-byte aligned");
    }
    const LnBwdArgs a{x, x_stride, dy, dy_stride, weight, (const float2*)stats, dx, params ? (float*)workspace : nullptr, nullptr, nullptr, rows, dim};
    cudaStream_t st = (cudaStream_t)stream;
#define CGB_CALL(T_, P_) ln_bwd<T_, P_>(a, dweight, dbias, st)
    CGB_LN_TYPES(CGB_CALL);
#undef CGB_CALL
}

}  // extern "C"
