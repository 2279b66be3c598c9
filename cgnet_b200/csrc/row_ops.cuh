// Element access shared by the kernels that walk rows of a (rows, columns) matrix of float32, bfloat16 or float16 values:
// 16-byte chunks that fall on 16-byte boundaries wherever the row starts, and sums over a warp or a block.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cgb200 {

constexpr int kNumSM = 148;   // streaming multiprocessors of a B200

template <typename T>
struct Chunk {
    static constexpr int N = 16 / (int)sizeof(T);   // values of one 16-byte access
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[4], const float*) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[8], const __nv_bfloat16*) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[8], const __half*) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __half2 h;
        memcpy(&h, &w[i], 4);
        const float2 f = __half22float2(h);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack16(const float (&v)[4], const float*) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack16(const float (&v)[8], const __nv_bfloat16*) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack16(const float (&v)[8], const __half*) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Values a row's first chunk lies before the row: chunk c of a row covers its values [c * N - phase, c * N - phase + N), so
// that every chunk starts on a 16-byte boundary whatever the row's own address; values outside [0, n) are never touched.
template <typename T>
__device__ __forceinline__ int row_phase(const T* row) {
    return (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % Chunk<T>::N);
}
// The 16 bytes of the chunk at value e0 (possibly negative) of a row of n values; values outside the row read as `fill`.  Kept apart
// from the conversion to float32, so that a thread's chunks are all on their way before the first is waited for.
//
// The value-by-value forms are kept out of line: inlined they are predicated, not branched around, and a layer norm whose rows are
// all aligned issued 640 instructions a chunk because of them (8192 x 4096 bf16: 92 us).
template <typename T>
__device__ __noinline__ uint4 load_pieces(const T* row, int64_t e0, int64_t n, float fill) {
    constexpr int N = Chunk<T>::N;
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = e0 + i >= 0 && e0 + i < n ? to_f32(row[e0 + i]) : fill;
    return pack16(v, (const T*)nullptr);      // the values came from this type: nothing is rounded
}
template <typename T>
__device__ __noinline__ void store_pieces(T* row, int64_t e0, int64_t n, uint4 u) {
    constexpr int N = Chunk<T>::N;
    T v[N];
    memcpy(v, &u, 16);
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (e0 + i >= 0 && e0 + i < n) row[e0 + i] = v[i];
}
template <typename T>
__device__ __forceinline__ uint4 load_raw(const T* row, int64_t e0, int64_t n, float fill) {
    if (e0 >= 0 && e0 + Chunk<T>::N <= n && aligned16(row + e0)) return *reinterpret_cast<const uint4*>(row + e0);
    return load_pieces(row, e0, n, fill);
}
template <typename T, int N = Chunk<T>::N>
__device__ __forceinline__ void load_chunk(const T* row, int64_t e0, int64_t n, float fill, float (&v)[N]) {
    unpack16(load_raw(row, e0, n, fill), v, (const T*)nullptr);
}
template <typename T, int N = Chunk<T>::N>
__device__ __forceinline__ void store_chunk(T* row, int64_t e0, int64_t n, const float (&v)[N]) {
    if (e0 >= 0 && e0 + N <= n && aligned16(row + e0)) {
        *reinterpret_cast<uint4*>(row + e0) = pack16(v, (const T*)nullptr);
    } else {
        store_pieces(row, e0, n, pack16(v, (const T*)nullptr));
    }
}
// Columns of rows that start anywhere: a thread owns chunk k = values [k N, k N + N) of every row, and moves them with 16-byte
// accesses all the same.  To read them it takes the two aligned groups they lie in and shifts; to write them, each thread puts
// together the aligned group that ends in its chunk, from its neighbour's values and its own.

// 16 bytes from byte `bytes` (0..15, a multiple of 2, the same in the whole warp) of the 32 of lo and hi.
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, int bytes) {
    uint32_t x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 6; ++j) x[j] = bytes & 8 ? x[j + 2] : x[j];
#pragma unroll
    for (int j = 0; j < 5; ++j) x[j] = bytes & 4 ? x[j + 1] : x[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __funnelshift_r(x[j], x[j + 1], (bytes & 2) * 8);
    return make_uint4(x[0], x[1], x[2], x[3]);
}
// Group g of a row of n values whose aligned groups start `ph` values before it; zeros outside the row.  `before`, `behind`: the
// matrix has a row of as many values before and behind this one, so that a group at the row's end may be read whole: what
// it holds of the neighbour is then in the result.
template <typename T>
__device__ __forceinline__ uint4 load_group(const T* row, int ph, int g, int n, bool before = false, bool behind = false) {
    constexpr int N = Chunk<T>::N;
    const int e0 = g * N - ph;
    if ((e0 >= 0 || before) && (e0 + N <= n || (behind && e0 < n))) return *reinterpret_cast<const uint4*>(row + e0);
    if (e0 < n) return load_pieces(row, e0, n, 0.f);
    return make_uint4(0, 0, 0, 0);
}
// Chunk k of such a row.
template <typename T>
__device__ __forceinline__ uint4 load_at(const T* row, int ph, int k, int n, bool before = false, bool behind = false) {
    const uint4 lo = load_group(row, ph, k, n, before, behind);
    if (ph == 0) return lo;
    return shifted(lo, load_group(row, ph, k + 1, n, before, behind), ph * (int)sizeof(T));
}
// The same where both groups are known to be whole.  Kept apart from the form above: behind a branch that may call load_pieces no
// load starts before the one in front of it has been shifted.
template <typename T>
__device__ __forceinline__ uint4 load_inside(const T* row, int ph, int k) {
    const uint4* g = reinterpret_cast<const uint4*>(row - ph) + k;
    return ph == 0 ? g[0] : shifted(g[0], g[1], ph * (int)sizeof(T));
}
// Writes the groups of a row of n values that end in this warp's chunks k0 + lane, k0 + 32 + lane, ... (CH of them, in `u`), `ph` as
// above.  `before` is the last chunk before this warp's (any value where there is none).  The values of the warp's last
// chunk that lie in the group behind it are the next warp's, except at the end of the row.
template <typename T, int CH>
__device__ __forceinline__ void store_groups(T* row, int ph, int k0, int n, const uint4 (&u)[CH], const uint4& before) {
    constexpr int N = Chunk<T>::N;
    const int lane = threadIdx.x & 31;
    uint4 old = before, first = before, last = before;
    int last_e0 = n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e0 = (k0 + 32 * c + lane) * N - ph;      // first value of the group
        uint4 out = u[c];
        if (ph != 0) {
            // lane 31 hands on what it had one step earlier: that is lane 0's neighbour
            const uint4 give = lane == 31 ? old : u[c];
            const int from = (lane + 31) & 31;
            const uint4 prev = make_uint4(__shfl_sync(0xffffffffu, give.x, from), __shfl_sync(0xffffffffu, give.y, from),
                                          __shfl_sync(0xffffffffu, give.z, from), __shfl_sync(0xffffffffu, give.w, from));
            out = shifted(c == 0 && lane == 0 ? before : prev, u[c], (N - ph) * (int)sizeof(T));
            old = u[c];
        }
        if (e0 >= 0 && e0 + N <= n) *reinterpret_cast<uint4*>(row + e0) = out;
        else if (e0 >= 0 && e0 < n) last = out, last_e0 = e0;
        if (c == 0) first = out;
    }
    // the groups at the row's ends, behind the loop: a call in it would keep its steps apart
    const int first_e0 = (k0 + lane) * N - ph;
    if (first_e0 < 0 && first_e0 + N > 0) store_pieces(row, first_e0, n, first);
    if (last_e0 < n) store_pieces(row, last_e0, n, last);
}

// N parameter values (of any of the three types) from value e0 on, as they lie in memory (zeros outside [0, n)), and as float32.
template <typename P, int N>
struct Params {
    static constexpr int W = N * (int)sizeof(P) / 16;
    uint4 u[W];
    __device__ __forceinline__ void load_aligned(const P* w) {
#pragma unroll
        for (int c = 0; c < W; ++c) u[c] = *(reinterpret_cast<const uint4*>(w) + c);
    }
    __device__ __forceinline__ void load(const P* w, int64_t e0, int64_t n) {
        if (e0 >= 0 && e0 + N <= n && aligned16(w + e0)) {
#pragma unroll
            for (int c = 0; c < W; ++c) u[c] = *(reinterpret_cast<const uint4*>(w + e0) + c);
        } else {
#pragma unroll
            for (int c = 0; c < W; ++c) u[c] = load_pieces(w, e0 + c * Chunk<P>::N, n, 0.f);
        }
    }
    // In two steps, so that no call and no wait stands between a thread's loads (w aligned; e0 multiples of N that grow by N from lane to
    // lane): what is whole is fetched at once, and the chunk that the end falls into is put together later from its values, which
    // the lanes have fetched one each (`mine`: value n / N * N + lane).
    __device__ __forceinline__ void load_whole(const P* w, int e0, int n) {
#pragma unroll
        for (int c = 0; c < W; ++c) u[c] = e0 + N <= n ? *(reinterpret_cast<const uint4*>(w + e0) + c) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void place_end(P mine, int e0, int n) {
        float t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = __shfl_sync(0xffffffffu, to_f32(mine), i);
        if (e0 != n / N * N) return;
#pragma unroll
        for (int c = 0; c < W; ++c) {
            float part[Chunk<P>::N];
#pragma unroll
            for (int i = 0; i < Chunk<P>::N; ++i) part[i] = t[c * Chunk<P>::N + i];
            u[c] = pack16(part, (const P*)nullptr);      // of this type already: nothing is rounded
        }
    }
    __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
        for (int c = 0; c < W; ++c) {
            float t[Chunk<P>::N];
            unpack16(u[c], t, (const P*)nullptr);
#pragma unroll
            for (int i = 0; i < Chunk<P>::N; ++i) v[c * Chunk<P>::N + i] = t[i];
        }
    }
};
template <typename P, int N>
__device__ __forceinline__ void load_params(const P* w, int64_t e0, int64_t n, float (&v)[N]) {
    if constexpr (N * sizeof(P) % 16 == 0) {
        Params<P, N> p;
        p.load(w, e0, n);
        p.get(v);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = e0 + i >= 0 && e0 + i < n ? to_f32(w[e0 + i]) : 0.f;
    }
}

// Two float32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum over the block in a fixed order, the same value in every thread.  `buf` holds 32 floats and may be reused by the next
// call only after another barrier: callers alternate between two.
__device__ __forceinline__ float block_sum(float v, float* buf) {
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = (int)(blockDim.x >> 5);
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    return warp_sum(lane < nw ? buf[lane] : 0.f);
}

}  // namespace cgb200
