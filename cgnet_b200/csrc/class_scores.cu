// What a classifier's scores are read for: log probabilities of given classes with entropy and the ranked best classes, and the
// distillation loss against a teacher's best scores; forward and backward.
//
// One pass over a row keeps, per thread, the running reference r (the largest score so far), s = sum 2^a and e = sum 2^a a,
// where a = (z - r) c, c = log2(e) / T.  From the joined (r, s, e) of a row
//     log p(j) = ln 2 ((z_j - r) c - log2 s),     H = ln 2 (log2 s - e / s).
// The difference is taken before the product: scores masked by the type's lowest value would overflow z c.  The backward passes
// read (r, 1 / s): p = 2^((z - r) c) / s carries no rounding of a stored logarithm.  r follows the largest score only when that
// is more than 2^kScMargin ahead: sums and products are in floating point, so a reference a little below the maximum is as exact,
// and almost no chunk after the first has to rescale.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "row_ops.cuh"

namespace cgb200 {

namespace cg = cooperative_groups;

constexpr int kScThreads = 256;
constexpr int kScUnroll = 4;                     // chunks a thread has in flight
constexpr int kScPickKeys = 512;                 // candidates a warp searches in registers
constexpr int kScCap = 2 * kScPickKeys;          // candidates a block keeps: two lists, one is sifted into the other
constexpr int kScChunks = 512;                   // chunks with a score that may rank, noted between two looks at them
constexpr int kScNewKeys = 256;                  // candidates expected between two looks
constexpr int kScMaxTop = 128;
constexpr int kScWarpValues = 32;                // values per lane of the kernel for short rows
constexpr int kScWarpList = 256;                 // classes a warp of it ranks against each other
constexpr float kScMargin = 10.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;
static_assert(kScMaxTop + kScNewKeys <= kScPickKeys * 3 / 4, "candidates between two looks should fit a list");

enum ScoreMode { kLogProbs = 0, kDistill = 1 };

struct ScoreArgs {
    const void* z;
    int64_t z_stride, rows;
    int classes;
    float scale;               // log2(e) / temperature
    float2* stats;             // (r, 1 / s) per row, distillation: (r, 1 / s, tmax, 1 / sum of weights); may be null
    // log probabilities
    const int64_t* targets;    // may be null
    float *log_prob, *entropy;
    int top;
    float* top_lp;
    int64_t* top_ids;
    // distillation
    const int64_t* t_ids;      // [rows][n_t]
    const void* t_scores;      // [rows][n_t]
    int n_t, t_dtype;
    float temperature;
    double inv_temperature;
    float* loss;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Order of the ranked classes as one integer: score, then index downwards.  NaN ranks highest, -0 equals +0.
__device__ __forceinline__ uint32_t order_of(float z) {
    if (z != z) return 0xfffffffeu;        // below the largest integer, which no key may be
    const uint32_t b = __float_as_uint(z + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t o) {
    if (o == 0xfffffffeu) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t key_of(float z, uint32_t idx) { return ((uint64_t)order_of(z) << 32) | (0xffffffffu - idx); }
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// Statistics of a row, or of a part of one, joined: reference, sums relative to it; m is r, or -inf where there is no score yet.
struct Stat {
    float m, r, s, e;
};
// The running form of one thread: sums of even and odd places side by side.
struct RunStat {
    float r, limit, margin;      // a chunk whose largest score is above `limit` moves the reference
    uint64_t s, e;
    __device__ __forceinline__ explicit RunStat(float scale) : r(0.f), limit(-INFINITY), margin(kScMargin / scale), s(0), e(0) {}
    __device__ __forceinline__ void raise(float nm, float scale) {
        if (limit == -INFINITY) {
            const uint64_t zero = pair(0.f, 0.f);
            s = mul2(s, zero), e = mul2(e, zero);      // nothing so far, or a NaN, which stays
        } else {
            const float d = fmaxf((r - nm) * scale, -1e5f), f = ex2(d);
            const uint64_t f2 = pair(f, f);
            e = mul2(f2, fma2(s, pair(d, d), e));
            s = mul2(f2, s);
        }
        r = nm, limit = nm + margin;
    }
    template <int N, bool ENT>
    __device__ __forceinline__ void add(const float (&v)[N], float cm, float scale) {
        if (cm > limit) raise(cm, scale);
        const uint64_t r2 = pair(-r, -r), c2 = pair(scale, scale);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 a = unpair(mul2(add2(pair(v[i], v[i + 1]), r2), c2));
            const uint64_t p = pair(ex2(a.x), ex2(a.y));
            s = add2(s, p);
            if (ENT) e = fma2(p, pair(fmaxf(a.x, -1e5f), fmaxf(a.y, -1e5f)), e);     // p is 0 there: the bound keeps 0 * -inf out
        }
    }
    __device__ __forceinline__ Stat stat() const {
        const float2 a = unpair(s), b = unpair(e);
        return Stat{limit == -INFINITY ? -INFINITY : r, r, a.x + a.y, b.x + b.y};
    }
};
// Joined over a warp, the same bits in every lane: one common reference, each lane's sums rescaled to it once, then added.  A lane
// without a score (m = -inf) has sums of 0, or NaN, which stays.
__device__ __forceinline__ Stat warp_join(Stat a, float scale) {
    float m = a.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float r = m == -INFINITY ? 0.f : m;
    const float d = a.m == -INFINITY ? 0.f : fmaxf((a.r - r) * scale, -1e5f), f = ex2(d);
    return Stat{m, r, warp_sum(a.s * f), warp_sum(f * (a.e + a.s * d))};
}
// Largest value of a chunk, NaN if one is.
__device__ __forceinline__ float chunk_max(const uint4& u, const float*) {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)), max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
}
template <typename T>
__device__ __forceinline__ float chunk_max(const uint4& u, const T*) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type h[4];
    memcpy(h, w, 16);
    const auto m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(to_f32(m.x), to_f32(m.y));
}
// A row of nothing but -inf has no distribution: log probabilities -inf, entropy 0, gradients 0.
__device__ __forceinline__ bool empty_row(const Stat& a) { return a.m == -INFINITY && a.s == 0.f; }
__device__ __forceinline__ float log_prob_of(const Stat& a, double log2_s, float z, float scale) {
    if (empty_row(a)) return -INFINITY;
    return (float)(kLn2 * (((double)z - (double)a.r) * (double)scale - log2_s));
}

__device__ __forceinline__ float load_score(const void* p, int dtype, int64_t i) {
    if (dtype == CGB200_F32) return ((const float*)p)[i];
    if (dtype == CGB200_BF16) return to_f32(((const __nv_bfloat16*)p)[i]);
    return to_f32(((const __half*)p)[i]);
}

// ---- teacher's side of a row ---------------------------------------------------------------------------------------
// Joined over the threads that share a row: a warp (buf unused) or the block.
__device__ __forceinline__ double row_sum_d(double v, double* buf, bool whole_block) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (!whole_block) return v;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) v += buf[i];
    return v;
}
__device__ __forceinline__ float row_max_f(float v, double* buf, bool whole_block) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (!whole_block) return v;
    float* f = (float*)buf;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) f[threadIdx.x >> 5] = v;
    __syncthreads();
    v = f[0];
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) v = fmaxf(v, f[i]);
    return v;
}
// One entry: class (-1: not there, or of weight 0 for lack of a class beyond the last, which `bad` tells), teacher's score and
// student's score.
struct Entry {
    int id;
    bool bad;
    float t, z;
};
template <typename T>
__device__ __forceinline__ Entry entry_of(const ScoreArgs& a, int64_t row, const T* zr, int k) {
    Entry e{-1, false, -INFINITY, 0.f};
    if (k >= a.n_t) return e;
    const int64_t id = a.t_ids[row * a.n_t + k];
    if (id < 0) return e;
    e.t = load_score(a.t_scores, a.t_dtype, row * a.n_t + k);
    e.bad = id >= a.classes;
    if (!e.bad) e.id = (int)id, e.z = to_f32(zr[id]);
    return e;
}
// Weight of an entry before the division by the sum of all: exp((t - tmax) / T).  What the exponent loses when it is rounded to float32,
// up to |exponent| 2^-24, is made good to first order.
__device__ __forceinline__ float weight_of(const ScoreArgs& a, float t, float tmax) {
    const double x = ((double)t - (double)tmax) * a.inv_temperature;
    const float hi = (float)x, w = expf(hi);
    return hi < -200.f ? w : fmaf(w, (float)(x - (double)hi), w);
}
// Loss of a row from its statistics; `first` is this thread's first entry, fetched while the row was read.  Leaves what the
// backward needs of the teacher, (tmax, 1 / sum of weights), 1 / sum = 0 for a row without entries.
template <typename T>
__device__ __forceinline__ float distill_loss(const ScoreArgs& a, int64_t row, const T* zr, const Stat& st, const Entry& first, int t, int G,
                                              double* buf, bool whole_block, float2& teacher) {
    float mx = first.t, some = first.t != -INFINITY || first.bad ? 1.f : 0.f;      // a NaN counts, and a class beyond the last
    for (int k = t + G; k < a.n_t; k += G) {
        const int64_t id = a.t_ids[row * a.n_t + k];
        const float v = id < 0 ? -INFINITY : load_score(a.t_scores, a.t_dtype, row * a.n_t + k);
        if (v != -INFINITY || id >= a.classes) some = 1.f;
        mx = fmaxf(mx, v);
    }
    const bool any = row_max_f(some, buf, whole_block) > 0.f;       // the same in all threads of the row
    if (!any) {
        teacher = make_float2(0.f, 0.f);
        return 0.f;
    }
    const float tmax = row_max_f(mx, buf, whole_block);
    // sum of w, and of w (log w - log p) with log p = ln 2 ((z - r) c - log2 s)
    const double log2_s = log2((double)st.s);
    const bool empty = empty_row(st);
    double sum = 0.0, acc = 0.0;
    Entry e = first;
    for (int k = t;;) {
        if (e.bad) sum += nan("");
        if (e.id >= 0) {
            const float w = weight_of(a, e.t, tmax);
            const double lp = empty ? -INFINITY : kLn2 * (((double)e.z - (double)st.r) * (double)a.scale - log2_s);
            sum += w;
            if (w != 0.f) acc += (double)w * (((double)e.t - (double)tmax) * a.inv_temperature - lp);
        }
        k += G;
        if (k >= a.n_t) break;
        e = entry_of(a, row, zr, k);
    }
    sum = row_sum_d(sum, buf, whole_block);
    acc = row_sum_d(acc, buf, whole_block);
    teacher = make_float2(tmax, (float)(1.0 / sum));
    return (float)((double)a.temperature * (double)a.temperature * (acc / sum - log(sum)));
}

// ---- rows a warp holds in registers --------------------------------------------------------------------------------
// One read of the row and no barrier.  Bound by instructions, of the ranking most of all: 8192 x 1000 bf16 with the 20 best classes
// 43 us, the distillation loss against 20 classes 17 us (the read alone would take 2.5).
template <typename T, int MODE, int CH>
__global__ void __launch_bounds__(kScThreads) scores_warp_kernel(ScoreArgs a) {
    constexpr int N = Chunk<T>::N;
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (kScThreads / 32) + (threadIdx.x >> 5);
    if (row >= a.rows) return;       // whole warps leave; nothing below is wider than a warp
    const T* zr = (const T*)a.z + row * a.z_stride;
    const int ph = row_phase(zr);
    uint4 raw[CH];
    float v[CH][N];
#pragma unroll
    for (int c = 0; c < CH; ++c) raw[c] = load_raw(zr, (lane + 32 * c) * N - ph, a.classes, -INFINITY);
    Entry first{};
    if (MODE == kDistill) first = entry_of(a, row, zr, lane);
    RunStat run(a.scale);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        unpack16(raw[c], v[c], (const T*)nullptr);
        run.add<N, MODE == kLogProbs>(v[c], chunk_max(raw[c], (const T*)nullptr), a.scale);
    }
    const Stat st = warp_join(run.stat(), a.scale);
    if (MODE == kDistill) {
        float2 teacher;
        const float loss = distill_loss(a, row, zr, st, first, lane, 32, nullptr, false, teacher);
        if (lane == 0) {
            a.loss[row] = loss;
            if (a.stats != nullptr) ((float4*)a.stats)[row] = make_float4(st.r, empty_row(st) ? 0.f : 1.f / st.s, teacher.x, teacher.y);
        }
        return;
    }
    if (a.stats != nullptr && lane == 0) a.stats[row] = make_float2(st.r, empty_row(st) ? 0.f : 1.f / st.s);
    const double log2_s = log2((double)st.s);
    if (lane == 0) {
        a.entropy[row] = empty_row(st) ? 0.f : (float)(kLn2 * (log2_s - (double)st.e / (double)st.s));
        if (a.targets != nullptr) {
            const int64_t t = a.targets[row];
            a.log_prob[row] = t < 0 ? 0.f : t >= a.classes ? __uint_as_float(0x7fffffffu) : log_prob_of(st, log2_s, to_f32(zr[t]), a.scale);
        }
    }
    if (a.top == 0) return;
    uint32_t order[CH][N];             // 0 beyond the row
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = (lane + 32 * c) * N - ph + i;
            order[c][i] = e >= 0 && e < a.classes ? order_of(v[c][i]) : 0u;
        }
    auto leave = [&](int k, uint64_t key) {
        a.top_ids[row * a.top + k] = index_of(key);
        a.top_lp[row * a.top + k] = log_prob_of(st, log2_s, score_of((uint32_t)(key >> 32)), a.scale);
    };
    if (a.top > 2) {
        // the top-th highest order, in its upper 16 bits; the classes from there on go to a list and are counted against each
        // other.  (Picking the best of all lanes `top` times over took a microsecond for each.)
        __shared__ uint64_t lists[kScThreads / 32][kScWarpList];
        uint64_t* list = lists[threadIdx.x >> 5];
        uint32_t t = 0;
        for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
            int n = 0;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < N; ++i) n += order[c][i] >= (t | bit);
            if (__reduce_add_sync(0xffffffffu, n) >= a.top) t |= bit;
        }
        int n = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool in = order[c][i] >= t && order[c][i] != 0;
                const unsigned votes = __ballot_sync(0xffffffffu, in);
                const int at = n + __popc(votes & ((1u << lane) - 1u));
                if (in && at < kScWarpList) list[at] = ((uint64_t)order[c][i] << 32) | (0xffffffffu - (uint32_t)((lane + 32 * c) * N - ph + i));
                n += __popc(votes);
            }
        if (n <= kScWarpList) {
            __syncwarp();
            for (int i = lane; i < n; i += 32) {
                const uint64_t key = list[i];
                int rank = 0;
                for (int j = 0; j < n; ++j) rank += list[j] > key;
                if (rank < a.top) leave(rank, key);
            }
            return;
        }
    }
    // one or two classes, or many of one score: the best of each lane, and the best of those, `top` times over
    uint64_t last = ~0ull, best = 0;
    for (int k = 0; k < a.top; ++k) {
        if (k == 0 || best == last) {       // this lane's best is not known, or was the one just taken
            best = 0;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint64_t key = ((uint64_t)order[c][i] << 32) | (0xffffffffu - (uint32_t)((lane + 32 * c) * N - ph + i));
                    if (order[c][i] != 0 && key < last && key > best) best = key;
                }
        }
        const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
        const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
        last = ((uint64_t)hi << 32) | lo;
        if (lane == 0) leave(k, last);
    }
}

// ---- long rows: a block, or a cluster of blocks, per row -------------------------------------------------------------
struct ScoreBase {
    Stat part[kScThreads / 32];
    Stat stat;
    double red[kScThreads / 32];
};
struct ScoreShared : ScoreBase {
    uint64_t buf[kScCap];          // candidates
    uint64_t best[kScMaxTop];      // this block's best, in order
    unsigned hist[256];
    int count, kept, n_best, chunks;
    int chunk[kScChunks];          // chunks with a score that may rank
    uint64_t prefix;
    unsigned want;
};

// A chunk with a score that may rank: only its number is noted in the loop over the row, by what is usually one lane of a warp;
// its scores are looked at afterwards, chunk by thread (expand_chunks).  Doing that in the loop took half of its instructions.
__device__ __forceinline__ void note_chunk(ScoreShared& sh, int c) {
    const int at = atomicAdd(&sh.chunks, 1);
    if (at < kScChunks) sh.chunk[at] = c;
}
// Largest t, in its upper 16 bits, that at least k of n <= kScPickKeys orders in shared memory (`step` words apart) reach; by the block's
// first warp, 16 halvings on registers.  0 where n < k.
__device__ __forceinline__ uint32_t kth_order(const uint32_t* v, int step, int n, int k) {
    uint32_t own[kScPickKeys / 32];
#pragma unroll
    for (int j = 0; j < kScPickKeys / 32; ++j) {
        const int i = threadIdx.x + 32 * j;
        own[j] = i < n ? v[i * step] : 0u;
    }
    uint32_t t = 0;
    const int groups = (n + 31) / 32;
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < kScPickKeys / 32; ++j)
            if (j < groups) c += own[j] >= (t | bit);
        if (__reduce_add_sync(0xffffffffu, c) >= k) t |= bit;
    }
    return t;
}
__device__ __forceinline__ void push(ScoreShared& sh, uint64_t key) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kScCap) sh.buf[at] = key;
}
// The scores of the noted chunks from thr on become candidates.  False where either did not fit: the row is then searched
// by radix_collect.  Ends behind a barrier; sh.count is the number of candidates.
template <typename T>
__device__ __forceinline__ bool expand_chunks(ScoreShared& sh, const T* zr, int ph, int classes, float thr) {
    constexpr int N = Chunk<T>::N;
    __syncthreads();
    const int n = sh.chunks;
    for (int i = threadIdx.x; i < min(n, kScChunks); i += kScThreads) {
        const int e0 = sh.chunk[i] * N - ph;
        float v[N];
        load_chunk(zr, e0, classes, -INFINITY, v);
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (!(v[j] < thr) && v[j] != -INFINITY) push(sh, key_of(v[j], (uint32_t)(e0 + j)));
    }
    __syncthreads();
    return n <= kScChunks && sh.count <= kScCap;
}
// Of n <= kScPickKeys candidates those whose order is at least the k-th highest's (in its upper 16 bits), which is returned:
// moved to the list's second half, sh.kept of them.  Ends behind a barrier.
__device__ __forceinline__ uint32_t sift(ScoreShared& sh, int n, int k) {
    if (threadIdx.x < 32) {
        const uint32_t t = kth_order((const uint32_t*)sh.buf + 1, 2, n, k);
        if (threadIdx.x == 0) sh.want = t, sh.kept = 0;
    }
    __syncthreads();
    const uint32_t t = sh.want;
    for (int i = threadIdx.x; i < n; i += kScThreads)
        if ((uint32_t)(sh.buf[i] >> 32) >= t) sh.buf[kScPickKeys + atomicAdd(&sh.kept, 1)] = sh.buf[i];
    __syncthreads();
    return t;
}
// The `k` highest of the first n candidates, in order, to sh.best (n_best of them).  All keys differ, so their order
// does not depend on the order in which they were collected.
__device__ void select_best(ScoreShared& sh, int n, int k) {
    if (n <= kScPickKeys) {
        const uint64_t* keys = sh.buf;
        int m = n;
        if (n > 64 && n > k) {
            sift(sh, n, k);
            keys = sh.buf + kScPickKeys;
            m = sh.kept;
        }
        for (int i = threadIdx.x; i < m; i += kScThreads) {
            const uint64_t key = keys[i];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < m; ++j) rank += keys[j] > key;
            if (rank < k) sh.best[rank] = key;
        }
    } else {
        for (int i = n + threadIdx.x; i < kScCap; i += kScThreads) sh.buf[i] = 0;
        for (int size = 2; size <= kScCap; size *= 2)
            for (int d = size / 2; d > 0; d /= 2) {
                __syncthreads();
                for (int i = threadIdx.x; i < kScCap / 2; i += kScThreads) {
                    const int lo = 2 * i - (i & (d - 1)), hi = lo + d;
                    const uint64_t x = sh.buf[lo], y = sh.buf[hi];
                    if ((x < y) == ((lo & size) == 0)) sh.buf[lo] = y, sh.buf[hi] = x;    // descending
                }
            }
        __syncthreads();
        for (int i = threadIdx.x; i < k && i < n; i += kScThreads) sh.best[i] = sh.buf[i];
    }
    if (threadIdx.x == 0) sh.n_best = min(n, k);
    __syncthreads();
}

__device__ __forceinline__ float threshold_of(uint32_t order) { return order <= order_of(-INFINITY) ? -INFINITY : score_of(order); }

// Too many candidates (long runs of equal or rising scores): the k-th highest key by radix, most significant byte first, until
// what lies above the byte found fits the candidates.  Keys differ, so eight bytes always do.
template <typename T>
__device__ void radix_collect(ScoreShared& sh, const T* zr, int ph, int c0, int c1, int classes, int k) {
    constexpr int N = Chunk<T>::N;
    __syncthreads();
    if (threadIdx.x == 0) sh.prefix = 0, sh.want = (unsigned)k;
    int shift = 56;
    for (;; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kScThreads) sh.hist[i] = 0;
        __syncthreads();
        const uint64_t prefix = sh.prefix;
        for (int c = c0 + (int)threadIdx.x; c < c1; c += kScThreads) {
            float v[N];
            load_chunk(zr, (int64_t)c * N - ph, classes, 0.f, v);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t e = (int64_t)c * N - ph + i;
                if (e < 0 || e >= classes) continue;
                const uint64_t key = key_of(v[i], (uint32_t)e);
                if (shift == 56 || (key >> (shift + 8)) == prefix) atomicAdd(&sh.hist[(key >> shift) & 255], 1u);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned above = 0;
            int d = 255;
            while (d > 0 && above + sh.hist[d] < sh.want) above += sh.hist[d--];
            sh.prefix = (prefix << 8) | (unsigned)d;
            sh.want -= above;                    // of the keys with this prefix
            sh.count = (int)sh.hist[d] + k - (int)sh.want;     // keys at or above the prefix
        }
        __syncthreads();
        const int n = sh.count;
        __syncthreads();
        if (n <= kScCap || shift == 0) break;
    }
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    const uint64_t prefix = sh.prefix;
    for (int c = c0 + (int)threadIdx.x; c < c1; c += kScThreads) {
        float v[N];
        load_chunk(zr, (int64_t)c * N - ph, classes, 0.f, v);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t e = (int64_t)c * N - ph + i;
            if (e < 0 || e >= classes) continue;
            const uint64_t key = key_of(v[i], (uint32_t)e);
            if ((key >> shift) >= prefix) push(sh, key);
        }
    }
    __syncthreads();
}

// A row per block, or per cluster of blocks where there are too few rows to fill the GPU.  One read of the scores: 2048 x 65536 bf16
// (268 MB) 57 us without ranking = 4.7 TB/s, 82 with the 20 best classes, whose looks at the candidates stop the block's stream;
// one row of 131072 12.6 us, which is the latency of its phases.
template <typename T, int MODE, bool CLUSTER>
__global__ void __launch_bounds__(kScThreads, MODE == kDistill ? 6 : 5) scores_row_kernel(ScoreArgs a, int blocks_per_row) {
    constexpr int N = Chunk<T>::N;
    constexpr bool ENT = MODE == kLogProbs;
    constexpr int kTile = kScThreads * kScUnroll;
    __shared__ typename std::conditional<ENT, ScoreShared, ScoreBase>::type sh;
    const int part = CLUSTER ? (int)(blockIdx.x % (unsigned)blocks_per_row) : 0;
    const int64_t row = CLUSTER ? (int64_t)(blockIdx.x / (unsigned)blocks_per_row) : (int64_t)blockIdx.x;
    const T* zr = (const T*)a.z + row * a.z_stride;
    const int ph = row_phase(zr);
    const int nc = (a.classes + ph + N - 1) / N;
    const int per = CLUSTER ? (nc + blocks_per_row - 1) / blocks_per_row : nc;
    const int c0 = min(nc, part * per), c1 = min(nc, c0 + per);
    const int first = max(0, c0 * N - ph), behind = min(a.classes, c1 * N - ph);   // this block's classes
    const bool tops = ENT && a.top > 0;
    const int want = tops ? min(a.top, max(0, behind - first)) : 0;      // entries it has to offer
    if constexpr (ENT) {
        if (threadIdx.x == 0) sh.count = 0, sh.chunks = 0;
    }
    RunStat run(a.scale);
    float thr = -INFINITY;
    // a row of random scores adds `top` candidates whenever what has been read of it doubles
    const int grow = tops ? 1 + kScNewKeys / a.top : 1;
    bool fits = true;
    // Chunks [f0, f1) lie inside the row; what is left at its two ends is one chunk each.
    const int f0 = c0 == 0 && ph > 0 ? 1 : c0, f1 = max(f0, min(c1, (a.classes + ph) / N));
    const uint4* src = reinterpret_cast<const uint4*>(zr - ph) + f0 + threadIdx.x;
    const uint4 none = load_raw(zr, 0, 0, -INFINITY);
    Entry entry{};
    if (!ENT && part == 0) entry = entry_of(a, row, zr, (int)threadIdx.x);
    int look = f0 + kTile * (grow - 1);       // chunk behind which the candidates are looked at
    for (int base = f0; base < f1; base += kTile) {
        uint4 raw[kScUnroll];
        if (base + kTile <= f1) {
#pragma unroll
            for (int u = 0; u < kScUnroll; ++u) raw[u] = src[u * kScThreads];
        } else {
#pragma unroll
            for (int u = 0; u < kScUnroll; ++u) raw[u] = base + u * kScThreads + (int)threadIdx.x < f1 ? src[u * kScThreads] : none;
        }
        src += kTile;
        float cms[kScUnroll];
#pragma unroll
        for (int u = 0; u < kScUnroll; ++u) {
            float v[N];
            unpack16(raw[u], v, (const T*)nullptr);
            const float cm = chunk_max(raw[u], (const T*)nullptr);
            run.add<N, ENT>(v, cm, a.scale);
            if constexpr (ENT) {
                cms[u] = cm;
                if (tops && base != f0 && !(cm <= thr)) note_chunk(sh, base + u * kScThreads + (int)threadIdx.x);
            }
        }
        if constexpr (ENT) {
            if (tops && base == f0) {
                // Threshold: the largest value (to the upper 16 bits of its order) that at least `top` chunks of the first tile reach:
                // nothing below it can rank, and nothing equal to it further right.  Chunk maxima are counted per pair of chunks.
                uint32_t* maxima = (uint32_t*)sh.buf;
#pragma unroll
                for (int u = 0; u < kScUnroll; u += 2)
                    maxima[u / 2 * kScThreads + threadIdx.x] = order_of(cms[u] > cms[u + 1] || !(cms[u + 1] == cms[u + 1]) ? cms[u] : cms[u + 1]);
                __syncthreads();
                if (threadIdx.x < 32) {
                    const uint32_t t = kth_order(maxima, 1, kScThreads * kScUnroll / 2, a.top);
                    if (threadIdx.x == 0) sh.want = t;
                }
                __syncthreads();
                thr = threshold_of(sh.want);
#pragma unroll
                for (int u = 0; u < kScUnroll; ++u)
                    if (!(cms[u] < thr) && cms[u] != -INFINITY) note_chunk(sh, base + u * kScThreads + (int)threadIdx.x);
            } else if (tops && base >= look) {
                // about as many candidates as a list holds by now: sift them, and raise the threshold to the k-th of them
                fits = expand_chunks(sh, zr, ph, a.classes, thr) && sh.count <= kScPickKeys && fits;
                const int n = sh.count;
                if (fits && n > a.top) {
                    thr = fmaxf(thr, threshold_of(sift(sh, n, a.top)));
                    const int kept = sh.kept;
                    for (int i = threadIdx.x; i < min(kept, kScPickKeys); i += kScThreads) sh.buf[i] = sh.buf[kScPickKeys + i];
                    if (threadIdx.x == 0) sh.count = kept;
                }
                if (threadIdx.x == 0) sh.chunks = 0;
                look = f0 + (int)min((int64_t)(base - f0 + kTile) * grow, (int64_t)1 << 30) - kTile;
                __syncthreads();
            }
        }
    }
    if (threadIdx.x < 2) {
        // the ends: thread 0 the first chunk, thread 1 the last
        const int c = threadIdx.x == 0 ? c0 : f1;
        if (threadIdx.x == 0 ? c0 < f0 : f1 < c1) {
            const uint4 end = load_raw(zr, (int64_t)c * N - ph, a.classes, -INFINITY);
            float v[N];
            unpack16(end, v, (const T*)nullptr);
            run.add<N, ENT>(v, chunk_max(end, (const T*)nullptr), a.scale);
            if constexpr (ENT) {
                if (tops) note_chunk(sh, c);
            }
        }
    }
    Stat st = run.stat();
    st = warp_join(st, a.scale);
    if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = st;
    __syncthreads();
    if (threadIdx.x < 32) {
        st = warp_join(threadIdx.x < kScThreads / 32 ? sh.part[threadIdx.x] : Stat{-INFINITY, 0.f, 0.f, 0.f}, a.scale);
        if (threadIdx.x == 0) sh.stat = st;
    }
    if constexpr (ENT) {
        if (tops) {
            fits = expand_chunks(sh, zr, ph, a.classes, thr) && fits;
            int n = sh.count;
            if (!fits) {
                radix_collect(sh, zr, ph, c0, c1, a.classes, want);
                n = sh.count;
            } else if (n < want) {
                // fewer scores than places: masked classes follow, lowest index first
                if (threadIdx.x < 32) {
                    int have = n;
                    for (int e = first; e < behind && have < want; e += 32) {
                        const int at = e + (int)threadIdx.x;
                        const bool masked = at < behind && to_f32(zr[at]) == -INFINITY;
                        const unsigned votes = __ballot_sync(0xffffffffu, masked);
                        const int place = have + __popc(votes & ((1u << threadIdx.x) - 1u));
                        if (masked && place < want) sh.buf[place] = key_of(-INFINITY, (uint32_t)at);
                        have += __popc(votes);
                    }
                }
                n = want;
                __syncthreads();
            }
            select_best(sh, n, want);
        }
    }
    if (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (part == 0) {
            if (threadIdx.x < 32) {
                Stat mine = (int)threadIdx.x < blocks_per_row ? cluster.map_shared_rank(&sh, (int)threadIdx.x)->stat : Stat{-INFINITY, 0.f, 0.f, 0.f};
                mine = warp_join(mine, a.scale);
                if (threadIdx.x == 0) sh.part[0] = mine;       // sh.stat is still being read
            }
            if constexpr (ENT) {
                if (tops) {
                    // the blocks' lists, as many at a time as fit beside the best so far
                    const int lists = kScCap / a.top - 1;
                    for (int p0 = 0; p0 < blocks_per_row; p0 += lists) {
                        if (threadIdx.x == 0) sh.count = 0;
                        __syncthreads();
                        for (int i = threadIdx.x; i < min(lists, blocks_per_row - p0) * a.top; i += kScThreads) {
                            const ScoreShared* o = cluster.map_shared_rank(&sh, p0 + i / a.top);
                            if (i % a.top < o->n_best) push(sh, o->best[i % a.top]);
                        }
                        if (p0 > 0 && (int)threadIdx.x < sh.n_best) push(sh, sh.best[threadIdx.x]);
                        __syncthreads();
                        const int n = sh.count;
                        __syncthreads();          // the lists, this block's own among them, have been read
                        select_best(sh, n, a.top);
                    }
                }
            }
            __syncthreads();
            st = sh.part[0];
        }
        cluster.sync();                   // no block leaves while its part is read
        if (part != 0) return;
    } else {
        __syncthreads();
        st = sh.stat;
    }
    if constexpr (!ENT) {
        // few entries are the first warp's work, the other warps are done
        const bool whole = a.n_t > 128;
        if (!whole && threadIdx.x >= 32) return;
        float2 teacher;
        const float loss = distill_loss(a, row, zr, st, entry, (int)threadIdx.x, whole ? kScThreads : 32, sh.red, whole, teacher);
        if (threadIdx.x == 0) {
            a.loss[row] = loss;
            if (a.stats != nullptr) ((float4*)a.stats)[row] = make_float4(st.r, empty_row(st) ? 0.f : 1.f / st.s, teacher.x, teacher.y);
        }
    } else {
        const double log2_s = log2((double)st.s);
        if (threadIdx.x == 0) {
            if (a.stats != nullptr) a.stats[row] = make_float2(st.r, empty_row(st) ? 0.f : 1.f / st.s);
            a.entropy[row] = empty_row(st) ? 0.f : (float)(kLn2 * (log2_s - (double)st.e / (double)st.s));
            if (a.targets != nullptr) {
                const int64_t t = a.targets[row];
                a.log_prob[row] = t < 0 ? 0.f : t >= a.classes ? __uint_as_float(0x7fffffffu) : log_prob_of(st, log2_s, to_f32(zr[t]), a.scale);
            }
        }
        for (int k = threadIdx.x; k < a.top; k += kScThreads) {
            const uint64_t key = sh.best[k];
            a.top_ids[row * a.top + k] = index_of(key);
            a.top_lp[row * a.top + k] = log_prob_of(st, log2_s, score_of((uint32_t)(key >> 32)), a.scale);
        }
    }
}

// ---- gradients with respect to the scores --------------------------------------------------------------------------
struct ScoreGradArgs {
    ScoreArgs f;
    void* dz;
    const float *g_lp, *g_ent, *g_loss;    // per row; g_lp or g_ent may be null
};

// Chunks [c_begin, c_end) of a row, dealt out to `step` threads, through `f` to the same places of another row.  f(e0, v, j) gets the
// first class of a chunk and the chunk's number among those that lie inside the row, counted from the block's first (-1 for
// the ones at the row's ends).  Five blocks of these loops per SM keep enough loads in flight; fetching the next chunks ahead in
// registers instead cost a block and was slower (201 against 190 us at 4096 x 50000 bf16).
template <typename T, typename F>
__device__ __forceinline__ void stream_chunks(const T* zr, T* dr, int n, int ph, int c_begin, int c_end, int t, int step, F f) {
    constexpr int N = Chunk<T>::N;
    float v[N];
    const int f0 = c_begin == 0 && ph > 0 ? 1 : c_begin, f1 = max(f0, min(c_end, (n + ph) / N)), inner = f1 - f0;
    const uint4* src = reinterpret_cast<const uint4*>(zr - ph) + f0;
    int j = t;
    if (aligned16(dr - ph)) {
        uint4* dst = reinterpret_cast<uint4*>(dr - ph) + f0;
        for (; j + (kScUnroll - 1) * step < inner; j += kScUnroll * step) {
            uint4 raw[kScUnroll];
#pragma unroll
            for (int u = 0; u < kScUnroll; ++u) raw[u] = src[j + u * step];
#pragma unroll
            for (int u = 0; u < kScUnroll; ++u) {
                unpack16(raw[u], v, (const T*)nullptr);
                f((f0 + j + u * step) * N - ph, v, j + u * step);
                dst[j + u * step] = pack16(v, (const T*)nullptr);
            }
        }
    }
    for (; j < inner; j += step) {
        unpack16(src[j], v, (const T*)nullptr);
        f((f0 + j) * N - ph, v, j);
        store_chunk(dr, (f0 + j) * N - ph, n, v);
    }
    if (t < 2 && (t == 0 ? c_begin < f0 : f1 < c_end)) {
        const int e0 = (t == 0 ? c_begin : f1) * N - ph;
        load_chunk(zr, e0, n, 0.f, v);
        f(e0, v, -1);
        store_chunk(dr, e0, n, v);
    }
}

// kScThreads / G rows of a block, G threads a row and `run` chunks of it per block.  log_probs:
//     dz_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)
// distillation:  dz_j = g T (p_j - sum_k q_k 1[id_k = j]).  The named classes are sorted first, with the place in that order where
// each run of 32 chunks begins, so that a warp knows the few entries of its chunks; writing them in a second step behind a
// barrier took a third as long again (190 against 141 us of streaming at 4096 x 50000 bf16, 819 MB: 5.8 TB/s).
template <typename T, int MODE>
__global__ void __launch_bounds__(kScThreads, 5) scores_grad_kernel(ScoreGradArgs a, int G, int run, int runs) {
    constexpr int N = Chunk<T>::N;
    extern __shared__ int dyn[];
    const int t = (int)threadIdx.x % G, sub = (int)threadIdx.x / G, rows_here = kScThreads / G;
    const int64_t row = (int64_t)(blockIdx.x / (unsigned)runs) * rows_here + sub;
    const bool on = row < a.f.rows;
    const int c_begin = (int)(blockIdx.x % (unsigned)runs) * run;
    const T* zr = (const T*)a.f.z + (on ? row : 0) * a.f.z_stride;
    T* dr = (T*)a.dz + (on ? row : 0) * a.f.classes;
    const int V = a.f.classes, ph = row_phase(zr);
    const float scale = a.f.scale;
    const int c_end = min(c_begin + run, (V + ph + N - 1) / N);
    if constexpr (MODE == kLogProbs) {
        if (!on) return;
        const float2 st = a.f.stats[row];
        const int64_t tgt = a.f.targets != nullptr ? a.f.targets[row] : -1;
        const bool dead = st.y == 0.f;                                          // a row without a distribution
        float g_lp = a.g_lp != nullptr && tgt >= 0 && !dead ? a.g_lp[row] : 0.f;
        if (tgt >= V && a.g_lp != nullptr) g_lp = __uint_as_float(0x7fffffffu);      // the entropy's gradient does not know the target
        const float g_ent = a.g_ent != nullptr && !dead ? a.g_ent[row] : 0.f;
        // -p (g_lp + g_H (ln 2 a + log(1 / s) + H)),  p = 2^a / s
        const float base = g_ent == 0.f ? g_lp : g_lp + g_ent * (logf(st.y) + a.f.entropy[row]), slope = g_ent * (float)kLn2;
        const int at = tgt >= V ? -1 : (int)tgt;
        stream_chunks(zr, dr, V, ph, c_begin, c_end, t, G, [&](int e0, float (&v)[N], int) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float y = (v[i] - st.x) * scale;
                v[i] = dead ? 0.f : -(ex2(y) * st.y) * fmaf(slope, fmaxf(y, -1e5f), base);
            }
            if (at >= e0 && at < e0 + N) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (e0 + i == at) v[i] += g_lp;
            }
        });
        return;
    }
    const int K = a.f.n_t, groups = (run + 31) / 32 + 1;
    int* named = dyn + sub * (3 * K + groups);           // as given, -1 for an entry that is not there
    int* ids = named + K;                                // in order
    float* wts = (float*)(ids + K);
    int* start = (int*)(wts + K);
    const float4 st = on ? ((const float4*)a.f.stats)[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    // a class beyond the last, or a NaN among the teacher's scores, left its sum NaN: then so is the whole row's gradient, as its loss
    const bool unknown = st.w != st.w;
    const bool dead = !unknown && (st.y == 0.f || st.w == 0.f);       // no row, no distribution, or no teacher
    const float g = dead ? 0.f : a.g_loss[row] * a.f.temperature, gp = unknown ? __uint_as_float(0x7fffffffu) : g * st.y;
    if (!dead)
        for (int k = t; k < K; k += G) {
            const int64_t id = a.f.t_ids[row * K + k];
            named[k] = id >= 0 && id < V ? (int)id : -1;
        }
    __syncthreads();
    if (!dead)
        for (int k = t; k < K; k += G) {
            const int id = named[k];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < K; ++j) rank += named[j] < id || (named[j] == id && j < k);
            ids[rank] = id;
            wts[rank] = id < 0 ? 0.f : g * (weight_of(a.f, load_score(a.f.t_scores, a.f.t_dtype, row * K + k), st.z) * st.w);
        }
    __syncthreads();
    if (!dead) {
        const int first = (c_begin == 0 && ph > 0 ? 1 : c_begin) * N - ph;
        for (int i = t; i < groups; i += G) {
            const int from = first + i * 32 * N;         // entries below this class lie before group i
            int lo = 0, hi = K;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (ids[mid] < from) lo = mid + 1;
                else hi = mid;
            }
            start[i] = lo;
        }
    }
    __syncthreads();
    if (!on) return;
    stream_chunks(zr, dr, V, ph, c_begin, c_end, t, G, [&](int e0, float (&v)[N], int j) {
        if (dead) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = 0.f;
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = gp * ex2((v[i] - st.x) * scale);
        const int k1 = j < 0 ? K : start[j / 32 + 1];
        for (int k = j < 0 ? 0 : start[j / 32]; k < k1; ++k) {
            const int at = ids[k] - e0;
            if (at >= 0 && at < N) {
                const float w = wts[k];
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i == at) v[i] -= w;
            }
        }
    });
}

// ---- launches ------------------------------------------------------------------------------------------------------
template <typename T, int MODE>
static int scores_fwd(const ScoreArgs& a, cudaStream_t st) {
    constexpr int N = Chunk<T>::N;
    const int kid = MODE == kLogProbs ? K_LOGP_FWD : K_DISTILL_FWD;
    const int64_t chunks = ((int64_t)a.classes + 2 * N - 2) / N;     // with any phase
    constexpr int CHW = kScWarpValues / N;
    if (chunks <= 32 * CHW) {
        const unsigned grid = (unsigned)((a.rows + kScThreads / 32 - 1) / (kScThreads / 32));
        launch_begin(kid, st);
        if (chunks <= 32) scores_warp_kernel<T, MODE, 1><<<grid, kScThreads, 0, st>>>(a);
        else scores_warp_kernel<T, MODE, CHW><<<grid, kScThreads, 0, st>>>(a);
        launch_end(kid, st);
        CGB_CUDA(cudaGetLastError());
        return CGB200_OK;
    }
    // few rows: up to 16 blocks share one, as long as each has a whole tile of it
    int c = 1;
    while (c < 16 && a.rows * c * 2 <= 2 * kNumSM && chunks >= (int64_t)2 * c * kScThreads * kScUnroll) c *= 2;
    if (c == 1) {
        launch_begin(kid, st);
        scores_row_kernel<T, MODE, false><<<(unsigned)a.rows, kScThreads, 0, st>>>(a, 1);
        launch_end(kid, st);
        CGB_CUDA(cudaGetLastError());
        return CGB200_OK;
    }
    auto kern = scores_row_kernel<T, MODE, true>;
    if (c > 8) CGB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.rows * c));
    cfg.blockDim = dim3(kScThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)c;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    launch_begin(kid, st);
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, kern, a, c);
    launch_end(kid, st);
    CGB_CUDA(rc);
    return CGB200_OK;
}

template <typename T, int MODE>
static int scores_bwd(const ScoreGradArgs& a, cudaStream_t st) {
    constexpr int N = Chunk<T>::N;
    const int kid = MODE == kLogProbs ? K_LOGP_BWD : K_DISTILL_BWD;
    const int64_t chunks = ((int64_t)a.f.classes + 2 * N - 2) / N;
    int G = 32;
    while (G < kScThreads && G * kScUnroll < chunks) G *= 2;
    // whole rows, or parts of them where the rows alone would not keep the SMs busy
    const int64_t groups = (a.f.rows + kScThreads / G - 1) / (kScThreads / G), tile = (int64_t)G * kScUnroll;
    const int64_t tiles = (chunks + tile - 1) / tile;
    const int64_t cut = std::max<int64_t>(1, std::min(tiles, (kNumSM * 8 + groups - 1) / groups));
    const int run = (int)std::min<int64_t>((tiles + cut - 1) / cut * tile, 1 << 15);      // bounds the table of starts
    const int runs = (int)((chunks + run - 1) / run);
    const int64_t blocks = (a.f.rows + kScThreads / G - 1) / (kScThreads / G) * runs;
    CGB_REQUIRE(blocks <= 0x7fffffff, "class scores: too many blocks for one launch");
    const size_t smem = MODE == kDistill ? (size_t)(kScThreads / G) * (3 * a.f.n_t + (run + 31) / 32 + 1) * sizeof(int) : 0;
    auto kern = scores_grad_kernel<T, MODE>;
    if (smem > 48 * 1024) CGB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    launch_begin(kid, st);
    kern<<<(unsigned)blocks, kScThreads, smem, st>>>(a, G, run, runs);
    launch_end(kid, st);
    CGB_CUDA(cudaGetLastError());
    return CGB200_OK;
}

static int score_check(const void* z, int64_t z_stride, int64_t rows, int64_t classes, int dtype) {
    CGB_REQUIRE(rows >= 0 && rows <= (1ll << 26) && classes > 0 && classes <= (1ll << 30), "class scores: sizes out of range");
    CGB_REQUIRE(dtype >= CGB200_F32 && dtype <= CGB200_F16, "class scores: unknown type");
    CGB_REQUIRE(rows == 0 || z != nullptr, "class scores: null buffer");
    CGB_REQUIRE(z_stride >= 0 && z_stride <= (1ll << 40), "class scores: row stride out of range");
    return CGB200_OK;
}
static int teacher_check(const int64_t* ids, const void* scores, int64_t n_t, int t_dtype, float temperature) {
    CGB_REQUIRE(n_t > 0 && n_t <= CGB200_MAX_TEACHER, "distillation: between 1 and 1024 teacher entries a row");
    CGB_REQUIRE(t_dtype >= CGB200_F32 && t_dtype <= CGB200_F16, "distillation: unknown type of the teacher's scores");
    CGB_REQUIRE(ids != nullptr && scores != nullptr, "distillation: null buffer");
    CGB_REQUIRE(temperature >= 1e-3f && temperature <= 1e3f, "distillation: temperature out of range (0.001 to 1000)");
    return CGB200_OK;
}

}  // namespace cgb200

using namespace cgb200;

#define CGB_SCORE_TYPES(FN_, MODE_, ...)                                   \
    do {                                                                   \
        if (dtype == CGB200_F32) return FN_<float, MODE_>(__VA_ARGS__);    \
        if (dtype == CGB200_BF16) return FN_<__nv_bfloat16, MODE_>(__VA_ARGS__); \
        return FN_<__half, MODE_>(__VA_ARGS__);                            \
    } while (0)

extern "C" {

int cgb200_log_probs_fwd(const void* logits, int64_t stride, const int64_t* targets, int top, float* log_prob, float* entropy,
                         float* top_log_probs, int64_t* top_ids, float* stats, int64_t rows, int64_t classes, int dtype, void* stream) {
    if (int rc = score_check(logits, stride, rows, classes, dtype)) return rc;
    CGB_REQUIRE(top >= 0 && top <= kScMaxTop && top <= classes, "log probabilities: top out of range (0 to 128, at most the number of classes)");
    if (rows == 0) return CGB200_OK;
    CGB_REQUIRE(entropy != nullptr && (targets == nullptr || log_prob != nullptr) && (top == 0 || (top_log_probs != nullptr && top_ids != nullptr)),
                "log probabilities: null buffer");
    CGB_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0, "log probabilities: stats must be 8-byte aligned");
    ScoreArgs a{};
    a.z = logits, a.z_stride = stride, a.rows = rows, a.classes = (int)classes, a.scale = kLog2e, a.stats = (float2*)stats;
    a.targets = targets, a.log_prob = log_prob, a.entropy = entropy, a.top = top, a.top_lp = top_log_probs, a.top_ids = top_ids;
    CGB_SCORE_TYPES(scores_fwd, kLogProbs, a, (cudaStream_t)stream);
}

int cgb200_log_probs_bwd(const void* logits, int64_t stride, const int64_t* targets, const float* entropy, const float* stats,
                         const float* g_log_prob, const float* g_entropy, void* dlogits, int64_t rows, int64_t classes, int dtype, void* stream) {
    if (int rc = score_check(logits, stride, rows, classes, dtype)) return rc;
    if (rows == 0) return CGB200_OK;
    CGB_REQUIRE(stats != nullptr && dlogits != nullptr && (g_entropy == nullptr || entropy != nullptr), "log probabilities: null buffer");
    CGB_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0, "log probabilities: stats must be 8-byte aligned");
    ScoreGradArgs a{};
    a.f.z = logits, a.f.z_stride = stride, a.f.rows = rows, a.f.classes = (int)classes, a.f.scale = kLog2e, a.f.stats = (float2*)stats;
    a.f.targets = targets, a.f.entropy = const_cast<float*>(entropy);
    a.dz = dlogits, a.g_lp = g_log_prob, a.g_ent = g_entropy;
    CGB_SCORE_TYPES(scores_bwd, kLogProbs, a, (cudaStream_t)stream);
}

int cgb200_distill_fwd(const void* logits, int64_t stride, const int64_t* teacher_ids, const void* teacher_scores, int n_teacher,
                       int teacher_dtype, float temperature, float* loss, float* stats, int64_t rows, int64_t classes, int dtype, void* stream) {
    if (int rc = score_check(logits, stride, rows, classes, dtype)) return rc;
    if (rows == 0) return CGB200_OK;
    if (int rc = teacher_check(teacher_ids, teacher_scores, n_teacher, teacher_dtype, temperature)) return rc;
    CGB_REQUIRE(loss != nullptr, "distillation: null buffer");
    CGB_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 15) == 0, "distillation: stats must be 16-byte aligned");
    ScoreArgs a{};
    a.z = logits, a.z_stride = stride, a.rows = rows, a.classes = (int)classes, a.scale = kLog2e / temperature, a.stats = (float2*)stats;
    a.t_ids = teacher_ids, a.t_scores = teacher_scores, a.n_t = n_teacher, a.t_dtype = teacher_dtype, a.temperature = temperature, a.loss = loss;
    a.inv_temperature = 1.0 / (double)temperature;
    CGB_SCORE_TYPES(scores_fwd, kDistill, a, (cudaStream_t)stream);
}

int cgb200_distill_bwd(const void* logits, int64_t stride, const int64_t* teacher_ids, const void* teacher_scores, int n_teacher,
                       int teacher_dtype, float temperature, const float* stats, const float* g_loss, void* dlogits, int64_t rows,
                       int64_t classes, int dtype, void* stream) {
    if (int rc = score_check(logits, stride, rows, classes, dtype)) return rc;
    if (rows == 0) return CGB200_OK;
    if (int rc = teacher_check(teacher_ids, teacher_scores, n_teacher, teacher_dtype, temperature)) return rc;
    CGB_REQUIRE(stats != nullptr && g_loss != nullptr && dlogits != nullptr, "distillation: null buffer");
    CGB_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 15) == 0, "distillation: stats must be 16-byte aligned");
    ScoreGradArgs a{};
    a.f.z = logits, a.f.z_stride = stride, a.f.rows = rows, a.f.classes = (int)classes, a.f.scale = kLog2e / temperature, a.f.stats = (float2*)stats;
    a.f.t_ids = teacher_ids, a.f.t_scores = teacher_scores, a.f.n_t = n_teacher, a.f.t_dtype = teacher_dtype, a.f.temperature = temperature;
    a.f.inv_temperature = 1.0 / (double)temperature;
    a.dz = dlogits, a.g_loss = g_loss;
    CGB_SCORE_TYPES(scores_bwd, kDistill, a, (cudaStream_t)stream);
}

}  // extern "C"
