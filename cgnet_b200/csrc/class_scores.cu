// What a classifier's scores are read for: log probabilities of given classes with entropy and the ranked best classes, and the
// distillation loss against a teacher's best scores; forward and backward.
//
// One pass over a row keeps, per thread, the running reference r (the largest score so far), s = sum 2^a and e = sum 2^a a,
// where a = (z - r) c, c = log2(e) / T.  From the joined (r, s, e) of a row
//     log p(j) = ln 2 ((z_j - r) c - log2 s),     H = ln 2 (log2 s - e / s).
// The difference is taken before the product: scores masked by the type's lowest value would overflow z c.  The backward passes
// read (r, 1 / s): p = 2^((z - r) c) / s carries no rounding of a stored logarithm.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "row_ops.cuh"

namespace cgb200 {

namespace cg = cooperative_groups;

constexpr int kScThreads = 256;
constexpr int kScUnroll = 4;                     // chunks a thread has in flight
constexpr int kScCap = 4096;                     // candidates a block collects before it has to fall back
constexpr int kScMaxTop = 128;                   // kScMaxTop threads' chunks of the first tile always fit the candidates
constexpr int kScWarpValues = 32;                // values per lane of the kernel for short rows
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;
static_assert(kScMaxTop * kScUnroll * 8 <= kScCap, "the first tile's candidates must fit");

enum ScoreMode { kLogProbs = 0, kDistill = 1 };

struct ScoreArgs {
    const void* z;
    int64_t z_stride, rows;
    int classes;
    float scale;               // log2(e) / temperature
    float2* stats;             // (r, 1 / s) per row; may be null
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
    if (z != z) return 0xffffffffu;
    const uint32_t b = __float_as_uint(z + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t o) {
    if (o == 0xffffffffu) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t key_of(float z, uint32_t idx) { return ((uint64_t)order_of(z) << 32) | (0xffffffffu - idx); }
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// Running statistics of a row, or of a part of one.
struct Stat {
    float m, r, s, e;    // largest score, the reference (the same, but 0 while m is -inf), sums relative to r
    __device__ __forceinline__ void clear() { m = -INFINITY, r = 0.f, s = 0.f, e = 0.f; }
    __device__ __forceinline__ void raise(float nm, float scale) {
                if (m == -INFINITY) {
            s *= 0.f, e *= 0.f;      // nothing so far, or a NaN, which stays
        } else {
            const float d = fmaxf((r - nm) * scale, -1e5f), f = ex2(d);
            e = f * (e + s * d);
            s *= f;
        }
        m = nm, r = nm;
    }
    template <int N, bool ENT>
    __device__ __forceinline__ void add(const float (&v)[N], float cm, float scale) {
        if (cm > m) raise(cm, scale);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float a = (v[i] - r) * scale;
            const float p = ex2(a);
            s += p;
            if (ENT) e = fmaf(p, fmaxf(a, -1e5f), e);     // p is 0 there: the bound keeps 0 * -inf out
        }
    }
    __device__ __forceinline__ void join(const Stat& o, float scale) {
        if (!(o.m > -INFINITY)) {             // nothing there, unless it holds a NaN
            s += o.s, e += o.e;
            return;
        }
        if (!(m > -INFINITY)) {
            const float s0 = s, e0 = e;
            *this = o;
            s += s0, e += e0;
            return;
        }
        const bool up = o.r > r;
        const float nr = up ? o.r : r;
        const float da = fmaxf((r - nr) * scale, -1e5f), db = fmaxf((o.r - nr) * scale, -1e5f), fa = ex2(da), fb = ex2(db);
        e = fa * (e + s * da) + fb * (o.e + o.s * db);
        s = fa * s + fb * o.s;
        m = up ? o.m : m, r = nr;
    }
    __device__ __forceinline__ Stat shfl_xor(int o) const {
        Stat x;
        x.m = __shfl_xor_sync(0xffffffffu, m, o), x.r = __shfl_xor_sync(0xffffffffu, r, o);
        x.s = __shfl_xor_sync(0xffffffffu, s, o), x.e = __shfl_xor_sync(0xffffffffu, e, o);
        return x;
    }
};
__device__ __forceinline__ Stat warp_join(Stat a, float scale) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stat b = a.shfl_xor(o);
        // both lanes of a pair join in the same order, so that all lanes end with the same bits
        Stat lo = (threadIdx.x & o) ? b : a;
        lo.join((threadIdx.x & o) ? a : b, scale);
        a = lo;
    }
    return a;
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
// Sums over the threads that share a row: a warp (buf unused) or the block.
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
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (float)buf[0];
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) v = fmaxf(v, (float)buf[i]);
    return v;
}
// Teacher's distribution over the classes it names: q(k) = exp(t_k / T - tmax / T) / sum.  Entries with a negative class are
// not there; a class beyond the last makes the row NaN.
struct Teacher {
    float tmax;
    double sum;
    bool any;
};
__device__ __forceinline__ Teacher teacher_of(const ScoreArgs& a, int64_t row, int t, int G, double* buf, bool whole_block) {
    const int64_t at = row * a.n_t;
    float mx = -INFINITY, some = 0.f;
    for (int k = t; k < a.n_t; k += G) {
        if (a.t_ids[at + k] < 0) continue;
        const float v = load_score(a.t_scores, a.t_dtype, at + k);
        if (v != -INFINITY) some = 1.f;
        mx = fmaxf(mx, v);
    }
    Teacher q;
    q.any = row_max_f(some, buf, whole_block) > 0.f;
    q.tmax = row_max_f(mx, buf, whole_block);
    double s = 0.0;
    for (int k = t; k < a.n_t; k += G) {
        const int64_t id = a.t_ids[at + k];
        if (id < 0) continue;
        s += id < a.classes ? exp(((double)load_score(a.t_scores, a.t_dtype, at + k) - (double)q.tmax) / (double)a.temperature) : nan("");
    }
    q.sum = q.any ? row_sum_d(s, buf, whole_block) : 1.0;     // `any` is the same in all threads of the row
    return q;
}
template <typename T>
__device__ __forceinline__ float distill_loss(const ScoreArgs& a, int64_t row, const T* zr, const Stat& st, int t, int G, double* buf,
                                              bool whole_block) {
    const Teacher q = teacher_of(a, row, t, G, buf, whole_block);
    if (!q.any) return 0.f;
    const int64_t at = row * a.n_t;
    const double log_sum = log(q.sum), log2_s = log2((double)st.s);
    double acc = 0.0;
    for (int k = t; k < a.n_t; k += G) {
        const int64_t id = a.t_ids[at + k];
        if (id < 0 || id >= a.classes) continue;
        const double lt = ((double)load_score(a.t_scores, a.t_dtype, at + k) - (double)q.tmax) / (double)a.temperature;
        const double w = exp(lt) / q.sum;
        if (w == 0.0) continue;
        const double lp = empty_row(st) ? -INFINITY : kLn2 * (((double)to_f32(zr[id]) - (double)st.r) * (double)a.scale - log2_s);
        acc += w * (lt - log_sum - lp);
    }
    acc = row_sum_d(acc, buf, whole_block);
    // a NaN of the sum (a class beyond the last) is in log_sum even where no entry was added
    if (q.sum != q.sum) acc = q.sum;
    return (float)((double)a.temperature * (double)a.temperature * acc);
}

// ---- rows a warp holds in registers --------------------------------------------------------------------------------
template <typename T, int MODE, int CH>
__global__ void __launch_bounds__(kScThreads) scores_warp_kernel(ScoreArgs a) {
    constexpr int N = Chunk<T>::N;
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (kScThreads / 32) + (threadIdx.x >> 5);
    if (row >= a.rows) return;       // whole warps leave; nothing below is wider than a warp
    const T* zr = (const T*)a.z + row * a.z_stride;
    const int ph = row_phase(zr);
    float v[CH][N];
    Stat st;
    st.clear();
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e0 = (lane + 32 * c) * N - ph;
        load_chunk(zr, e0, a.classes, -INFINITY, v[c]);
        float cm = v[c][0];
#pragma unroll
        for (int i = 1; i < N; ++i) cm = max_nan(cm, v[c][i]);
        st.add<N, MODE == kLogProbs>(v[c], cm, a.scale);
    }
    st = warp_join(st, a.scale);
    if (a.stats != nullptr && lane == 0) a.stats[row] = make_float2(st.r, empty_row(st) ? 0.f : 1.f / st.s);
    if (MODE == kDistill) {
        const float loss = distill_loss(a, row, zr, st, lane, 32, nullptr, false);
        if (lane == 0) a.loss[row] = loss;
        return;
    }
    const double log2_s = log2((double)st.s);
    if (lane == 0) {
        a.entropy[row] = empty_row(st) ? 0.f : (float)(kLn2 * (log2_s - (double)st.e / (double)st.s));
        if (a.targets != nullptr) {
            const int64_t t = a.targets[row];
            a.log_prob[row] = t < 0 ? 0.f : t >= a.classes ? __uint_as_float(0x7fffffffu) : log_prob_of(st, log2_s, to_f32(zr[t]), a.scale);
        }
    }
    if (a.top == 0) return;
    // the best of each lane, and the best of those, `top` times over
    uint64_t last = ~0ull, best = 0;
    for (int k = 0; k < a.top; ++k) {
        if (k == 0 || best == last) {       // this lane's best is not known, or was the one just taken
            best = 0;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int e = (lane + 32 * c) * N - ph + i;
                    if (e < 0 || e >= a.classes) continue;
                    const uint64_t key = key_of(v[c][i], (uint32_t)e);
                    if (key < last && key > best) best = key;
                }
        }
        const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
        const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
        last = ((uint64_t)hi << 32) | lo;
        if (lane == 0) {
            a.top_ids[row * a.top + k] = index_of(last);
            a.top_lp[row * a.top + k] = log_prob_of(st, log2_s, score_of(hi), a.scale);
        }
    }
}

// ---- long rows: a block, or a cluster of blocks, per row -------------------------------------------------------------
struct ScoreShared {
    uint64_t buf[kScCap];          // candidates
    uint64_t best[kScMaxTop];      // this block's best, in order
    Stat part[kScThreads / 32];
    Stat stat;
    float tmax[kScThreads];
    unsigned hist[256];
    int count, n_best;
    float thr;
    uint64_t prefix;
    unsigned want;
    double red[kScThreads / 32];
};

__device__ __forceinline__ void push(ScoreShared& sh, uint64_t key) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kScCap) sh.buf[at] = key;
}

// The `k` highest of the first n candidates, in order, to sh.best (n_best of them).  All keys differ, so their order
// does not depend on the order in which they were collected.
__device__ void select_best(ScoreShared& sh, int n, int k) {
    if (n <= 512) {
        for (int i = threadIdx.x; i < n; i += kScThreads) {
            const uint64_t key = sh.buf[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += sh.buf[j] > key;
            if (rank < k) sh.best[rank] = key;
        }
    } else {
        int p = 1024;
        while (p < n) p *= 2;
        for (int i = n + threadIdx.x; i < p; i += kScThreads) sh.buf[i] = 0;
        for (int size = 2; size <= p; size *= 2)
            for (int d = size / 2; d > 0; d /= 2) {
                __syncthreads();
                for (int i = threadIdx.x; i < p / 2; i += kScThreads) {
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

template <typename T, int MODE, bool CLUSTER>
__global__ void __launch_bounds__(kScThreads) scores_row_kernel(ScoreArgs a, int blocks_per_row) {
    constexpr int N = Chunk<T>::N;
    constexpr bool ENT = MODE == kLogProbs;
    __shared__ ScoreShared sh;
    const int part = CLUSTER ? (int)(blockIdx.x % (unsigned)blocks_per_row) : 0;
    const int64_t row = CLUSTER ? (int64_t)(blockIdx.x / (unsigned)blocks_per_row) : (int64_t)blockIdx.x;
    const T* zr = (const T*)a.z + row * a.z_stride;
    const int ph = row_phase(zr);
    const int nc = (a.classes + ph + N - 1) / N;
    const int per = CLUSTER ? (nc + blocks_per_row - 1) / blocks_per_row : nc;
    const int c0 = min(nc, part * per), c1 = min(nc, c0 + per);
    const int full0 = ph > 0 ? 1 : 0, full1 = (a.classes + ph) / N;     // chunks [full0, full1) lie inside the row
    const int first = max(0, c0 * N - ph), behind = min(a.classes, c1 * N - ph);   // this block's classes
    const bool tops = ENT && a.top > 0;
    const int want = tops ? min(a.top, max(0, behind - first)) : 0;      // entries it has to offer
    if (threadIdx.x == 0) sh.count = 0;
    Stat st;
    st.clear();
    float thr = INFINITY;
    for (int base = c0; base < c1; base += kScThreads * kScUnroll) {
        uint4 raw[kScUnroll];
        const bool inside = base >= full0 && base + kScThreads * kScUnroll <= min(c1, full1);
        if (inside) {
#pragma unroll
            for (int u = 0; u < kScUnroll; ++u)
                raw[u] = *reinterpret_cast<const uint4*>(zr + ((int64_t)(base + u * kScThreads + (int)threadIdx.x) * N - ph));
        } else {
#pragma unroll
            for (int u = 0; u < kScUnroll; ++u) {
                const int c = base + u * kScThreads + (int)threadIdx.x;
                float v[N];
                load_chunk(zr, (int64_t)c * N - ph, c < c1 ? a.classes : 0, -INFINITY, v);
                raw[u] = pack16(v, (const T*)nullptr);       // the values came from this type: nothing is rounded
            }
        }
        float tm = -INFINITY;
#pragma unroll
        for (int u = 0; u < kScUnroll; ++u) {
            float v[N];
            unpack16(raw[u], v, (const T*)nullptr);
            float cm = v[0];
#pragma unroll
            for (int i = 1; i < N; ++i) cm = max_nan(cm, v[i]);
            st.add<N, ENT>(v, cm, a.scale);
            tm = fmaxf(tm, cm);
            if (tops && base != c0 && !(cm <= thr)) {
                const int e0 = (base + u * kScThreads + (int)threadIdx.x) * N - ph;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (!(v[i] <= thr)) push(sh, key_of(v[i], (uint32_t)(e0 + i)));
            }
        }
        if (tops && base == c0) {
            // Threshold: at least `top` threads of the first tile hold a score of at least the top-th highest of the threads'
            // maxima, so nothing below it can rank, and nothing equal to it further right.
            sh.tmax[threadIdx.x] = tm;
            __syncthreads();
            int above = 0, same = 0;
            for (int j = 0; j < kScThreads; ++j) {
                const float o = sh.tmax[j];
                above += o > tm;
                same += o == tm && j < (int)threadIdx.x;
            }
            if (above + same == a.top - 1) sh.thr = tm;
            __syncthreads();
            thr = sh.thr;
#pragma unroll
            for (int u = 0; u < kScUnroll; ++u) {
                const int e0 = (base + u * kScThreads + (int)threadIdx.x) * N - ph;
                float v[N];
                unpack16(raw[u], v, (const T*)nullptr);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (!(v[i] < thr) && v[i] != -INFINITY) push(sh, key_of(v[i], (uint32_t)(e0 + i)));
            }
        }
    }
    st = warp_join(st, a.scale);
    if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = st;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kScThreads / 32; ++w) st.join(sh.part[w], a.scale);
        sh.stat = st;
    }
    if (tops) {
        int n = sh.count;
        if (n > kScCap) {
            radix_collect(sh, zr, ph, c0, c1, a.classes, want);
            n = sh.count;
        } else if (n < want) {
            // fewer scores than places: masked classes follow, lowest index first
            if (threadIdx.x == 0)
                for (int e = first; e < behind && n < want; ++e)
                    if (to_f32(zr[e]) == -INFINITY) sh.buf[n++] = key_of(-INFINITY, (uint32_t)e);
            n = want;
            __syncthreads();
        }
        select_best(sh, n, want);
    }
    if (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (part == 0) {
            if (threadIdx.x == 0) {
                st = sh.stat;
                for (int p = 1; p < blocks_per_row; ++p) st.join(cluster.map_shared_rank(&sh, p)->stat, a.scale);
                sh.stat = st;
                sh.count = 0;
            }
            __syncthreads();
            if (tops) {
                for (int i = threadIdx.x; i < blocks_per_row * kScMaxTop; i += kScThreads) {
                    const ScoreShared* o = cluster.map_shared_rank(&sh, i / kScMaxTop);
                    if (i % kScMaxTop < o->n_best) push(sh, o->best[i % kScMaxTop]);
                }
                __syncthreads();
                const int n = sh.count;
                __syncthreads();          // the remote lists, block 0's own among them, have been read
                select_best(sh, n, a.top);
            }
        }
        cluster.sync();                   // no block leaves while its lists are read
        if (part != 0) return;
    } else {
        __syncthreads();
    }
    st = sh.stat;
    if (a.stats != nullptr && threadIdx.x == 0) a.stats[row] = make_float2(st.r, empty_row(st) ? 0.f : 1.f / st.s);
    if (MODE == kDistill) {
        const float loss = distill_loss(a, row, zr, st, (int)threadIdx.x, kScThreads, sh.red, true);
        if (threadIdx.x == 0) a.loss[row] = loss;
        return;
    }
    const double log2_s = log2((double)st.s);
    if (threadIdx.x == 0) {
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

// ---- gradients with respect to the scores --------------------------------------------------------------------------
struct ScoreGradArgs {
    ScoreArgs f;
    void* dz;
    const float *g_lp, *g_ent, *g_loss;    // per row; g_lp or g_ent may be null
};

// kScThreads / G rows of a block, G threads a row and `run` chunks of it per block.  log_probs:
//     dz_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)
// distillation:  dz_j = g T (p_j - sum_k q_k 1[id_k = j]); the named classes are written a second time, each by its first entry.
template <typename T, int MODE>
__global__ void __launch_bounds__(kScThreads) scores_grad_kernel(ScoreGradArgs a, int G, int run, int runs) {
    constexpr int N = Chunk<T>::N;
    __shared__ double red[kScThreads / 32];
    extern __shared__ int sids[];                       // distillation: classes of this block's rows
    const int t = (int)threadIdx.x % G, sub = (int)threadIdx.x / G, rows_here = kScThreads / G;
    const int64_t row = (int64_t)(blockIdx.x / (unsigned)runs) * rows_here + sub;
    const bool on = row < a.f.rows;
    const int c_begin = (int)(blockIdx.x % (unsigned)runs) * run;
    const T* zr = (const T*)a.f.z + (on ? row : 0) * a.f.z_stride;
    T* dr = (T*)a.dz + (on ? row : 0) * a.f.classes;
    const int V = a.f.classes, ph = row_phase(zr);
    const float2 st = on ? a.f.stats[row] : make_float2(0.f, 0.f);
    const float scale = a.f.scale;
    const int c_end = min(c_begin + run, (V + ph + N - 1) / N);
    if (MODE == kLogProbs) {
        if (!on) return;
        const int64_t tgt = a.f.targets != nullptr ? a.f.targets[row] : -1;
        const bool dead = st.y == 0.f;                                          // a row without a distribution
        float g_lp = a.g_lp != nullptr && tgt >= 0 && !dead ? a.g_lp[row] : 0.f;
        if (tgt >= V) g_lp = __uint_as_float(0x7fffffffu);
        const float g_ent = a.g_ent != nullptr && !dead ? a.g_ent[row] : 0.f;
        const float H = a.g_ent != nullptr ? a.f.entropy[row] : 0.f;
        const float ln2 = (float)kLn2, lg = log2f(st.y);
        for (int c = c_begin + t; c < c_end; c += G) {
            const int64_t e0 = (int64_t)c * N - ph;
            float v[N];
            load_chunk(zr, e0, V, 0.f, v);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float y = (v[i] - st.x) * scale;
                const float p = ex2(y) * st.y;
                float d = -g_lp * p;
                if (g_ent != 0.f) d -= g_ent * p * (ln2 * (fmaxf(y, -1e5f) + lg) + H);
                if (dead) d = 0.f;
                if (e0 + i == tgt) d += g_lp;
                v[i] = d;
            }
            store_chunk(dr, e0, V, v);
        }
        return;
    }
    const bool whole = G > 32;       // then the block has one row
    Teacher q{};
    if (on) q = teacher_of(a.f, row, t, G, red, whole);
    const bool dead = !on || !q.any || st.y == 0.f;
    const float g = dead ? 0.f : a.g_loss[row] * a.f.temperature;
    if (on) {
        for (int c = c_begin + t; c < c_end; c += G) {
            const int64_t e0 = (int64_t)c * N - ph;
            float v[N];
            load_chunk(zr, e0, V, 0.f, v);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = dead ? 0.f : g * (ex2((v[i] - st.x) * scale) * st.y);
            store_chunk(dr, e0, V, v);
        }
    }
    int* ids = sids + sub * a.f.n_t;
    if (on && !dead)
        for (int k = t; k < a.f.n_t; k += G) {
            const int64_t id = a.f.t_ids[row * a.f.n_t + k];
            ids[k] = id >= 0 && id < V ? (int)id : -1;
        }
    __syncthreads();                 // the list is there, and what the block wrote above is in order before what follows
    if (dead) return;
    const int e_lo = c_begin * N - ph, e_hi = c_end * N - ph;
    for (int k = t; k < a.f.n_t; k += G) {
        const int id = ids[k];
        if (id < e_lo || id >= e_hi || id < 0) continue;
        double w = 0.0;
        bool mine = true;
        for (int j = 0; j < a.f.n_t; ++j) {
            if (ids[j] != id) continue;
            if (j < k) {
                mine = false;
                break;
            }
            w += exp(((double)load_score(a.f.t_scores, a.f.t_dtype, row * a.f.n_t + j) - (double)q.tmax) / (double)a.f.temperature) / q.sum;
        }
        if (mine) dr[id] = from_f32<T>(g * (float)((double)(ex2((to_f32(zr[id]) - st.x) * scale) * st.y) - w));
    }
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
    const int G = chunks <= 32 ? 32 : kScThreads;
    const int run = kScThreads * kScUnroll;
    const int runs = G == 32 ? 1 : (int)((chunks + run - 1) / run);
    const int64_t blocks = (a.f.rows + kScThreads / G - 1) / (kScThreads / G) * runs;
    CGB_REQUIRE(blocks <= 0x7fffffff, "class scores: too many blocks for one launch");
    const size_t smem = MODE == kDistill ? (size_t)(kScThreads / G) * a.f.n_t * sizeof(int) : 0;
    launch_begin(kid, st);
    scores_grad_kernel<T, MODE><<<(unsigned)blocks, kScThreads, smem, st>>>(a, G, run, runs);
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
    ScoreArgs a{};
    a.z = logits, a.z_stride = stride, a.rows = rows, a.classes = (int)classes, a.scale = kLog2e / temperature, a.stats = (float2*)stats;
    a.t_ids = teacher_ids, a.t_scores = teacher_scores, a.n_t = n_teacher, a.t_dtype = teacher_dtype, a.temperature = temperature, a.loss = loss;
    CGB_SCORE_TYPES(scores_fwd, kDistill, a, (cudaStream_t)stream);
}

int cgb200_distill_bwd(const void* logits, int64_t stride, const int64_t* teacher_ids, const void* teacher_scores, int n_teacher,
                       int teacher_dtype, float temperature, const float* stats, const float* g_loss, void* dlogits, int64_t rows,
                       int64_t classes, int dtype, void* stream) {
    if (int rc = score_check(logits, stride, rows, classes, dtype)) return rc;
    if (rows == 0) return CGB200_OK;
    if (int rc = teacher_check(teacher_ids, teacher_scores, n_teacher, teacher_dtype, temperature)) return rc;
    CGB_REQUIRE(stats != nullptr && g_loss != nullptr && dlogits != nullptr, "distillation: null buffer");
    ScoreGradArgs a{};
    a.f.z = logits, a.f.z_stride = stride, a.f.rows = rows, a.f.classes = (int)classes, a.f.scale = kLog2e / temperature, a.f.stats = (float2*)stats;
    a.f.t_ids = teacher_ids, a.f.t_scores = teacher_scores, a.f.n_t = n_teacher, a.f.t_dtype = teacher_dtype, a.f.temperature = temperature;
    a.dz = dlogits, a.g_loss = g_loss;
    CGB_SCORE_TYPES(scores_bwd, kDistill, a, (cudaStream_t)stream);
}

}  // extern "C"
