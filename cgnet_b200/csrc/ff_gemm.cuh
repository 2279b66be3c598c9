// Tensor-core products of the gated feed-forward block (gated_ff.cu): one persistent kernel for out[i][j] = sum_k A[i][k] B[j][k] over
// a list of problems, with the gated epilogue or a plain one.
//
// Block: 128 rows i x BN columns j, 64 terms k per stage.  One thread issues the tiled bulk copies (64 x 64 boxes, 128-byte swizzle) of a
// stage, one thread the tcgen05.mma of the stages before, eight warps read finished accumulators from tensor memory and write
// them out while the next tile is multiplied into the other accumulator.  An operand may have its k axis (rows of the product in
// memory) or its i / j axis contiguous; the copies are the same, only coordinates and descriptors differ, so no operand is ever
// transposed in memory.
//
// float32 operands come as three bfloat16 planes (8 + 8 + 8 bits, together exact).  Of the nine plane products the six that reach
// 2^-24 are taken; the leading one has its own accumulator, because the tensor core truncates each addition and the small
// products would otherwise add steps to its long chain.  Every kFfFlush stages the accumulators are added, rounded, to sums in registers.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "row_ops.cuh"
#include "tc_ptx.cuh"

namespace cgb200 {

constexpr int kFfBM = 128, kFfBK = 64;
constexpr int kFfThreads = 384;                // producer, issuer, allocator, idle; eight epilogue warps
constexpr int kFfEpiWarps = 8;
constexpr int kFfBox = 64 * 64 * 2;            // bytes of one copy
constexpr int kFfStageBytes = 192 * 1024;      // all stages of a block
constexpr int kFfFlush = 4;                    // stages between flushes of the three-plane form (16 truncating additions)
constexpr int kFfStaging = 32 * 32;            // floats of an epilogue warp's staging area
constexpr size_t kFfSmem = 1024 + kFfStageBytes + kFfEpiWarps * kFfStaging * sizeof(float);
static_assert(kFfSmem <= kMaxDynSmem, "stages and staging must fit a block's shared memory");

// Tensor maps of a launch: operands (the backward's dg and du; half precision's scaled copies by rows and by units), outputs
enum FfMap { kMapX, kMapWg, kMapWu, kMapDg, kMapDu, kMapDgRows, kMapDuRows, kMapDgCols, kMapDuCols, kMapOut, kMapOutWg, kMapOutWu, kMaps };

struct FfProblem {
    int a_map[2], b_map[2];     // tensor maps of A and B: by source of the contraction (dx), set of rows (dW: A), half of the columns (forward: B)
    int a_mn, b_mn;             // 1: the operand's i / j axis is the contiguous one
    int sources, kblk;          // the contraction runs over `sources` x kblk stages
    int sets, tiles_i, tiles_j; // row tiles of each set of rows, column tiles
    int splits, kper;           // the contraction in parts of kper stages
    int unit0;                  // first work unit of this problem
    int64_t n_i;                // rows of a set
    int n_j;
    int h_aligned;              // the forward: rows of h start on 16-byte boundaries
    void* out[2];               // per set; the forward: h
    int out_map[2];             // tensor map of the output by bulk copies, -1: written by threads; the forward: [0] g and u, -1: not kept
    float* part;                // [splits][sets * n_i][n_j] where splits > 1
    // half precision's backward, per set: whether a tile of rows is read from the scaled copy, that copy's map (by source or set, as
    // a_map), and the largest value of each row, which tells its scale; null: never
    const uint32_t *flag[2], *amax[2];
    int a_scaled[2];
};
struct FfGemmArgs {
    CUtensorMap map[kMaps];
    FfProblem p[2];
    int problems, units;
    uint32_t idesc_type;        // operand format bits of the instruction descriptor
    int act;
    uint32_t polls;
};

__device__ __forceinline__ void tma_box(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_16bit(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
        :
        : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
        "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// 16 columns at either address
__device__ __forceinline__ void tmem_ld16x2(uint32_t at0, uint32_t at1, float (&v)[32]) {
    uint32_t a[16], b[16];
    tmem_ld16(at0, a);
    tmem_ld16(at1, b);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(a[i]), v[16 + i] = __uint_as_float(b[i]);
}
// Descriptor of an operand tile made of 64 x 64 boxes in the 128-byte swizzle.  k contiguous: a box is 64 rows of 128 bytes, 8-row
// groups 1024 bytes apart.  i / j contiguous: a box is 64 k-rows of 64 values; groups of 8 k are 1024 bytes apart (stride offset),
// the next 64 values one box (leading offset).  [61,64) = 2 is the 128-byte swizzle.
__device__ __forceinline__ uint64_t box_desc(uint32_t saddr, int mn) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(mn ? kFfBox >> 4 : 1) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}

// Half precision keeps a row or unit of dg and du as it is where its largest value is in this range: a subnormal value's rounding, 2^-25,
// is then at most 2^-10 of the largest one's.
__device__ __forceinline__ bool fits_half(uint32_t amax) { return amax == 0 || (amax >= __float_as_uint(0.0625f) && amax <= __float_as_uint(65504.f)); }
// Power of two that brings values up to `amax` (the bits of a float32, 0: none) below 2^15, and its inverse.  The largest factor is
// 2^126, so that the inverse is not subnormal.
__device__ __forceinline__ uint32_t scale_exponent(uint32_t amax) { return amax == 0 ? 127u : min(127 + 14 + 127 - (amax >> 23), 253u); }
__device__ __forceinline__ float scale_of(uint32_t amax) { return __uint_as_float(scale_exponent(amax) << 23); }
__device__ __forceinline__ float unscale_of(uint32_t amax) { return __uint_as_float((254u - scale_exponent(amax)) << 23); }

// act(g) and its derivative
template <int ACT, bool GRAD>
__device__ __forceinline__ float2 activate_as(float g) {
    if (ACT == CGB200_ACT_RELU) return g > 0.f ? make_float2(g, 1.f) : make_float2(g != g ? g : 0.f, 0.f);
    if (ACT == CGB200_ACT_SILU) {
        // below -88 the exponential leaves float32's range, and g may be -inf; a NaN fails the comparison
        const float s = g < -88.f ? 0.f : __fdividef(1.f, 1.f + __expf(-g));
        return g < -88.f ? make_float2(0.f, 0.f) : make_float2(g * s, GRAD ? s * (1.f + g * (1.f - s)) : 0.f);
    }
    const float c = 0.5f * erfcf(-0.70710678118654752f * g);
    return make_float2(c == 0.f ? 0.f : g * c, GRAD ? c + (fabsf(g) > 20.f ? 0.f : g * __expf(-0.5f * g * g) * 0.39894228040143268f) : 0.f);
}
template <bool GRAD>
__device__ __forceinline__ float2 activate(int act, float g) {
    if (act == CGB200_ACT_RELU) return activate_as<CGB200_ACT_RELU, GRAD>(g);
    if (act == CGB200_ACT_SILU) return activate_as<CGB200_ACT_SILU, GRAD>(g);
    return activate_as<CGB200_ACT_GELU, GRAD>(g);
}
// The same, one copy of it, for kernels that want short code
__device__ __noinline__ float2 activate_shared(int act, float g) { return activate<true>(act, g); }

struct FfUnit {
    const FfProblem* p;
    int set, split, k0, k1;
    int64_t i0;
    int j0;        // in columns of the product's output
};
// Tiles in groups of eight row tiles, columns next: the blocks at work at one time share rows of A and of B in L2.
__device__ __forceinline__ FfUnit ff_unit(const FfGemmArgs& a, int u, int jw) {
    FfUnit t;
    t.p = &a.p[a.problems > 1 && u >= a.p[1].unit0 ? 1 : 0];
    const FfProblem& p = *t.p;
    int v = u - p.unit0;
    const int per_set = p.tiles_i * p.tiles_j, tiles = p.sets * per_set;
    t.split = v / tiles;
    v -= t.split * tiles;
    t.set = v / per_set;
    v -= t.set * per_set;
    const int group = v / (8 * p.tiles_j), first = group * 8, height = min(8, p.tiles_i - first);
    v -= first * p.tiles_j;
    t.i0 = (int64_t)(first + v % height) * kFfBM;
    t.j0 = v / height * jw;
    t.k0 = t.split * p.kper;
    t.k1 = min(p.sources * p.kblk, t.k0 + p.kper);
    return t;
}

// Outputs leave through a warp's 4 KB of shared memory by bulk copies of 32 rows x 64 bytes (64-byte swizzle: the 16-byte pieces of a
// row are permuted by its number, so that neither side has bank conflicts): a quarter of the load/store instructions of turning
// the rows by hand, which competed with the products for shared memory.
__device__ __forceinline__ void tma_store(const CUtensorMap* map, const void* src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(c0),
                 "r"(c1), "r"(c2)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until at most N of this thread's stores still read their shared memory
template <int N>
__device__ __forceinline__ void tma_store_wait() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
// 64 bytes of this lane's row into a 2 KB block
__device__ __forceinline__ void put_row(char* block, const uint4 (&u)[4]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(block + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = u[j];
}
__device__ __forceinline__ void pack_row(const float* v, uint4 (&u)[4], const float*) {      // 16 values
#pragma unroll
    for (int j = 0; j < 4; ++j)
        u[j] = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
}
template <typename T>
__device__ __forceinline__ void pack_row(const float* v, uint4 (&u)[4], const T*) {          // 32 values
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = v[8 * j + i];
        u[j] = pack16(t, (const T*)nullptr);
    }
}
// 32 x W values, row = lane, to columns col0.. of rows row0.. of a row-major matrix of any alignment: turned in shared memory, so that
// a warp writes neighbouring columns.
template <int W, typename O>
__device__ __forceinline__ void write_block(const float* v, float* st, O* out, int64_t row0, int64_t n_rows, int64_t ld, int col0, int n_cols) {
    const int lane = threadIdx.x & 31, cc = lane % W;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < W; ++c) st[lane * W + (c ^ (lane % W))] = v[c];
    __syncwarp();
    if (col0 + cc < n_cols) {
        const int n = (int)min((int64_t)32, n_rows - row0);
        O* o = out + row0 * ld + col0 + cc;
#pragma unroll 8
        for (int r = lane / W; r < n; r += 32 / W) o[r * ld] = from_f32<O>(st[r * W + (cc ^ (r % W))]);
    }
}
// h = act(g) u of 16 columns of this lane's row, in place of g
template <int ACT>
__device__ __forceinline__ void gate(float (&g)[16], const float (&u)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) g[i] = activate_as<ACT, false>(g[i]).x * u[i];
}

// Alone on the GPU at 8192 rows, 2048 -> 5120, bf16: forward 237 us in inference (1450 TFLOP/s), 301 when g and u are kept (336 MB
// more to write), both backward products 456 us (1.5 PFLOP/s, tensor pipe 83 %).  Not the epilogue but the main loop bounds the
// forward: 625 cycles per 64-term stage in inference and 750 in training against 512 of MMA, because the 48 KB a stage brings into
// the SM share the way from L2 with what the epilogue writes.  Height of a group of row tiles (4, 8, 16, 32): within 3 %.
template <int PLANES, int BN, typename T, bool FWD>
__global__ void __launch_bounds__(kFfThreads, 1) ff_gemm_kernel(const __grid_constant__ FfGemmArgs a) {
    constexpr int kStage = PLANES * (kFfBM + BN) * kFfBK * 2;
    constexpr int kStages = kFfStageBytes / kStage;
    constexpr int kAccCols = PLANES == 1 ? BN : 2 * BN;      // columns of one accumulator
    constexpr int kTmemCols = 2 * kAccCols;
    constexpr int JW = FWD ? BN / 2 : BN;                    // output columns of a tile
    constexpr int kFlush = PLANES == 1 ? 1 << 30 : kFfFlush;
    static_assert(kTmemCols <= 512, "two accumulators must fit the tensor memory");
    extern __shared__ char dyn[];
    __shared__ uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], stopped;
    __shared__ uint32_t tmem_ptr;
    __shared__ int failed_flag;
    volatile int* failed = &failed_flag;
    char* base = dyn + ((1024 - (smem_u32(dyn) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        failed_flag = 0;
        for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        for (int s = 0; s < 2; ++s) mbar_init(&acc_full[s], 1), mbar_init(&acc_empty[s], kFfEpiWarps);
        mbar_init(&stopped, 1);
        fence_mbar_init();
    }
    if (warp == 2) tmem_alloc(&tmem_ptr, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_ptr, polls = a.polls;
    constexpr bool SCALED = !FWD && std::is_same<T, __half>::value;
    auto scaled = [&](const FfUnit& t) { return SCALED && t.p->flag[t.set] != nullptr && t.p->flag[t.set][t.i0 / kFfBM] != 0; };

    // Units are listed longest first; blocks take them in turn, there and back, so that who had a long one gets a short one next.
    // (In an odd round the places may lie beyond the last unit for this block while other blocks still have one: it is done then.)
    auto unit_of = [&](int n) { return n * (int)gridDim.x + (n & 1 ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x); };

    // The two issuing roles run on one elected thread: under elect.sync the compiler knows that, and keeps what the copies and
    // products take in uniform registers (under `lane == 0` a copy took 80 cycles to issue and bounded the kernel).
    if (warp == 0) {
        if (elect_one()) {
            int s = 0, issued = 0;
            uint32_t ph = 1;
            bool ok = true;
            for (int n = 0, u; (u = unit_of(n)) < a.units && ok; ++n) {
                const FfUnit t = ff_unit(a, u, JW);
                // in registers: what the loop looked up in the arguments each time cost it more than the copies' own time
                const int kblk = t.p->kblk, a_mn = t.p->a_mn, b_mn = t.p->b_mn, i0 = (int)t.i0, j0 = t.j0, k1 = t.k1;
                const bool two = t.p->sources > 1;
                const int* maps = scaled(t) ? t.p->a_scaled : t.p->a_map;
                const CUtensorMap* a0 = &a.map[maps[t.p->sets > 1 ? t.set : 0]];
                const CUtensorMap* a1 = &a.map[maps[1]];
                const CUtensorMap *b0 = &a.map[t.p->b_map[0]], *b1 = &a.map[t.p->b_map[1]];
                for (int it = t.k0; it < k1; ++it) {
                    if (!mbar_wait(&empty[s], ph, failed, polls)) {
                        ok = false;
                        break;
                    }
                    const bool src = two && it >= kblk;
                    const int k = (src ? it - kblk : it) * kFfBK;
                    const CUtensorMap* am = src ? a1 : a0;
                    char* d = base + s * kStage;
                    mbar_arrive_expect_tx(&full[s], kStage);
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
#pragma unroll
                        for (int b = 0; b < kFfBM / 64; ++b, d += kFfBox) {
                            const int i = i0 + 64 * b;
                            tma_box(d, am, a_mn ? i : k, a_mn ? k : i, q, &full[s]);
                        }
                    }
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
#pragma unroll
                        for (int b = 0; b < BN / 64; ++b, d += kFfBox) {
                            const int second = FWD && b >= BN / 128;      // the up projection's half of the columns
                            const int j = j0 + 64 * (b - second * (BN / 128));
                            tma_box(d, (FWD ? second : src) ? b1 : b0, b_mn ? j : k, b_mn ? k : j, q, &full[s]);
                        }
                    }
                    ++issued;
                    if (++s == kStages) s = 0, ph ^= 1;
                }
            }
            if (!ok) {
                // let the copies in flight land before the block gives up its shared memory: the last kStages issued ones
                for (int n = max(0, issued - kStages); n < issued; ++n) mbar_drain(&full[n % kStages], (n / kStages) & 1, polls);
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            int s = 0, acc = 0;
            uint32_t ph = 0, acc_ph = 1;
            bool ok = true;
            for (int n = 0, u; (u = unit_of(n)) < a.units && ok; ++n) {
                const FfUnit t = ff_unit(a, u, JW);
                const int a_mn = t.p->a_mn, b_mn = t.p->b_mn, k1 = t.k1;
                const uint32_t idesc = (1u << 4) | a.idesc_type | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(BN >> 3) << 17) |
                                       ((uint32_t)(kFfBM >> 4) << 24);
                const uint32_t a_step = a_mn ? 2048 : 32, b_step = b_mn ? 2048 : 32;
                const uint64_t da0 = box_desc(smem_u32(base), a_mn), db0 = box_desc(smem_u32(base) + PLANES * kFfBM * kFfBK * 2, b_mn);
                for (int it = t.k0; it < k1;) {
                    if (!mbar_wait(&acc_empty[acc], acc_ph, failed, polls)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem + acc * kAccCols;
                    const int stop = min(k1 - it, kFlush) + it;
                    bool first = true;
                    for (; it < stop; ++it) {
                        if (!mbar_wait(&full[s], ph, failed, polls)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t da = desc_advance(da0, s * kStage), db = desc_advance(db0, s * kStage);
                        if constexpr (PLANES == 1) {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                mma_16bit(d, desc_advance(da, k * a_step), desc_advance(db, k * b_step), idesc, !first || k > 0);
                        } else {
                            constexpr uint32_t pa = kFfBM * kFfBK * 2, pb = BN * kFfBK * 2;     // bytes of a plane
                            constexpr int qa[5] = {0, 2, 1, 0, 1}, qb[5] = {2, 0, 1, 1, 0};
#pragma unroll
                            for (int x = 0; x < 5; ++x)
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    mma_16bit(d + BN, desc_advance(da, qa[x] * pa + k * a_step), desc_advance(db, qb[x] * pb + k * b_step), idesc,
                                              !first || x > 0 || k > 0);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                mma_16bit(d, desc_advance(da, k * a_step), desc_advance(db, k * b_step), idesc, !first || k > 0);
                        }
                        first = false;
                        tc_commit(&empty[s]);
                        if (++s == kStages) s = 0, ph ^= 1;
                    }
                    if (!ok) break;
                    tc_commit(&acc_full[acc]);
                    if (++acc == 2) acc = 0, acc_ph ^= 1;
                }
            }
            if (!ok) {      // the products issued so far end before the block gives up its memories
                tc_commit(&stopped);
                mbar_drain(&stopped, 0, polls);
            }
        }
    } else if (warp >= 4) {
        const int ew = warp - 4, quad = ew & 3, side = ew >> 2;      // 32 rows of the tile, half of its columns
        float* st = (float*)(base + kFfStageBytes) + ew * kFfStaging;
        int acc = 0, flip = 0;         // flip: the half of the staging area that the next 16-bit block goes through
        uint32_t acc_ph = 0;
        bool ok = true;
        for (int n = 0, u; (u = unit_of(n)) < a.units; ++n) {
            const FfUnit t = ff_unit(a, u, JW);
            const FfProblem& p = *t.p;
            const int64_t row0 = t.i0 + quad * 32;
            const bool rows_here = row0 < p.n_i;
            // a block of columns of this warp's half: 32 of a plain product, 16 of g and as many of u
            constexpr int kCols = FWD ? 16 : 32, kBlocks = JW / 2 / kCols;
            // The copies that this warp has started still read the staging area until they are waited for, and a block goes from units that
            // leave by copies to units that threads write: those wait too (write_block's barrier holds the other lanes back).
            auto staging_free = [&] {
                if (lane == 0) tma_store_wait<0>();
            };
            const float back = scaled(t) && row0 + lane < p.n_i ? unscale_of(p.amax[t.set][row0 + lane]) : 1.f;
            auto emit = [&](int c, const float* given, const float* w) {
                const int col0 = t.j0 + side * (JW / 2) + c * kCols;
                if (!rows_here || col0 >= p.n_j) return;
                char* bytes = (char*)st;
                float unscaled[SCALED ? 32 : 1];
                const float* v = given;
                if constexpr (SCALED) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) unscaled[i] = given[i] * back;
                    v = unscaled;
                }
                if constexpr (FWD) {
                    float g[16], u[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) g[i] = v[i], u[i] = w[i];
                    const bool keep = p.out_map[0] >= 0;
                    if (keep) {
                        staging_free();
                        __syncwarp();
                        uint4 q[4];
                        pack_row(g, q, (const float*)nullptr);
                        put_row(bytes, q);
                        pack_row(u, q, (const float*)nullptr);
                        put_row(bytes + 2048, q);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) tma_store(&a.map[p.out_map[0]], bytes, col0, (int)row0, 0);
                    }
                    if (a.act == CGB200_ACT_RELU) gate<CGB200_ACT_RELU>(g, u);
                    else if (a.act == CGB200_ACT_SILU) gate<CGB200_ACT_SILU>(g, u);
                    else gate<CGB200_ACT_GELU>(g, u);
                    T* h = (T*)p.out[0] + (row0 + lane) * p.n_j + col0;
                    if (p.h_aligned && col0 + 16 <= p.n_j) {
                        if (row0 + lane < p.n_i) {
#pragma unroll
                            for (int j = 0; j < 16 / Chunk<T>::N; ++j) {
                                float x[Chunk<T>::N];
#pragma unroll
                                for (int i = 0; i < Chunk<T>::N; ++i) x[i] = g[j * Chunk<T>::N + i];
                                *(reinterpret_cast<uint4*>(h) + j) = pack16(x, (const T*)nullptr);
                            }
                        }
                    } else {
                        staging_free();
                        write_block<16>(g, st, (T*)p.out[0], row0, p.n_i, p.n_j, col0, p.n_j);
                        fence_proxy_async();
                    }
                } else if (p.splits > 1) {
                    float* part = p.part + ((int64_t)t.split * p.sets + t.set) * p.n_i * p.n_j;
                    staging_free();
                    write_block<32>(v, st, part, row0, p.n_i, p.n_j, col0, p.n_j);
                } else if (p.out_map[t.set] >= 0) {
                    const CUtensorMap* map = &a.map[p.out_map[t.set]];
                    uint4 q[4];
                    if constexpr (sizeof(T) == 2) {
                        if (lane == 0) tma_store_wait<1>();
                        __syncwarp();
                        pack_row(v, q, (const T*)nullptr);
                        put_row(bytes + flip, q);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) tma_store(map, bytes + flip, col0, (int)row0, 0);
                        flip ^= 2048;
                    } else {
                        staging_free();
                        __syncwarp();
                        pack_row(v, q, (const float*)nullptr);
                        put_row(bytes, q);
                        pack_row(v + 16, q, (const float*)nullptr);
                        put_row(bytes + 2048, q);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store(map, bytes, col0, (int)row0, 0);
                            if (col0 + 16 < p.n_j) tma_store(map, bytes + 2048, col0 + 16, (int)row0, 0);
                        }
                    }
                } else if (p.out[t.set] != nullptr) {
                    staging_free();
                    write_block<32>(v, st, (T*)p.out[t.set], row0, p.n_i, p.n_j, col0, p.n_j);
                }
            };
            const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
            if constexpr (PLANES == 1) {
                ok = ok && mbar_wait_warp(&acc_full[acc], acc_ph, failed, polls);
                tc_fence_after();
                const uint32_t d = lanes + acc * kAccCols + side * (JW / 2);
                // not unrolled: the epilogue's code has to stay in the instruction cache beside the two other roles'
#pragma unroll 1
                for (int c = 0; c < kBlocks; ++c) {
                    float v[32];           // a forward's: g, then u
                    if (ok) {
                        if (FWD) tmem_ld16x2(d + c * 16, d + BN / 2 + c * 16, v);
                        else tmem_ld32(d + c * 32, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(kNaNBits);
                    }
                    if (c == kBlocks - 1 && ok) {      // all of this accumulator is in registers or written
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acc_empty[acc]);
                    }
                    emit(c, v, v + 16);
                }
                if (++acc == 2) acc = 0, acc_ph ^= 1;
            } else {
                // 32 columns each of this warp's half of the tile; a forward's: g's, then u's
                constexpr int kSums = JW / 64;
                static_assert(kSums * 64 == JW && kAccCols + JW / 2 + (FWD ? BN / 2 : 0) + 32 * kSums + BN <= kTmemCols,
                              "the last column read (second accumulator, right half, small products) must be one of the block's");
                float sum[FWD ? 2 * kSums : kSums][32];
#pragma unroll
                for (int c = 0; c < (FWD ? 2 * kSums : kSums); ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[c][i] = 0.f;
                for (int it = t.k0; it < t.k1; it += kFlush) {
                    ok = ok && mbar_wait_warp(&acc_full[acc], acc_ph, failed, polls);
                    tc_fence_after();
                    if (ok) {
                        const uint32_t d = lanes + acc * kAccCols + side * (JW / 2);
#pragma unroll
                        for (int c = 0; c < (FWD ? 2 * kSums : kSums); ++c) {
                            const uint32_t at = d + (FWD && c >= kSums ? BN / 2 + (c - kSums) * 32 : c * 32);
                            float lead[32], rest[32];
                            tmem_ld32(at, lead);
                            tmem_ld32(at + BN, rest);
#pragma unroll
                            for (int i = 0; i < 32; ++i) sum[c][i] += lead[i] + rest[i];
                        }
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acc_empty[acc]);
                    }
                    if (++acc == 2) acc = 0, acc_ph ^= 1;
                }
                if (!ok) {
#pragma unroll
                    for (int c = 0; c < (FWD ? 2 * kSums : kSums); ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) sum[c][i] = __uint_as_float(kNaNBits);
                }
#pragma unroll
                for (int c = 0; c < kBlocks; ++c) {
                    if (FWD) emit(c, &sum[c / 2][c % 2 * 16], &sum[kSums + c / 2][c % 2 * 16]);
                    else emit(c, sum[c], sum[c]);
                }
            }
        }
        if (lane == 0) tma_store_wait<0>();      // the stores have read their memory before the block gives it up
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) tmem_dealloc(tmem, kTmemCols);
}

}  // namespace cgb200
