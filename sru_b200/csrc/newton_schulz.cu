// The orthogonalised update of a weight matrix: Newton-Schulz steps on a gradient (or momentum) G,
//
//   X_0 = G / (|G|_F + eps),     X <- a X + (b A + c A^2) X,   A = X X^T,
//
// with X the smaller side first (G^T is iterated where G is taller than wide; the steps commute with the transpose).
// The factor is taken together as X <- M X with M = a I + b A + c A A, so that a step is three products:
//
//   A = X X^T            m x m over n     both operands K-major (rows of X)
//   M = a I + b A + c AA m x m over m     A is symmetric: its rows serve as both operands
//   X = M X              m x n over m     X is the MN-major operand
//
// Iterates, A and M are held in fp16 and accumulated in float32 in tensor memory.  Everything is bounded (|X|_2 <= 1 at
// the start and about 1.2 later, |M| below 10), so fp16's eleven bits are worth more than bf16's range.  But X has small
// elements (1 / sqrt(mn) at the start, 2.8e-4 at 2048 x 6144, and far less beside a few large rows), and fp16 is subnormal
// below 6.1e-5: what is held is 2^k X, k = 12 with the usual coefficients (iterate_exponent).  The powers of two come in with
// the norm and go out where A and the result are rounded, so they cost no rounding.  M's diagonal, which is most of M in the
// last steps, keeps float32's bits as a factor per row (row_factor).  Off exact steps (64-bit steps with these roundings; with bf16
// iterates; 768 x 2304): normal 0.8e-3; 9.0e-3, singular values as 1 / i 4.0e-3; 3.2e-2, as 1 / i^2 2.1e-2; 1.7e-1.  Most of the latter
// is X_0's rounding, which the steps multiply by up to a^steps along the smallest singular directions.
//
// That is enough for a result in bf16, not for one in fp16, which has as many bits as such iterates.  There X, A and M are pairs of
// fp16 (PAIR: the value rounded, and the rest rounded), 22 bits; each product is three, lower times lower left out, in one
// accumulator, and an epilogue stores both parts.  The result is the exact steps rounded once: 2.1e-4 off where eleven bits
// give 0.8e-3 (2.1e-4 and 2e-2 for 1 / i^2).  2048 x 6144 1366 us instead of 495, 256 x 1024 145 instead of 87.  Pairs take a launch
// per product: the one-SM and the one-cluster form below have neither the shared memory nor the bits for them.
//
// The products run on pairs of SMs (cta_group::2, 256 x BN tiles) in a persistent grid over (matrix, tile).  A product costs
// about 5 us beside its multiplications (load latency 1.1, accumulator to shared memory 0.8, stores and end of the grid 2, next
// kernel 1.2), which is most of the time up to 1024 x 1024.  Long products take 440 cycles per 64 of K with 128 columns and 521
// with 256 where the tensor cores need 256 and 512: 24 and 32 KB a SM, close to the 64 bytes a cycle that L2 hands it.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "f32x2.cuh"
#include "tcgen05.cuh"

namespace srub {

namespace {

constexpr int kBK = 64;
constexpr int kABytes = 128 * kBK * 2;          // a CTA's 128 rows of the first operand per stage
constexpr int kEpilogueWarps = 8;               // per quarter of the rows, one for each half of the columns
constexpr int kNsThreads = 64 + 32 * kEpilogueWarps;
constexpr int kMaxParts = 256;                  // partial sums of squares per matrix

enum { kPlain = 0, kCombine = 1 };

struct NsArgs {
    int M, N, K, batch, tiles_m, tiles_n;
    int symmetric;                  // only tiles that reach the diagonal or lie right of it; the others are mirrored
    int per_matrix;                 // tiles computed per matrix
    float ca, cb, cc;
    float by;                       // a plain product's factor: 2^-2k for A, 2^-k for the result
    int last;                       // it writes the caller's matrix
    float *fix;                     // row factors of M (batch, fix_pitch): written with M, applied to M X; pairs have none
    int fix_pitch;
    int *err;
};

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar & 0xFEFFFFFFu), "r"(x), "r"(y), "r"(z)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ uint4 shared_16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ void store_halves(uint32_t at, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

// Eight values times a power of two, two at a time.
__device__ __forceinline__ void times(float (&v)[8], float by) {
    const F2 by2 = f2_splat(by);
#pragma unroll
    for (int j = 0; j < 8; j += 2) f2_split(f2_mul(f2_make(v[j], v[j + 1]), by2), v[j], v[j + 1]);
}

__device__ __forceinline__ void pack_halves(uint32_t (&w)[4], const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
}
// What rounding v to w has left out, rounded in turn: v = w + lo to 22 bits, or to the last bit of fp16's smallest step.
__device__ __forceinline__ void pack_rest(uint32_t (&lo)[4], const uint32_t (&w)[4], const float (&v)[8]) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
        rest[2 * j] = v[2 * j] - h.x;
        rest[2 * j + 1] = v[2 * j + 1] - h.y;
    }
    pack_halves(lo, rest);
}
__device__ __forceinline__ void shared_store(uint32_t at, const uint32_t (&w)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
// Eight values of a row, columns j0 on, at [column][row]: the 32 lanes of a store fill 64 contiguous bytes.
__device__ __forceinline__ void shared_turn(uint32_t turned, int j0, int lane, const uint32_t (&w)[4]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(turned + (j0 + j) * 64 + lane * 2), "h"((uint16_t)(w[j >> 1] >> (16 * (j & 1)))) : "memory");
}

// M = a I + b A + c A A is near a multiple of I in the last steps, so most of what its rounding does is done on the diagonal, where an
// element's error of up to 2^-11 scales its row of M X.  The ratio of the diagonal element to its rounding is kept in
// float32 and applied where M X is rounded: 16 x 300 to 24 x 1000 1.5e-3 to 1.8e-3 off exact steps without, 1.2e-3 to 1.4e-3 with it, 768
// x 2304 1.1e-3 and 0.8e-3; in bf16 results over 200 shapes at most 1.36 times what rounding alone does, 1.7 times without.  It costs
// nothing in one SM, six 2048 x 512 165.4 -> 168.2 us in clusters, 2048 x 6144 0.4 %.
__device__ __forceinline__ float row_factor(float v) {
    const float h = __half2float(__float2half_rn(v));
    return h == 0.0f || isinf(h) ? 1.0f : __fdividef(v, h);
}

// Element i mod N of N values, by halves: log2 N selections deep where a chain of N cost a cluster's product 1 us.
template <int N> __device__ __forceinline__ float pick(const float (&v)[N], int i) {
    float p[N];
#pragma unroll
    for (int j = 0; j < N; ++j) p[j] = v[j];
#pragma unroll
    for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
        for (int j = 0; j < w; ++j) p[j] = i & w ? p[j + w] : p[j];
    return p[0];
}

// Pairs: a product of sums of two is three products, the small ones first, while the accumulator is small and its own
// rounding with it.  Block kb of 3 * blocks -> block of the reduction; *za, *zb: the operands' matrices (upper parts first,
// `batch` of them, then the lower ones).
__device__ __forceinline__ int pair_block(int kb, int blocks, int batch, int *za, int *zb) {
    const int part = kb / blocks;
    *zb += part == 0 ? batch : 0;
    *za += part == 1 ? batch : 0;
    return kb - part * blocks;
}

// Unit -> matrix and tile.  A symmetric product keeps, of 256-row block i, the tiles from column 256 i on.
template <int BN> __device__ __forceinline__ void ns_unit(const NsArgs &g, int unit, int *z, int *mb, int *nb) {
    *z = unit / g.per_matrix;
    int t = unit - *z * g.per_matrix;
    if (g.symmetric) {
        int i = 0, left = g.tiles_n;
        while (t >= left) { t -= left; left -= 256 / BN; ++i; }
        *mb = i;
        *nb = 256 / BN * i + t;
    } else {
        *mb = t / g.tiles_n;
        *nb = t - *mb * g.tiles_n;
    }
}

// TURN: the product may be symmetric.  PAIR: operands and output are pairs.
template <int BN, bool TURN, bool PAIR> struct NsShape {
    static constexpr int kParts = PAIR ? 2 : 1;
    static constexpr int kBBytes = BN / 2 * kBK * 2;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kCols = BN / 2;                        // columns of an epilogue warp
    static constexpr int kOut = 32 * kCols * 2;                 // its 32 rows, boxes of 64 columns
    static constexpr int kTurned = TURN ? kCols * 32 * 2 : 0;      // the same transposed, for the mirrored tile
    static constexpr int kStages = PAIR ? (BN == 128 ? 4 : 3) : BN == 128 ? 6 : TURN ? 3 : 5;
    static constexpr int kBars = 1024;
    static constexpr int kStaging = kParts * (kOut + kTurned);  // of a warp: the parts, the parts transposed
    static constexpr int kSmem = kStages * kStageBytes + kEpilogueWarps * kStaging + 1024 + kBars;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// AMN, BMN: the first operand is stored (K, M), the second (K, N) (MN-major), else (M, K) and (N, K).
//
// Epilogue.  A thread gets one ROW of the accumulator; written from there to global memory every store instruction would
// touch 32 rows, and the four warps of a CTA took 0.5 us per 32 columns that way (half of a 128 x 384 update's time).  The
// warp stages its rows in shared memory in the 128-byte swizzle of the output's tensor map instead and hands boxes of
// 32 x 64 to the copy engine, which clips what lies outside the matrix.  kCombine's A comes the same way into the same
// place, asked for before the accumulator is ready.  A tile right of the diagonal of a symmetric product is staged a second
// time transposed and stored as its mirror image.
template <int BN, bool AMN, bool BMN, int MODE, bool PAIR>
__global__ void __launch_bounds__(kNsThreads, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_t,
                  const __grid_constant__ CUtensorMap map_d, const NsArgs g) {
    constexpr bool TURN = !AMN && !BMN;
    using S = NsShape<BN, TURN, PAIR>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *staging = smem + S::kStages * S::kStageBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(staging + kEpilogueWarps * S::kStaging);
    const uint32_t bar_full = smem_u32(bars);                 // in the leader: loads of both CTAs
    const uint32_t bar_empty = bar_full + 8 * S::kStages;
    const uint32_t bar_tfull = bar_empty + 8 * S::kStages;    // [2]
    const uint32_t bar_tempty = bar_tfull + 16;               // [2] in the leader
    const uint32_t bar_d = bar_tempty + 16;                   // one per epilogue warp
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S::kStages + 4 + kEpilogueWarps);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int nunits = g.per_matrix * g.batch;
    const int blocks = (g.K + kBK - 1) / kBK, nkb = PAIR ? 3 * blocks : blocks;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(bar_tfull + 8 * i, 1); mbar_init(bar_tempty + 8 * i, 2 * kEpilogueWarps); }
        for (int i = 0; i < kEpilogueWarps; ++i) mbar_init(bar_d + 8 * i, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc2(smem_u32(tmem_slot), 2 * BN);
        tmem_relinquish2();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    early_next_kernel();
    previous_kernel_done();

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int unit = pair; unit < nunits && ok; unit += npairs) {
                int z, mb, nb;
                ns_unit<BN>(g, unit, &z, &mb, &nb);
                const int m0 = mb * 256 + (int)rank * 128, n0 = nb * BN + (int)rank * (BN / 2);
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!mbar_wait_bounded(bar_empty + 8 * stage, phase ^ 1)) { atomicExch(g.err, 31); ok = false; break; }
                    const uint32_t full = bar_full + 8 * stage;
                    if (rank == 0) mbar_arrive_expect_tx(full, 2 * S::kStageBytes);
                    const uint32_t sa = smem_u32(smem + stage * S::kStageBytes), sb = sa + kABytes;
                    int za = z, zb = z;
                    const int k0 = (PAIR ? pair_block(kb, blocks, g.batch, &za, &zb) : kb) * kBK;
                    if (!AMN) {
                        tma_load_3d_pair(sa, &map_a, full, k0, m0, za);
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j) tma_load_3d_pair(sa + j * 8192, &map_a, full, m0 + j * 64, k0, za);
                    }
                    if (!BMN) {
                        tma_load_3d_pair(sb, &map_b, full, k0, n0, zb);
                    } else {
#pragma unroll
                        for (int j = 0; j < BN / 128; ++j) tma_load_3d_pair(sb + j * 8192, &map_b, full, n0 + j * 64, k0, zb);
                    }
                    if (++stage == S::kStages) { stage = 0; phase ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            // instruction descriptor: float32 accumulator, fp16 operands, the operands' majors, N / 8, M / 16
            constexpr uint32_t idesc = (1u << 4) | ((AMN ? 1u : 0u) << 15) | ((BMN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((256u >> 4) << 24);
            constexpr uint32_t a_step = AMN ? 2048u : 32u, a_lbo = AMN ? 8192u : 16u;
            constexpr uint32_t b_step = BMN ? 2048u : 32u, b_lbo = BMN ? 8192u : 16u;
            int stage = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int unit = pair; unit < nunits && ok; unit += npairs, ++it) {
                const int acc = it & 1;
                if (!mbar_wait_bounded(bar_tempty + 8 * acc, ((it >> 1) & 1) ^ 1)) { atomicExch(g.err, 32); break; }
                tc_fence_after();
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!mbar_wait_bounded(bar_full + 8 * stage, phase)) { atomicExch(g.err, 33); ok = false; break; }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + stage * S::kStageBytes), sb = sa + kABytes;
#pragma unroll
                    for (int k16 = 0; k16 < kBK / 16; ++k16)
                        tc_mma_pair(tmem_base + acc * BN, make_desc(sa + k16 * a_step, a_lbo, 1024),
                                    make_desc(sb + k16 * b_step, b_lbo, 1024), idesc, (kb | k16) ? 1u : 0u);
                    tc_commit_pair(bar_empty + 8 * stage);
                    if (++stage == S::kStages) { stage = 0; phase ^= 1; }
                }
                if (ok) tc_commit_pair(bar_tfull + 8 * acc);
            }
        }
    } else {
        const int q = warp & 3;                 // TMEM lane quarter: 32 of the CTA's 128 rows
        const int half = (warp - 2) >> 2, first = half * S::kCols;      // half of the columns
        const uint32_t bar_mine = bar_d + 8 * (half * 4 + q);
        const uint32_t tempty_leader = map_to_cta(bar_tempty, 0);
        const uint32_t out = smem_u32(staging + (half * 4 + q) * S::kStaging), turned = out + S::kParts * S::kOut;
        const int parts = PAIR && !g.last ? 2 : 1;          // of the output
        int it = 0;
        for (int unit = pair; unit < nunits; unit += npairs, ++it) {
            int z, mb, nb;
            ns_unit<BN>(g, unit, &z, &mb, &nb);
            const int acc = it & 1;
            const int row0 = mb * 256 + (int)rank * 128 + q * 32, row = row0 + lane;
            const bool mirror = TURN && g.symmetric && mb < nb / (256 / BN);   // the transposed tile is computed by nobody
            if (lane == 0) {
                bulk_wait_read_all();           // the stores of the tile before have left the staging
                if (MODE == kCombine) {
                    mbar_arrive_expect_tx(bar_mine, S::kParts * S::kOut);
#pragma unroll
                    for (int b = 0; b < S::kParts * S::kCols / 64; ++b)
                        tma_load_3d(out + b * 4096, &map_d, bar_mine, nb * BN + first + b % (S::kCols / 64) * 64, row0,
                                    z + b / (S::kCols / 64) * g.batch);
                }
            }
            __syncwarp();
            const float by = !PAIR && BMN && row < g.M ? g.by * __ldcg(g.fix + (int64_t)z * g.fix_pitch + row) : g.by;
            bool ok = mbar_wait_bounded(bar_tfull + 8 * acc, (it >> 1) & 1);
            if (MODE == kCombine) ok = mbar_wait_bounded(bar_mine, it & 1) && ok;
            if (!ok) { if (lane == 0) atomicExch(g.err, 34); break; }
            tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < S::kCols / 32; ++cc) {
                const int col0 = nb * BN + first + cc * 32;
                if (col0 >= g.N) break;
                uint32_t r[32];
                tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN + first + cc * 32, r);
                tmem_ld_wait();
                const uint32_t line = out + (cc >> 1) * 4096 + lane * 128;
                float diagonal = 1.0f;
#pragma unroll
                for (int j0 = 0; j0 < 32; j0 += 8) {
                    const uint32_t at = line + ((((cc & 1) * 4 + j0 / 8) ^ (lane & 7)) << 4);
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[j0 + j]);
                    if (MODE == kCombine) {
                        const uint4 d = shared_16(at);
                        const __half2 *a2 = reinterpret_cast<const __half2 *>(&d);
                        uint4 d_lo = make_uint4(0, 0, 0, 0);
                        if (PAIR) d_lo = shared_16(at + S::kOut);
                        const __half2 *lo2 = reinterpret_cast<const __half2 *>(&d_lo);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            float a = (j & 1) ? __high2float(a2[j >> 1]) : __low2float(a2[j >> 1]);
                            if (PAIR) a += (j & 1) ? __high2float(lo2[j >> 1]) : __low2float(lo2[j >> 1]);
                            v[j] = fmaf(g.cc, v[j], fmaf(g.cb, a, row == col0 + j0 + j ? g.ca : 0.0f));
                        }
                        // in the block of 32 x 32 on the diagonal
                        if (!PAIR && col0 == row0) diagonal = lane >> 3 == j0 / 8 ? pick(v, lane) : diagonal;
                    } else if (!PAIR && AMN) {      // X^T M: M's rows are the result's columns
                        const float4 *f = reinterpret_cast<const float4 *>(g.fix + (int64_t)z * g.fix_pitch + col0 + j0);
                        const float4 f0 = __ldcg(f), f1 = __ldcg(f + 1);
                        times(v, g.by);
                        v[0] *= f0.x; v[1] *= f0.y; v[2] *= f0.z; v[3] *= f0.w;
                        v[4] *= f1.x; v[5] *= f1.y; v[6] *= f1.z; v[7] *= f1.w;
                    } else if ((!PAIR && BMN) || g.by != 1.0f) {
                        times(v, by);
                    }
                    uint32_t w[4];
                    if (MODE == kPlain && !PAIR && g.last) {    // bf16; of pairs the result is fp16, like all before it
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                            w[j] = *reinterpret_cast<const uint32_t *>(&h);
                        }
                    } else {
                        pack_halves(w, v);
                    }
                    shared_store(at, w);
                    if (TURN && mirror) shared_turn(turned, cc * 32 + j0, lane, w);
                    if (PAIR && parts == 2) {
                        uint32_t lo[4];
                        pack_rest(lo, w, v);
                        shared_store(at + S::kOut, lo);
                        if (TURN && mirror) shared_turn(turned + S::kTurned, cc * 32 + j0, lane, lo);
                    }
                }
                if (MODE == kCombine && !PAIR && col0 == row0 && row < g.M) g.fix[(int64_t)z * g.fix_pitch + row] = row_factor(diagonal);
            }
            tc_fence_before();
            fence_proxy_async();                // the staged values become visible to the copy engine
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_cluster_relaxed(tempty_leader + 8 * acc);
                if (row0 < g.M) {
                    for (int part = 0; part < parts; ++part) {
                        const int to = z + part * g.batch;
#pragma unroll
                        for (int b = 0; b < S::kCols / 64; ++b)
                            if (nb * BN + first + b * 64 < g.N)
                                tma_store_3d(&map_c, out + part * S::kOut + b * 4096, nb * BN + first + b * 64, row0, to);
                        if (TURN && mirror && nb * BN + first < g.N)
                            tma_store_3d(&map_t, turned + part * S::kTurned, row0, nb * BN + first, to);
                    }
                }
                bulk_commit();
            }
        }
        if (lane == 0) bulk_wait_read_all();    // the writes themselves are complete when the grid is
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc2(tmem_base, 2 * BN);
    }
}

// A = X X^T of few tiles over a long reduction: S pairs of SMs, one cluster, share a 256 x 128 tile.  Each sums its part of K in
// its own tensor memory; then pair s gets columns [s, s + 1) * 128 / S of the others' sums through distributed shared
// memory, adds them in a fixed order and stores those columns.
template <int S, bool PAIR> struct SplitShape {
    static constexpr int kE = 128 / S;                          // columns that a pair finishes
    static constexpr int kU = kE < 32 ? kE : 32;                // of them, an epilogue warp's
    static constexpr int kStageBytes = kABytes + 64 * kBK * 2, kStages = PAIR ? 4 : 5, kParts = PAIR ? 2 : 1;
    static constexpr int kSums = (S - 1) * 128 * kE * 4;        // the others' sums of its columns
    static constexpr int kOut = 32 * kU * 2;                    // a warp's 32 rows, and once more transposed
    static constexpr int kSmem = kStages * kStageBytes + kSums + kEpilogueWarps * kParts * 2 * kOut + 1024 + 1024;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

template <int S, bool PAIR>
__global__ void __launch_bounds__(kNsThreads, 1)
ns_gram_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_t, const NsArgs g) {
    using P = SplitShape<S, PAIR>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sums = smem_u32(smem + P::kStages * P::kStageBytes);     // [S - 1][kE / 4][128 rows] groups of four columns
    uint8_t *staging = smem + P::kStages * P::kStageBytes + P::kSums;
    uint64_t *bars = reinterpret_cast<uint64_t *>(staging + kEpilogueWarps * P::kParts * 2 * P::kOut);
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * P::kStages, bar_tfull = bar_empty + 8 * P::kStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * P::kStages + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), side = rank & 1;   // in the cluster, in the pair
    const int s = (int)(rank >> 1);
    const uint16_t both = (uint16_t)(3u << (2 * s));
    int z, mb, nb;
    ns_unit<128>(g, blockIdx.x / (2 * S), &z, &mb, &nb);
    const int blocks = (g.K + kBK - 1) / kBK, nkb = PAIR ? 3 * blocks : blocks, kb0 = nkb * s / S, kb1 = nkb * (s + 1) / S;

    if (threadIdx.x == 0) {
        for (int i = 0; i < P::kStages; ++i) { mbar_init(bar_full + 8 * i, 1); mbar_init(bar_empty + 8 * i, 1); }
        mbar_init(bar_tfull, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc2(smem_u32(tmem_slot), 256);      // 128 columns, and room to read 32 from any column on
        tmem_relinquish2();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    early_next_kernel();
    previous_kernel_done();

    const int q = warp & 3, half = (warp - 2) >> 2;             // of an epilogue warp
    const uint32_t tmem_rows = tmem_base + ((uint32_t)(q * 32) << 16);
    const int row = q * 32 + lane;                              // of the CTA's 128
    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_bounded(bar_empty + 8 * stage, phase ^ 1)) { atomicExch(g.err, 31); break; }
                const uint32_t full = bar_full + 8 * stage, sa = smem_u32(smem + stage * P::kStageBytes);
                if (side == 0) mbar_arrive_expect_tx(full, 2 * P::kStageBytes);
                int za = z, zb = z;
                const int k0 = (PAIR ? pair_block(kb, blocks, g.batch, &za, &zb) : kb) * kBK;
                tma_load_3d_pair(sa, &map_a, full, k0, mb * 256 + (int)side * 128, za);
                tma_load_3d_pair(sa + kABytes, &map_b, full, k0, nb * 128 + (int)side * 64, zb);
                if (++stage == P::kStages) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && side == 0) {
            constexpr uint32_t idesc = (1u << 4) | ((128u >> 3) << 17) | ((256u >> 4) << 24);
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_bounded(bar_full + 8 * stage, phase)) { atomicExch(g.err, 33); ok = false; break; }
                tc_fence_after();
                const uint32_t sa = smem_u32(smem + stage * P::kStageBytes), sb = sa + kABytes;
#pragma unroll
                for (int k16 = 0; k16 < kBK / 16; ++k16)
                    tc_mma_pair(tmem_base, make_desc(sa + k16 * 32, 16, 1024), make_desc(sb + k16 * 32, 16, 1024), idesc,
                                (kb > kb0 || k16) ? 1u : 0u);
                tc_commit_pair(bar_empty + 8 * stage, both);
                if (++stage == P::kStages) { stage = 0; phase ^= 1; }
            }
            if (ok) tc_commit_pair(bar_tfull, both);
        }
    } else {
        if (!mbar_wait_bounded(bar_tfull, 0) && lane == 0) atomicExch(g.err, 34);
        tc_fence_after();
    }
    if (warp >= 2) {
#pragma unroll 1
        for (int c0 = half * 32; c0 < 128; c0 += 64) {
            if (S <= 4 && c0 / P::kE == s) continue;            // its own
            uint32_t r[32];
            tmem_ld32(tmem_rows + c0, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                const int to = (c0 + j) / P::kE, slot = s < to ? s : s - 1;
                if (to == s) continue;
                const uint32_t at = map_to_cta(sums + ((slot * (P::kE / 4) + (c0 + j) % P::kE / 4) * 128 + row) * 16, 2 * to + side);
                asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};"
                             ::"r"(at), "r"(r[j]), "r"(r[j + 1]), "r"(r[j + 2]), "r"(r[j + 3]) : "memory");
            }
        }
    }
    __syncwarp();
    cluster_sync_all();         // all sums are here
    if (warp >= 2 && half * P::kU < P::kE) {
        const int c0 = s * P::kE + half * P::kU, col0 = nb * 128 + c0, row0 = mb * 256 + (int)side * 128 + q * 32;
        const bool mirror = mb < nb / 2;
        const uint32_t out = smem_u32(staging + (half * 4 + q) * P::kParts * 2 * P::kOut), turned = out + P::kParts * P::kOut;
        uint32_t r[32];
        tmem_ld32(tmem_rows + c0, r);
        tmem_ld_wait();
#pragma unroll
        for (int j0 = 0; j0 < P::kU; j0 += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[j0 + j]);
#pragma unroll
            for (int slot = 0; slot < S - 1; ++slot)
#pragma unroll
                for (int j = 0; j < 8; j += 4) {
                    const uint4 w = shared_16(sums + ((slot * (P::kE / 4) + (half * P::kU + j0 + j) / 4) * 128 + row) * 16);
                    v[j] += __uint_as_float(w.x);
                    v[j + 1] += __uint_as_float(w.y);
                    v[j + 2] += __uint_as_float(w.z);
                    v[j + 3] += __uint_as_float(w.w);
                }
            times(v, g.by);
            uint32_t w[4];
            pack_halves(w, v);
            shared_store(out + lane * (P::kU * 2) + j0 * 2, w);
            if (mirror) shared_turn(turned, j0, lane, w);
            if (PAIR) {
                uint32_t lo[4];
                pack_rest(lo, w, v);
                shared_store(out + P::kOut + lane * (P::kU * 2) + j0 * 2, lo);
                if (mirror) shared_turn(turned + P::kOut, j0, lane, lo);
            }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0 && row0 < g.M && col0 < g.N) {
            for (int part = 0; part < P::kParts; ++part) {
                tma_store_3d(&map_c, out + part * P::kOut, col0, row0, z + part * g.batch);
                if (mirror) tma_store_3d(&map_t, turned + part * P::kOut, row0, col0, z + part * g.batch);
            }
            bulk_commit();
            bulk_wait_read_all();
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc2(tmem_base, 256);
    }
}

// ---- one cluster per matrix ---------------------------------------------------------------------------------------
// Matrices whose products are shorter than what lies between them: one cluster of SM pairs takes a matrix through all its
// steps, a cluster barrier between the products in place of a launch.  Iterates, A and M stay in L2.  The pairs share the 256 x
// 128 tiles of each product; where X X^T has fewer tiles than the cluster pairs, several pairs share a tile's reduction, as
// above.  A product costs 4 us beside its multiplications (in cycles: first operands 1500, accumulator to shared memory 800, to
// L2 1300, the stores made visible to the copy engine 1000, the barrier 700).
struct NsCluster {
    int m, n, steps;
    float ca, cb, cc;
    __half *x0, *x1, *a, *mm;       // rows of ldx, ldm elements
    int64_t ldx, ldm;
    void *out;                      // the last product's, (m, n) or, turned, (n, m), contiguous; NULL: it goes to x like the others
    int turned, turned_wide;        // turned_wide: its rows are 16-byte aligned
    float gram_by, out_by;          // 2^-2k, 2^-k
    float *fix;                     // row factors of M (batch, fix_pitch)
    int fix_pitch;
    int *err;
};

// What joining the sums of a tile costs beside the sums themselves, in blocks of 64 of the reduction of a 256 x 128 tile (0.26 us),
// from the times with and without it over reductions of 256 to 4096: between the pairs of a cluster that takes a matrix through
// all steps 7 (two pairs) to 13 (four), in the launch of its own 3 (two), 4 to 6 (four) and 5 to 10 (eight).
constexpr int kClusterJoin = 10, kSplitJoin = 4;

// Pairs that share a tile of X X^T.  Five steps with one / two / four pairs, us: 200 x 256 72 / 78 / 83, 200 x 768 83 / 84 / 85, 200 x 1024
// 88 / 87 / 87, 200 x 4096 166 / 137 / 125, 384 x 1152 116 / 120, 384 x 1536 125 / 125.
__host__ __device__ inline int pairs_per_tile(int tiles, int pairs, int blocks) {
    int s = 1;
    while (s < 8 && tiles * s * 2 <= pairs) s *= 2;
    return blocks - blocks / s < kClusterJoin ? 1 : s;
}

// M X on 256 columns a tile where pairs have more than one tile of 128: what L2 hands an SM then keeps the tensor cores busy (521
// cycles a block for twice the columns instead of 440), but the epilogue is twice as long.  Six 512 x 2048 182 -> 166 us.
__host__ __device__ inline bool wide_tiles(int narrow, int pairs, int blocks) { return blocks >= 6 && narrow > pairs; }

struct ClusterShape {
    static constexpr int kStageBytes = kABytes + 128 * kBK * 2, kStages = 5;
    static constexpr int kOut = 32 * 64 * 2;                    // an epilogue warp's 32 rows and 64 columns; once more transposed
    static constexpr int kSmem = kStages * kStageBytes + kEpilogueWarps * 2 * kOut + 1024 + 1024;
    static_assert(kSmem <= 227 * 1024 && 7 * 128 * 16 * 4 <= kEpilogueWarps * 2 * kOut, "shared memory");
};

__global__ void __launch_bounds__(kNsThreads, 1)
ns_cluster_kernel(const __grid_constant__ CUtensorMap map_x0a, const __grid_constant__ CUtensorMap map_x0b,
                  const __grid_constant__ CUtensorMap map_x1a, const __grid_constant__ CUtensorMap map_x1b,
                  const __grid_constant__ CUtensorMap map_aa, const __grid_constant__ CUtensorMap map_ab,
                  const __grid_constant__ CUtensorMap map_ac, const __grid_constant__ CUtensorMap map_ma, const NsCluster g) {
    using P = ClusterShape;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *staging = smem + P::kStages * P::kStageBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(staging + kEpilogueWarps * 2 * P::kOut);
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * P::kStages, bar_tfull = bar_empty + 8 * P::kStages;
    const uint32_t bar_tempty = bar_tfull + 16, bar_d = bar_tempty + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * P::kStages + 4 + kEpilogueWarps);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), side = rank & 1;
    uint32_t ctas;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const int pair = (int)(rank >> 1), pairs = (int)(ctas >> 1), z = (int)(blockIdx.x / ctas);
    const uint16_t both = (uint16_t)(3u << (2 * pair));
    const int rows = (g.m + 255) / 256, cols = (g.m + 127) / 128;
    const int nkb_n = (g.n + kBK - 1) / kBK, nkb_m = (g.m + kBK - 1) / kBK;
    const int square = rows * (cols - rows + 1);                // tiles of a symmetric product
    const int S = pairs_per_tile(square, pairs, nkb_n);

    if (threadIdx.x == 0) {
        for (int i = 0; i < P::kStages; ++i) { mbar_init(bar_full + 8 * i, 1); mbar_init(bar_empty + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(bar_tfull + 8 * i, 1); mbar_init(bar_tempty + 8 * i, 2 * kEpilogueWarps); }
        for (int i = 0; i < kEpilogueWarps; ++i) mbar_init(bar_d + 8 * i, 1);
        fence_mbar_init();
    }
    if (threadIdx.x == 32)
        for (const CUtensorMap *map : {&map_x0a, &map_x0b, &map_x1a, &map_x1b, &map_aa, &map_ab, &map_ac, &map_ma})
            asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    __syncwarp();
    if (warp == 1) {
        tmem_alloc2(smem_u32(tmem_slot), 512);
        tmem_relinquish2();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    early_next_kernel();
    previous_kernel_done();

    // a role's place in the ring and in the accumulators, over all products
    int stage = 0, it = 0;
    uint32_t phase = 0, d_phase = 0;
    bool dead = false;              // a wait gave up: this warp waits for no more mbarriers, but keeps up with the cluster's
    const int q = warp & 3, half = (warp - 2) >> 2;             // of an epilogue warp
    const uint32_t tmem_rows = tmem_base + ((uint32_t)(q * 32) << 16), bar_mine = bar_d + 8 * (half * 4 + q);
    const uint32_t tempty_leader = map_to_cta(bar_tempty, rank & ~1u);
    const uint32_t out = smem_u32(staging + (half * 4 + q) * 2 * P::kOut), turned = out + P::kOut;

    for (int product = 0; product < 3 * g.steps; ++product) {
        const int kind = product % 3, cur = (product / 3) & 1;  // 0: A = X X^T, 1: M, 2: X = M X
        const int split = kind == 0 ? S : 1, mine = pair / split, part = pair % split;
        const bool wide = kind == 2 && wide_tiles(rows * ((g.n + 127) / 128), pairs, nkb_m);
        const int BN = wide ? 256 : 128;
        const int units = kind == 2 ? rows * ((g.n + BN - 1) / BN) : square;
        const int nkb = kind == 0 ? nkb_n : nkb_m, kb0 = nkb * part / split, kb1 = nkb * (part + 1) / split;
        auto tile = [&](int unit, int *mb, int *nb) {
            if (kind == 2) {
                *nb = unit / rows;
                *mb = unit - *nb * rows;
            } else {
                int i = 0, left = cols;
                while (unit >= left) { unit -= left; left -= 2; ++i; }
                *mb = i;
                *nb = 2 * i + unit;
            }
        };
        if (warp == 0) {
            if (lane == 0) {
                const CUtensorMap *ma = kind == 0 ? (cur ? &map_x1a : &map_x0a) : kind == 1 ? &map_aa : &map_ma;
                const CUtensorMap *mbp = kind == 1 ? &map_ab : cur ? &map_x1b : &map_x0b;
                for (int unit = mine; unit < units && !dead; unit += pairs) {
                    int mb, nb;
                    tile(unit, &mb, &nb);
                    const int m0 = mb * 256 + (int)side * 128, n0 = nb * BN + (int)side * (BN / 2);
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!mbar_wait_bounded(bar_empty + 8 * stage, phase ^ 1)) { atomicExch(g.err, 36); dead = true; break; }
                        const uint32_t full = bar_full + 8 * stage, sa = smem_u32(smem + stage * P::kStageBytes);
                        if (side == 0) mbar_arrive_expect_tx(full, 2 * (kABytes + BN / 2 * kBK * 2));
                        tma_load_3d_pair(sa, ma, full, kb * kBK, m0, z);
                        if (kind == 2) {
                            tma_load_3d_pair(sa + kABytes, mbp, full, n0, kb * kBK, z);
                            if (wide) tma_load_3d_pair(sa + kABytes + 8192, mbp, full, n0 + 64, kb * kBK, z);
                        } else tma_load_3d_pair(sa + kABytes, mbp, full, kb * kBK, n0, z);
                        if (++stage == P::kStages) { stage = 0; phase ^= 1; }
                    }
                }
            }
        } else if (warp == 1) {
            if (lane == 0 && side == 0) {
                const uint32_t idesc = (1u << 4) | ((kind == 2 ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((256u >> 4) << 24);
                const uint32_t b_step = kind == 2 ? 2048u : 32u, b_lbo = kind == 2 ? 8192u : 16u;
                for (int unit = mine; unit < units && !dead; unit += pairs, ++it) {
                    const int acc = it & 1;
                    if (!mbar_wait_bounded(bar_tempty + 8 * acc, ((it >> 1) & 1) ^ 1)) { atomicExch(g.err, 37); dead = true; break; }
                    tc_fence_after();
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!mbar_wait_bounded(bar_full + 8 * stage, phase)) { atomicExch(g.err, 38); dead = true; break; }
                        tc_fence_after();
                        const uint32_t sa = smem_u32(smem + stage * P::kStageBytes), sb = sa + kABytes;
#pragma unroll
                        for (int k16 = 0; k16 < kBK / 16; ++k16)
                            tc_mma_pair(tmem_base + acc * 256, make_desc(sa + k16 * 32, 16, 1024),
                                        make_desc(sb + k16 * b_step, b_lbo, 1024), idesc, (kb > kb0 || k16) ? 1u : 0u);
                        tc_commit_pair(bar_empty + 8 * stage, both);
                        if (++stage == P::kStages) { stage = 0; phase ^= 1; }
                    }
                    if (!dead) tc_commit_pair(bar_tfull + 8 * acc, both);
                }
            }
        } else if (split == 1) {
            const bool last = kind == 2 && g.out && product == 3 * g.steps - 1;
            const int64_t ld = kind == 2 ? (last ? g.n : g.ldx) : g.ldm;
            const float by = kind == 0 ? g.gram_by : last ? g.out_by : 1.0f;
            __half *dst = kind == 0 ? g.a + z * (g.m * g.ldm) : kind == 1 ? g.mm + z * (g.m * g.ldm)
                          : last ? static_cast<__half *>(g.out) + z * ((int64_t)g.m * g.n) : (cur ? g.x0 : g.x1) + z * (g.m * g.ldx);
            const int N = kind == 2 ? g.n : g.m;
            for (int unit = mine; unit < units; unit += pairs, ++it) {
                int mb, nb;
                tile(unit, &mb, &nb);
                const int acc = it & 1, row0 = mb * 256 + (int)side * 128 + q * 32, row = row0 + lane;
                const bool turn = last && g.turned, across = turn || (kind < 2 && mb < nb / 2);
                const int64_t ld_across = turn ? g.m : ld;
                if (kind == 1) {
                    if (lane == 0) {
                        if (unit != mine) fence_proxy_async();      // the staging was read with plain loads
                        mbar_arrive_expect_tx(bar_mine, P::kOut);
                        tma_load_3d(out, &map_ac, bar_mine, nb * 128 + half * 64, row0, z);
                    }
                    __syncwarp();
                }
                // written by another CTA of the cluster: past L1, and asked for before the accumulator is ready
                const float row_by = kind == 2 && row < g.m ? by * __ldcg(g.fix + (int64_t)z * g.fix_pitch + row) : by;
                bool ok = dead || mbar_wait_bounded(bar_tfull + 8 * acc, (it >> 1) & 1);
                if (kind == 1) {
                    ok = (dead || mbar_wait_bounded(bar_mine, d_phase)) && ok;
                    d_phase ^= 1;
                }
                if (!ok) {
                    dead = true;
                    if (lane == 0) atomicExch(g.err, 39);
                }
                tc_fence_after();
                for (int c64 = 0; c64 < BN / 2; c64 += 64) {
                    const int first = nb * BN + half * (BN / 2) + c64;
                    uint32_t both_r[2][32];
                    tmem_ld32(tmem_rows + acc * 256 + half * (BN / 2) + c64, both_r[0]);
                    tmem_ld32(tmem_rows + acc * 256 + half * (BN / 2) + c64 + 32, both_r[1]);
                    tmem_ld_wait();
                    if (c64 + 64 == BN / 2) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_relaxed(tempty_leader + 8 * acc);
                    }
                    if (kind == 1 && (row0 & ~63) == first && row < g.m) {      // the diagonal's elements are among these: one per lane
                        const int at = (row0 & 32) + lane;
                        uint16_t a;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(a) : "r"(out + lane * 128 + (((at >> 3) ^ (lane & 7)) << 4) + (at & 7) * 2));
                        float sums[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) sums[j] = __uint_as_float(row0 & 32 ? both_r[1][j] : both_r[0][j]);
                        const float m = fmaf(g.cc, pick(sums, lane), fmaf(g.cb, __half2float(__ushort_as_half(a)), g.ca));
                        g.fix[(int64_t)z * g.fix_pitch + row] = row_factor(m);
                    }
#pragma unroll
                    for (int cc = 0; cc < 2; ++cc) {
                        const int col0 = first + cc * 32;
                        const uint32_t (&r)[32] = both_r[cc];
#pragma unroll
                        for (int j0 = 0; j0 < 32; j0 += 8) {
                            const uint32_t at = out + lane * 128 + (((cc * 4 + j0 / 8) ^ (lane & 7)) << 4);
                            float v[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[j0 + j]);
                            if (kind == 1) {
                                const uint4 d = shared_16(at);
                                const __half2 *a2 = reinterpret_cast<const __half2 *>(&d);
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const float a = (j & 1) ? __high2float(a2[j >> 1]) : __low2float(a2[j >> 1]);
                                    v[j] = fmaf(g.cc, v[j], fmaf(g.cb, a, row == col0 + j0 + j ? g.ca : 0.0f));
                                }
                            } else {
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[j] *= row_by;
                            }
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if (last) {                     // the result is bf16
                                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                                    w[j] = *reinterpret_cast<const uint32_t *>(&h);
                                } else {
                                    const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                                    w[j] = *reinterpret_cast<const uint32_t *>(&h);
                                }
                            }
                            if (!turn) asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                            if (across) {                       // element (row, col) at [col][row]
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(turned + (cc * 32 + j0 + j) * 64 + lane * 2),
                                                 "h"((unsigned short)(w[j >> 1] >> (16 * (j & 1)))) : "memory");
                            }
                        }
                    }
                    __syncwarp();
                    if (!turn) {
                        uint4 w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {           // 4 rows of 128 bytes
                            const int rr = i * 4 + (lane >> 3);
                            w[i] = shared_16(out + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                        }
                        const int rr = lane >> 3, col = first + (lane & 7) * 8;
                        __half *to = dst + (row0 + rr) * ld + col;
#pragma unroll
                        for (int i = 0; i < 8; ++i, to += 4 * ld)
                            if (row0 + rr + i * 4 < g.m && col < N) *reinterpret_cast<uint4 *>(to) = w[i];
                    }
                    if (across) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {           // 8 rows of 64 bytes
                            const int rr = i * 8 + (lane >> 2), col = row0 + (lane & 3) * 8;
                            const uint4 w = shared_16(turned + rr * 64 + (lane & 3) * 16);
                            if (first + rr < N && col < g.m) {
                                __half *to = dst + (first + rr) * ld_across + col;
                                if (!turn || g.turned_wide) {
                                    *reinterpret_cast<uint4 *>(to) = w;
                                } else {
                                    const __half *e = reinterpret_cast<const __half *>(&w);
#pragma unroll
                                    for (int k = 0; k < 8; ++k)
                                        if (col + k < g.m) to[k] = e[k];
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (split > 1) {
            // the pairs' sums of a tile, joined: pair `part` of the tile finishes columns [part, part + 1) * E
            const int E = 128 / split, acc = it & 1;
            const bool on = warp >= 2 && mine < units;
            int mb, nb;
            tile(min(mine, units - 1), &mb, &nb);
            const int row = q * 32 + lane;
            const uint32_t sums = smem_u32(staging);        // [split - 1][E / 4][128 rows] groups of four columns
            if (on) {
                if (!dead && !mbar_wait_bounded(bar_tfull + 8 * acc, (it >> 1) & 1)) {
                    dead = true;
                    if (lane == 0) atomicExch(g.err, 39);
                }
                tc_fence_after();
            }
            if (on) {
#pragma unroll 1
                for (int c0 = half * 16; c0 < 128; c0 += 32) {
                    const int to = c0 / E, slot = part < to ? part : part - 1;
                    if (to == part) continue;
                    uint32_t r[16];
                    tmem_ld16(tmem_rows + acc * 256 + c0, r);
                    tmem_ld_wait();
                    const uint32_t at = map_to_cta(sums + ((slot * (E / 4) + c0 % E / 4) * 128 + row) * 16, 2 * (mine * split + to) + side);
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                        asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};"
                                     ::"r"(at + j / 4 * 2048), "r"(r[j]), "r"(r[j + 1]), "r"(r[j + 2]), "r"(r[j + 3]) : "memory");
                }
            }
            __syncwarp();
            cluster_sync_all();         // all sums are here
            if (on) {
#pragma unroll 1
                for (int e0 = half * 16; e0 < E; e0 += 32) {
                    uint32_t r[16];
                    tmem_ld16(tmem_rows + acc * 256 + part * E + e0, r);
                    tmem_ld_wait();
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                    for (int slot = 0; slot < split - 1; ++slot)
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const uint4 w = shared_16(sums + ((slot * (E / 4) + (e0 + j) / 4) * 128 + row) * 16);
                            v[j] += __uint_as_float(w.x);
                            v[j + 1] += __uint_as_float(w.y);
                            v[j + 2] += __uint_as_float(w.z);
                            v[j + 3] += __uint_as_float(w.w);
                        }
                    const int i = mb * 256 + (int)side * 128 + row, col0 = nb * 128 + part * E + e0;
                    __half *dst = g.a + z * (g.m * g.ldm);
                    __half h[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) h[j] = __float2half_rn(v[j] * g.gram_by);
                    if (i < g.m) {
#pragma unroll
                        for (int j = 0; j < 16; j += 8) {
                            Pack<__half, 8> o;
#pragma unroll
                            for (int k = 0; k < 8; ++k) o.v[k] = h[j + k];
                            if (col0 + j < g.m) *reinterpret_cast<Pack<__half, 8> *>(dst + i * g.ldm + col0 + j) = o;
                        }
                        if (mb < nb / 2) {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (col0 + j < g.m) dst[(col0 + j) * g.ldm + i] = h[j];
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(tempty_leader + 8 * acc);
            }
            if (on) ++it;
        }
        // this product's stores, before the next one's copies
        if (warp >= 2) {
            fence_proxy_async_all();
        }
        __syncwarp();
        cluster_sync_all();
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc2(tmem_base, 512);
    }
}

// ---- norm, first iterate, result ------------------------------------------------------------------------------------
struct NsEdge {
    const void *src;
    void *dst;
    double *part;
    int parts;
    int m, n;                       // the iterate's sizes (m <= n)
    int64_t s_i, s_j, s_b;          // strides of the caller's matrix along the iterate's rows, columns, and batch
    int64_t ldx, x_batch;           // the iterate's row pitch and matrix pitch
    int64_t x_lo;                   // pairs: from an upper part to its lower part; 0: there are none
    int64_t lines, len, pitch;      // the source as lines along its contiguous direction
    bool wide;                      // lines are 16-byte aligned
    double eps;
    float up, down;                 // 2^k, 2^-k
};

// N elements from p + k on, of which those below `len` count (the others are 0); wide: p is 16-byte aligned and N * size a
// multiple of 16.
template <typename T, int N> __device__ __forceinline__ void load_line(float (&v)[N], const T *p, int64_t k, int64_t len, bool wide) {
    if (wide && k + N <= len) {
        Pack<T, N> t = *reinterpret_cast<const Pack<T, N> *>(p + k);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = Cvt<T>::to_f(t.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = k + i < len ? Cvt<T>::to_f(p[k + i]) : 0.0f;
    }
}

// The sum of eight squares in 64 bits.  The largest value's exponent scales them all into [2, 4) and below, where float32
// holds the sum of their squares whatever the range of v (an infinity or a NaN stays one); one conversion to 64 bits for
// eight values, which are slow (a 128 x 384 float32 norm took 6900 cycles of one SM with one per value).
__device__ __forceinline__ double squares(const float (&v)[8]) {
    float top = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    const int ex = min(max((int)(__float_as_uint(top) >> 23), 1), 254);
    const float by = __uint_as_float((uint32_t)(255 - ex) << 23);        // 2^(128 - ex)
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = v[i] * by;
        t = fmaf(x, x, t);
    }
    return (double)t * __hiloint2double((1023 + 2 * (ex - 128)) << 20, 0);
}

// Partial sums of squares in 64 bits (squares of the extremes of bf16 leave float32's range).  Units of UNIT
// elements of a line along the contiguous direction, one warp each, in a fixed order: 2048, or 512 where that leaves most SMs
// without one (256 x 1024 in 64 CTAs instead of 16: 1.3 us less).
template <typename T, int UNIT> __global__ void __launch_bounds__(256) ns_norm_kernel(const NsEdge e) {
    __shared__ double s[8];
    early_next_kernel();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T *g = static_cast<const T *>(e.src) + blockIdx.y * e.s_b;
    const int64_t per = (e.len + UNIT - 1) / UNIT, units = e.lines * per;
    double t = 0.0;
    for (int64_t u = (int64_t)blockIdx.x * 8 + warp; u < units; u += gridDim.x * 8) {
        const int64_t l = u / per, k0 = (u - l * per) * UNIT + lane * 8;
        const T *p = g + l * e.pitch;
#pragma unroll 4
        for (int k = 0; k < UNIT; k += 256) {
            if (k0 + k >= e.len) break;
            float v[8];
            load_line<T, 8>(v, p, k0 + k, e.len, e.wide);
            t += squares(v);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) s[warp] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) t += s[w];
        e.part[(int64_t)blockIdx.y * e.parts + blockIdx.x] = t;
    }
}

// 2^k / (|G|_F + eps) as two factors that are applied one after the other.  The norm of float32 or bf16 values spans 2^-149 to 2^140
// and more, and its reciprocal leaves float32's range at both ends; a takes half of the exponent, b the rest of it and
// the fraction.  a is a power of two, so that there is one rounding.
struct NsScale {
    float a, b;
    __device__ __forceinline__ float operator()(float v) const { return v * a * b; }
};
__device__ __forceinline__ NsScale ns_factors(double norm, float up) {
    const int h = min(max(((__double2hiint(norm) >> 20) & 0x7ff) - 1023, -160), 160) >> 1;
    const float b = (float)(up / norm * __hiloint2double((1023 + h) << 20, 0));
    // a norm of 0 leaves an infinity, and 0 * inf is the definition's 0 / 0; the smallest eps are not 0, and zeros stay zeros
    return {__uint_as_float((uint32_t)(127 - h) << 23), norm > 0.0 ? fminf(b, 3.402823466e38f) : b};
}
// From the partial sums, by every block for itself.
__device__ __forceinline__ NsScale ns_scale(const NsEdge &e, int64_t z, NsScale *shared) {
    early_next_kernel();
    previous_kernel_done();
    if (threadIdx.x < 32) {
        double sum = 0.0;
        for (int p = threadIdx.x; p < e.parts; p += 32) sum += e.part[z * e.parts + p];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) *shared = ns_factors(sqrt(sum) + e.eps, e.up);
    }
    __syncthreads();
    return *shared;
}

// 2^k X_0 in fp16 where the iterate's rows are contiguous in the source: 8 columns per thread.
template <typename T> __global__ void __launch_bounds__(256) ns_first_rows_kernel(const NsEdge e) {
    __shared__ NsScale shared;
    const NsScale scale = ns_scale(e, blockIdx.y, &shared);
    const T *g = static_cast<const T *>(e.src) + blockIdx.y * e.s_b;
    __half *x = static_cast<__half *>(e.dst) + blockIdx.y * e.x_batch;
    const int64_t per = e.ldx / 8, groups = per * e.m;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < groups; u += (int64_t)gridDim.x * 256) {
        const int64_t i = u / per, j = (u - i * per) * 8;
        float v[8];
        load_line<T, 8>(v, g + i * e.s_i, j, e.n, e.wide);
        Pack<__half, 8> h, lo;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float t = scale(v[k]);
            h.v[k] = __float2half_rn(t);
            lo.v[k] = __float2half_rn(t - __half2float(h.v[k]));
        }
        *reinterpret_cast<Pack<__half, 8> *>(x + i * e.ldx + j) = h;
        if (e.x_lo) *reinterpret_cast<Pack<__half, 8> *>(x + e.x_lo + i * e.ldx + j) = lo;
    }
}

// 2^k X_0 where the iterate's columns are contiguous in the source (tall matrices): tiles of 64 x 64 through shared memory.
template <typename T> __global__ void __launch_bounds__(256) ns_first_turned_kernel(const NsEdge e) {
    __shared__ NsScale shared;
    __shared__ float tile[64][65];
    const NsScale scale = ns_scale(e, blockIdx.z, &shared);
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const T *g = static_cast<const T *>(e.src) + blockIdx.z * e.s_b;
    __half *x = static_cast<__half *>(e.dst) + blockIdx.z * e.x_batch;
    const int64_t i0 = (int64_t)blockIdx.y * 64, j0 = (int64_t)blockIdx.x * 64;
#pragma unroll
    for (int k = 0; k < 64; k += 8) {
        const int64_t j = j0 + ty + k;
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
            const int64_t i = i0 + tx + c;
            tile[ty + k][tx + c] = (i < e.m && j < e.n) ? scale(Cvt<T>::to_f(g[i + j * e.s_j])) : 0.0f;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 64; k += 8) {
        const int64_t i = i0 + ty + k, j = j0 + 2 * tx;
        if (i < e.m && j < e.ldx) {         // ldx is a multiple of 8
            const float a = tile[2 * tx][ty + k], b = tile[2 * tx + 1][ty + k];
            const __half2 h = __floats2half2_rn(a, b);
            *reinterpret_cast<__half2 *>(x + i * e.ldx + j) = h;
            if (e.x_lo) *reinterpret_cast<__half2 *>(x + e.x_lo + i * e.ldx + j) = __floats2half2_rn(a - __low2float(h), b - __high2float(h));
        }
    }
}

// The last iterate into the caller's contiguous matrix and type, where the last product cannot write it.
template <typename T> __global__ void __launch_bounds__(256) ns_last_kernel(const NsEdge e) {
    __shared__ float tile[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const __half *x = static_cast<const __half *>(e.src) + blockIdx.z * e.x_batch;
    T *out = static_cast<T *>(e.dst) + blockIdx.z * e.s_b;
    const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;
    const bool across = e.s_j != 1;
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
        const int i = i0 + ty + k, j = j0 + tx;
        float v = 0.0f;
        if (i < e.m && j < e.n) {
            v = __half2float(x[i * e.ldx + j]);
            if (e.x_lo) v += __half2float(x[e.x_lo + i * e.ldx + j]);
            v *= e.down;
        }
        if (across) tile[ty + k][tx] = v;
        else if (i < e.m && j < e.n) out[i * e.s_i + j] = Cvt<T>::from_f(v);
    }
    if (!across) return;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
        const int i = i0 + tx, j = j0 + ty + k;
        if (i < e.m && j < e.n) out[i + j * e.s_j] = Cvt<T>::from_f(tile[tx][ty + k]);
    }
}

// ---- small matrices ------------------------------------------------------------------------------------------------
// One CTA takes a whole matrix through all its steps when the iterate fits in shared memory: X (at most 128 x 768 in fp16)
// as 64-column tiles of 128 rows in the 128-byte swizzle, which the tensor cores read as the K-major operand of X X^T and as
// the MN-major operand of M X alike, and one 128 x 128 matrix that holds A and then, in place, M.  Nothing leaves the SM
// between load and store.  Bound by the latency of the chain (product, accumulator to registers, shared memory, next
// product; 4.5 us a step at 128 x 384 and 35 in all, 92 in a cluster).
constexpr int kSmallM = 128, kSmallN = 768, kSmallThreads = 512;
constexpr int kTileBytes = 128 * 64 * 2;

__device__ __forceinline__ uint32_t tile_at(int row, int col) {     // byte offset of 8 columns' group in the tiles
    return (uint32_t)(col >> 6) * kTileBytes + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) << 4);
}
struct NsSmall {
    NsEdge e;                       // source and sizes; dst is the result
    int64_t o_i, o_j, o_b;          // strides of the result along the iterate's rows, columns, and batch
    int steps;
    float ca, cb, cc, gram_by;      // gram_by: 2^-2k
    bool out_wide;                  // rows of the result are 16-byte aligned
    int *err;
};

template <typename T>
__global__ void __launch_bounds__(kSmallThreads, 1) ns_small_kernel(const NsSmall a) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ double sums[kSmallThreads / 32];
    __shared__ uint64_t bars[2];
    __shared__ uint32_t tmem_slot;
    __shared__ float fix[kSmallM];      // row factors of M
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const NsEdge &e = a.e;
    const int tiles = (e.n + 63) / 64;
    const uint32_t am = smem_u32(smem), x = am + 2 * kTileBytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q = warp & 3, part = warp >> 2, row = q * 32 + lane;      // accumulator row and column part of this thread
    const T *g = static_cast<const T *>(e.src) + blockIdx.x * e.s_b;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&bars[0]), 1);
        mbar_init(smem_u32(&bars[1]), 1);
        fence_mbar_init();
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(&tmem_slot), 512);
        tmem_relinquish();
    }
    // the norm, in 64 bits and a fixed order
    double t = 0.0;
    {
        constexpr int G = 4;            // groups of 8 elements requested together
        const int groups = (int)((e.len + 7) / 8), units = (int)e.lines * groups;
        for (int u0 = threadIdx.x; u0 < units; u0 += G * kSmallThreads) {
            float v[G][8];
#pragma unroll
            for (int k = 0; k < G; ++k) {
                const int u = u0 + k * kSmallThreads, l = e.lines == 1 ? 0 : u / groups;
                load_line<T, 8>(v[k], g + l * e.pitch, (int64_t)(u - l * groups) * 8, u < units ? e.len : 0, e.wide && u < units);
            }
#pragma unroll
            for (int k = 0; k < G; ++k)
                t += squares(v[k]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) sums[warp] = t;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    t = 0.0;
    for (int w = 0; w < kSmallThreads / 32; ++w) t += sums[w];
    const NsScale scale = ns_factors(sqrt(t) + e.eps, e.up);
    // groups of 8 columns, row by row: this thread's first one, and its next from the one before
    const int first_row = (int)threadIdx.x / (tiles * 8), first_col = (int)threadIdx.x - first_row * tiles * 8;
    const int step_rows = kSmallThreads / (tiles * 8), step_cols = kSmallThreads - step_rows * tiles * 8;
    if (e.s_j == 1) {
        constexpr int G = 4;
        // from the last row to the first: what the norm read last is still in L1
        for (int i = kSmallM - 1 - first_row, c = first_col; i >= 0;) {
            float v[G][8];
            int at[G];
#pragma unroll
            for (int k = 0; k < G; ++k) {
                at[k] = i >= 0 ? (int)tile_at(i, c * 8) : -1;
                const bool in = i >= 0 && i < e.m;
                load_line<T, 8>(v[k], g + max(i, 0) * e.s_i, c * 8, in ? e.n : 0, e.wide && in);
                i -= step_rows;
                c += step_cols;
                if (c >= tiles * 8) { c -= tiles * 8; --i; }
            }
#pragma unroll
            for (int k = 0; k < G; ++k) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[k][i] = scale(v[k][i]);
                if (at[k] >= 0) store_halves(x + at[k], v[k]);
            }
        }
    } else {
#pragma unroll 4
        for (int u = threadIdx.x; u < kSmallM * tiles * 64; u += kSmallThreads) {
            const int i = u & (kSmallM - 1), j = u / kSmallM;
            const float v = (i < e.m && j < e.n) ? scale(Cvt<T>::to_f(g[i + j * e.s_j])) : 0.0f;
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(x + tile_at(i, j & ~7) + (j & 7) * 2), "h"(__half_as_ushort(__float2half_rn(v))) : "memory");
        }
    }

    constexpr uint32_t kDesc = (1u << 4) | ((128u >> 4) << 24);
    uint32_t phase[2] = {0, 0};
    bool ok = true;
    // everyone's shared-memory writes are done and visible to the tensor cores
    auto settle = [&]() {
        fence_proxy_async();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    };
    auto arrive = [&](int bar) {
        const bool here = mbar_wait_bounded(smem_u32(&bars[bar]), phase[bar]);
        phase[bar] ^= 1;
        if (!here && lane == 0) atomicExch(a.err, 35);
        ok = __syncthreads_and(here);
        tc_fence_after();
    };
    const F2 cb2 = f2_make(a.cb, a.cb), cc2 = f2_make(a.cc, a.cc);
    const int k_m = (e.m + 15) / 16, k_n = (e.n + 15) / 16, groups = (tiles + 3) / 4;
    settle();
    for (int s = 0; s < a.steps && ok; ++s) {
        // A = X X^T
        if (threadIdx.x == 0) {
            for (int k = 0; k < k_n; ++k) {
                const uint64_t d = make_desc(x + (k >> 2) * kTileBytes + (k & 3) * 32, 16, 1024);
                tc_mma(tmem, d, d, kDesc | ((128u >> 3) << 17), k ? 1u : 0u);
            }
            tc_commit(smem_u32(&bars[0]));
        }
        __syncwarp();
        arrive(0);
        if (!ok) break;
        uint32_t r[32];
        tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + part * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int j0 = 0; j0 < 32; j0 += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[j0 + j]);
            times(v, a.gram_by);
            store_halves(am + tile_at(row, part * 32 + j0), v);
        }
        settle();
        // M = a I + b A + c A A, over A
        if (threadIdx.x == 0) {
            for (int k = 0; k < k_m; ++k) {
                const uint64_t d = make_desc(am + (k >> 2) * kTileBytes + (k & 3) * 32, 16, 1024);
                tc_mma(tmem + 128, d, d, kDesc | ((128u >> 3) << 17), k ? 1u : 0u);
            }
            tc_commit(smem_u32(&bars[0]));
        }
        __syncwarp();
        arrive(0);
        if (!ok) break;
        tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + 128 + part * 32, r);
        tmem_ld_wait();
        float diagonal = 1.0f;
#pragma unroll
        for (int j0 = 0; j0 < 32; j0 += 8) {
            const int col = part * 32 + j0;
            const uint32_t at = am + tile_at(row, col);
            const uint4 w = shared_16(at);
            const __half2 *a2 = reinterpret_cast<const __half2 *>(&w);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float2 old = __half22float2(a2[j >> 1]);
                const F2 m = f2_fma(cc2, f2_make(__uint_as_float(r[j0 + j]), __uint_as_float(r[j0 + j + 1])), f2_mul(cb2, f2_make(old.x, old.y)));
                f2_split(m, v[j], v[j + 1]);
            }
            if (part == q) {                        // the diagonal's block
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += lane == j0 + j ? a.ca : 0.0f;
                diagonal = lane >> 3 == j0 / 8 ? pick(v, lane) : diagonal;
            }
            store_halves(at, v);
        }
        if (part == q) fix[row] = row_factor(diagonal);
        settle();
        // X = M X, 256 columns at a time; a column of the product needs that column of X alone, so it is replaced in place
        auto multiply = [&](int group) {
            if (threadIdx.x == 0) {
                const int n = min(4, tiles - 4 * group) * 64;
                for (int k = 0; k < k_m; ++k)
                    tc_mma(tmem + (group & 1) * 256, make_desc(am + (k >> 2) * kTileBytes + (k & 3) * 32, 16, 1024),
                           make_desc(x + group * 4 * kTileBytes + k * 2048, kTileBytes, 1024),
                           kDesc | (1u << 16) | ((uint32_t)(n >> 3) << 17), k ? 1u : 0u);
                tc_commit(smem_u32(&bars[group & 1]));
            }
            __syncwarp();
        };
        multiply(0);
        if (groups > 1) multiply(1);
        const float row_by = fix[row];
        for (int group = 0; group < groups && ok; ++group) {
            arrive(group & 1);
            if (!ok) break;
            const int col0 = group * 256 + part * 64;
            if (col0 < tiles * 64) {
#pragma unroll
                for (int half = 0; half < 64; half += 32) {
                    tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + (group & 1) * 256 + part * 64 + half, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j0 = 0; j0 < 32; j0 += 8) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[j0 + j]);
                        times(v, row_by);
                        store_halves(x + tile_at(row, col0 + half + j0), v);
                    }
                }
            }
            if (group + 2 < groups) {
                settle();
                multiply(group + 2);
            }
        }
        settle();
    }
    __syncthreads();
    using TO = __nv_bfloat16;
    TO *out = static_cast<TO *>(e.dst) + blockIdx.x * a.o_b;
    if (a.o_j == 1) {
        const __nv_bfloat162 down = __float2bfloat162_rn(e.down);       // exact behind the rounding, too
#pragma unroll 4
        for (int i = first_row, c = first_col; i < e.m;) {
            const int j = c * 8;
            const uint4 w = shared_16(x + tile_at(i, j));
            const __half2 *h = reinterpret_cast<const __half2 *>(&w);
            Pack<TO, 8> o;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = __half22float2(h[k]);
                const __nv_bfloat162 b = __hmul2(__floats2bfloat162_rn(f.x, f.y), down);
                o.v[2 * k] = __low2bfloat16(b);
                o.v[2 * k + 1] = __high2bfloat16(b);
            }
            TO *p = out + i * a.o_i + j;
            if (a.out_wide && j + 8 <= e.n) *reinterpret_cast<Pack<TO, 8> *>(p) = o;
            else
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (j + k < e.n) p[k] = o.v[k];
            i += step_rows;
            c += step_cols;
            if (c >= tiles * 8) { c -= tiles * 8; ++i; }
        }
    } else {
        for (int u = threadIdx.x; u < kSmallM * e.n; u += kSmallThreads) {
            const int i = u & (kSmallM - 1), j = u / kSmallM;
            if (i >= e.m) continue;
            uint16_t h;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(x + tile_at(i, j & ~7) + (j & 7) * 2));
            out[i + j * a.o_j] = Cvt<TO>::from_f(__half2float(__ushort_as_half(h)) * e.down);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct NsPlan {
    int64_t m, n, batch, ldx, ldm;
    int parts;                                // of an iterate, A and M: 2 for pairs
    int64_t fix_pitch;                        // whole tiles, so that factors behind the last row can be read
    size_t part_bytes, x_bytes, a_bytes, fix_bytes;      // each rounded to 256
    size_t total() const { return part_bytes + 2 * x_bytes + 2 * a_bytes + fix_bytes; }
};

NsPlan ns_plan(int64_t batch, int64_t rows, int64_t cols, bool pairs) {
    auto round = [](size_t v) { return (v + 255) / 256 * 256; };
    NsPlan p;
    p.m = std::min(rows, cols); p.n = std::max(rows, cols); p.batch = batch;
    p.ldx = (p.n + 7) / 8 * 8; p.ldm = (p.m + 7) / 8 * 8;
    p.part_bytes = round((size_t)batch * kMaxParts * sizeof(double));
    p.parts = pairs ? 2 : 1;
    p.x_bytes = round((size_t)p.parts * batch * p.m * p.ldx * 2);
    p.a_bytes = round((size_t)p.parts * batch * p.m * p.ldm * 2);
    p.fix_pitch = (p.m + 255) / 256 * 256;
    p.fix_bytes = pairs ? 0 : round((size_t)batch * p.fix_pitch * sizeof(float));
    return p;
}

// k of the held iterates 2^k X: as large as elements up to 2^14 allow, a quarter of fp16's range, and 12 at most, which brings
// the elements of 2048 x 6144 far above its subnormal end.  |x_ij| <= |X|_2 <= r, the largest value that the singular values' map
// p(s) = a s + b s^3 + c s^5 takes step by step from [0, 1] on: its ends and its turning points.
int iterate_exponent(int steps, double a, double b, double c) {
    double r = 1.0;
    auto value = [&](double s) { return std::fabs(s * (a + s * s * (b + s * s * c))); };
    for (int i = 0; i < steps; ++i) {
        double top = value(r);
        auto turn = [&](double square) { if (square > 0.0 && square < r * r) top = std::max(top, value(std::sqrt(square))); };
        // p' = a + 3 b s^2 + 5 c s^4; a root that is no number, or none, is not below r^2
        const double q = -0.5 * (3.0 * b + std::copysign(std::sqrt(9.0 * b * b - 20.0 * a * c), b));
        turn(q / (5.0 * c));
        turn(a / q);
        if (!(top < 16384.0)) return 0;                     // not a number, too
        if (top <= r) break;
        r = top;
    }
    return std::min(12, std::ilogb(16384.0 / r));
}

// (inner, rows, batch) fp16 matrices; boxes of 64 x box_rows elements in the 128-byte swizzle (of 32 elements: as they
// are); outside reads as zero and is not written.
int ns_map(CUtensorMap *map, const void *base, int64_t inner, int64_t rows, int64_t batch, int64_t ld, int box_rows, int box_cols = 64) {
    auto fn = get_encode_fn();
    if (!fn) return set_error(SRU_ERR_CUDA, "cuTensorMapEncodeTiled entry point not found");
    cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)batch};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(ld * rows) * 2};
    cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(SRU_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return 0;
}

// One matrix (or batch) as the products see it: first operand, second operand, output and its mirror image.
struct NsMaps { CUtensorMap a, b, c, t, wide_t; };
int ns_maps(NsMaps *m, const void *base, int64_t inner, int64_t rows, int64_t batch, int64_t ld) {
    int rc = ns_map(&m->a, base, inner, rows, batch, ld, 128);
    if (!rc) rc = ns_map(&m->b, base, inner, rows, batch, ld, 64);
    if (!rc) rc = ns_map(&m->c, base, inner, rows, batch, ld, 32);
    if (!rc) rc = ns_map(&m->t, base, inner, rows, batch, ld, 64, 32);
    if (!rc) rc = ns_map(&m->wide_t, base, inner, rows, batch, ld, 128, 32);
    return rc;
}

template <int BN, bool AMN, bool BMN, int MODE, bool PAIR>
int ns_product(const NsMaps &a, const NsMaps &b, const NsMaps &out, const NsMaps &d, NsArgs g, int sms, cudaStream_t st) {
    using S = NsShape<BN, !AMN && !BMN, PAIR>;
    auto kernel = ns_product_kernel<BN, AMN, BMN, MODE, PAIR>;
    static bool attr_set[64] = {false};
    int dev = 0;
    SRUB_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        SRUB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
        attr_set[dev] = true;
    }
    g.tiles_m = (g.M + 255) / 256;
    g.tiles_n = (g.N + BN - 1) / BN;
    int64_t per = 0;
    if (g.symmetric) for (int i = 0; i < g.tiles_m; ++i) per += g.tiles_n - 256 / BN * i;
    else per = (int64_t)g.tiles_m * g.tiles_n;
    if (per * g.batch > 0x7fffffff) return set_error(SRU_ERR_UNSUPPORTED, "orthogonalize: too many tiles");
    g.per_matrix = (int)per;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(2u * (unsigned)std::min<int64_t>(per * g.batch, sms / 2), 1, 1);
    cfg.blockDim = dim3(kNsThreads, 1, 1);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1] = early_launch();
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SRUB_LAUNCH(&cfg, kernel, AMN ? a.b : a.a, BN == 256 && !BMN ? b.a : b.b, out.c, BN == 256 ? out.wide_t : out.t, d.c, g);
    return 0;
}

// The same product split over the reduction: see choose_split.
template <int S, bool PAIR> int ns_gram_split(const NsMaps &a, const void *out, int64_t ldm, NsArgs g, cudaStream_t st) {
    using P = SplitShape<S, PAIR>;
    auto kernel = ns_gram_split_kernel<S, PAIR>;
    static bool attr_set[64] = {false};
    int dev = 0;
    SRUB_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        SRUB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kSmem));
        SRUB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        attr_set[dev] = true;
    }
    CUtensorMap c, t;
    int rc = ns_map(&c, out, g.M, g.M, P::kParts * g.batch, ldm, 32, P::kU);
    if (!rc) rc = ns_map(&t, out, g.M, g.M, P::kParts * g.batch, ldm, P::kU, 32);
    if (rc) return rc;
    g.tiles_m = (g.M + 255) / 256;
    g.tiles_n = (g.M + 127) / 128;
    g.per_matrix = g.tiles_m * g.tiles_n - g.tiles_m * (g.tiles_m - 1);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(2 * S * g.per_matrix * g.batch), 1, 1);
    cfg.blockDim = dim3(kNsThreads, 1, 1);
    cfg.dynamicSmemBytes = P::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2 * S; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1] = early_launch();
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SRUB_LAUNCH(&cfg, kernel, a.a, a.b, c, t, g);
    return 0;
}

int ns_cluster(const NsMaps &x0, const NsMaps &x1, const NsMaps &a, const NsMaps &m, const NsCluster &g, int64_t batch, int ctas, cudaStream_t st) {
    static bool attr_set[64] = {false};
    int dev = 0;
    SRUB_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        SRUB_CUDA_CHECK(cudaFuncSetAttribute(ns_cluster_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ClusterShape::kSmem));
        SRUB_CUDA_CHECK(cudaFuncSetAttribute(ns_cluster_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(ctas * batch), 1, 1);
    cfg.blockDim = dim3(kNsThreads, 1, 1);
    cfg.dynamicSmemBytes = ClusterShape::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1] = early_launch();
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SRUB_LAUNCH(&cfg, ns_cluster_kernel, x0.a, x0.b, x1.a, x1.b, a.a, a.b, a.c, m.a, g);
    return 0;
}

// Pairs that share a tile of X X^T, by the number of tiles and the 64-element blocks of the reduction: as many as the GPU holds
// clusters for (7, 15 and 33 of 16, 8 and 4 CTAs) while joining the sums is shorter than what that saves.  Five steps in a captured
// graph with 1 / 2 / 4 / 8 pairs: 100 x 4096 144 / 111 / 93 / 87 us, 100 x 2048 104 / 89 / 82 / 82, 200 x 512 82 / 81 / 80 / 85, 200 x 4096
// 153 / 118 / 101 / 95, 512 x 512 99 / 96 / 95 / 99, 512 x 4096 170 / 135 / 117 / 115; with 1 / 2: 1024 x 1024 133 / 126, 1024 x 4096 201 / 168,
// four 300 x 512 (16 tiles) 87 / 88, four 300 x 1536 108 / 101.
int choose_split(int64_t tiles, int64_t blocks) {
    if (tiles <= 7 && blocks >= 64) return 8;
    if (tiles <= 15 && blocks >= 8) return 4;
    if (tiles <= 33 && blocks >= 8) return 2;
    return 1;
}

// CTAs of a cluster that takes a matrix through all its steps, or 0: a launch per product.  Both are counted in blocks (as above)
// that a pair of SMs works through in a step; a tile's epilogue takes as long as six, a wide one's twelve, joined sums what stands
// above.  A cluster where it has at most four more, which its cheaper change from product to product makes up for (2 us a step
// between launches of a stream), and the GPU holds clusters for the batch (7 of 16 CTAs, 15 of 8).  Launches / cluster on a stream,
// us, and what the cluster has more: seven 256 x 512 98 / 81 (-8), 500 x 500 128 / 116 (-6), 130 x 200 91 / 77 (-6), 200 x 768 98 / 89 (-4),
// 256 x 1024 96 / 87 (0), seven 300 x 1500 136 / 132 (0), six 512 x 2048 174 / 160 (0), fifteen 384 x 384 115 / 103 (0); 200 x 2048 106 / 105
// (6), 384 x 1024 109 / 111 (6), 512 x 1024 114 / 118 (6), five 512 x 2048 153 / 159 (12), ten 512 x 512 125 / 130 (16), three 300 x 1500
// 115 / 127 (18), six 600 x 600 143 / 175 (32).  In a captured graph launches follow each other faster, and a cluster is up to 4 us slower
// where the count is 0.
int choose_cluster(int64_t m, int64_t n, int64_t batch, int sms) {
    if (batch > 15) return 0;
    const int64_t ctas = batch <= 7 ? 16 : 8, pairs = ctas / 2, rows = (m + 255) / 256, square = rows * ((m + 127) / 128 - rows + 1);
    const int64_t blocks_m = (m + kBK - 1) / kBK, blocks_n = (n + kBK - 1) / kBK;
    const int64_t narrow = rows * ((n + 127) / 128), wide = rows * ((n + 255) / 256), wide_cost = std::max<int64_t>(blocks_m * 6 / 5, 12);
    auto tiles = [](int64_t count, int64_t pairs, int64_t cost) { return (count + pairs - 1) / pairs * cost; };
    auto gram = [&](int64_t count, int64_t pairs, int split, int join) {
        return tiles(count * split, pairs, std::max<int64_t>(blocks_n / split, 6)) + (split > 1 ? join : 0) +
               tiles(count, pairs, std::max<int64_t>(blocks_m, 6));
    };
    const int64_t here = gram(square, pairs, pairs_per_tile((int)square, (int)pairs, (int)blocks_n), kClusterJoin) +
                         (wide_tiles((int)narrow, (int)pairs, (int)blocks_m) ? tiles(wide, pairs, wide_cost)
                                                                             : tiles(narrow, pairs, std::max<int64_t>(blocks_m, 6)));
    const int64_t launches = gram(square * batch, sms / 2, choose_split(square * batch, blocks_n), kSplitJoin) + tiles(wide * batch, sms / 2, wide_cost);
    return here <= launches + 4 ? (int)ctas : 0;
}

// X X^T and A A.  A 256 x 128 tile takes a pair of SMs about as long as one of 256 x 256 (0.28 us per 64 of the reduction: its
// operands keep shared memory just as busy), but has the shorter epilogue and room for twice the stages.  It is taken where
// the tiles all find a pair of their own, and for small matrices.  Five steps with 128 / 256 columns: 4096 x 4096 1268 / 1120
// us, four 2048 x 2048 745 / 660, six 1024 x 2048 378 / 310, but twelve 700 x 1400 322 / 330.
// Pairs have no room to stage the wider tile's parts and their mirror images.
template <int MODE, bool PAIR> int ns_gram(const NsMaps &a, const NsMaps &out, const NsMaps &d, const NsArgs &g, int sms, cudaStream_t st) {
    const int64_t rows = (g.M + 255) / 256, narrow = rows * ((g.M + 127) / 128) - rows * (rows - 1);
    if (PAIR || narrow * g.batch <= sms / 2 || g.M < 1024) return ns_product<128, false, false, MODE, PAIR>(a, a, out, d, g, sms, st);
    if constexpr (!PAIR) return ns_product<256, false, false, MODE, PAIR>(a, a, out, d, g, sms, st);
    return 0;
}

// One step by a launch per product: X -> next, the last of all to the caller's matrix if `to` is not null.
template <bool PAIR>
int ns_step(const NsMaps &x, const NsMaps &next, const NsMaps &am, const NsMaps &mm, const NsMaps *to, const void *a_buf, const NsPlan &p,
            NsArgs g, float gram_by, float down, bool tall, int sms, cudaStream_t st) {
    g.M = (int)p.m; g.N = (int)p.m; g.K = (int)p.n; g.symmetric = 1; g.by = gram_by;
    const int64_t tiles = ((p.m + 255) / 256) * ((p.m + 127) / 128 - (p.m + 255) / 256 + 1) * p.batch;
    const int split = choose_split(tiles, (PAIR ? 3 : 1) * ((p.n + kBK - 1) / kBK));
    int rc = split == 8 ? ns_gram_split<8, PAIR>(x, a_buf, p.ldm, g, st) : split == 4 ? ns_gram_split<4, PAIR>(x, a_buf, p.ldm, g, st)
             : split == 2 ? ns_gram_split<2, PAIR>(x, a_buf, p.ldm, g, st) : ns_gram<kPlain, PAIR>(x, am, am, g, sms, st);
    g.K = (int)p.m;
    if (!rc) rc = ns_gram<kCombine, PAIR>(am, mm, am, g, sms, st);
    if (rc) return rc;
    g.N = (int)p.n; g.symmetric = 0; g.last = to != nullptr; g.by = to ? down : 1.0f;
    if (!to || !tall) return ns_product<256, false, true, kPlain, PAIR>(mm, x, to ? *to : next, am, g, sms, st);
    g.M = (int)p.n; g.N = (int)p.m;         // X^T = X_before^T M, rows as the caller has them
    return ns_product<128, true, false, kPlain, PAIR>(x, mm, *to, am, g, sms, st);
}

int launch_early(dim3 grid, void (*kernel)(NsEdge), const NsEdge &e, cudaStream_t st) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute early = early_launch();
    cfg.gridDim = grid; cfg.blockDim = dim3(256); cfg.stream = st;
    cfg.attrs = &early; cfg.numAttrs = 1;
    SRUB_LAUNCH(&cfg, kernel, e);
    return 0;
}

template <typename T> int ns_small(const NsSmall &a, int64_t batch, cudaStream_t st) {
    auto kernel = ns_small_kernel<T>;
    const int bytes = (2 + (a.e.n + 63) / 64) * kTileBytes + 1024;
    static bool attr_set[64] = {false};
    int dev = 0;
    SRUB_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        SRUB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 + kSmallN / 64) * kTileBytes + 1024));
        attr_set[dev] = true;
    }
    kernel<<<(unsigned)batch, kSmallThreads, bytes, st>>>(a);
    SRUB_LAUNCHED();
    return 0;
}

}  // namespace

}  // namespace srub

using namespace srub;

extern "C" {

size_t sru_b200_orthogonalize_workspace_bytes_for(int64_t batch, int64_t rows, int64_t cols, int out_dtype) {
    if (batch < 1 || rows < 1 || cols < 1) return 0;
    return ns_plan(batch, rows, cols, out_dtype != SRU_BF16).total();
}

size_t sru_b200_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols) {
    return sru_b200_orthogonalize_workspace_bytes_for(batch, rows, cols, SRU_F16);
}

int sru_b200_orthogonalize(void *out, const void *grad, int64_t batch, int64_t rows, int64_t cols, int64_t stride_batch,
                           int64_t stride_row, int64_t stride_col, int steps, double ca, double cb, double cc, double eps,
                           int grad_dtype, int out_dtype, void *workspace, size_t workspace_bytes, void *stream) {
    if (batch < 0 || rows < 0 || cols < 0 || batch > 65535 || rows > (1 << 20) || cols > (1 << 20))
        return set_error(SRU_ERR_BAD_ARG, "bad sizes: %lld matrices of %lld x %lld", (long long)batch, (long long)rows, (long long)cols);
    if (steps < 0 || steps > 1000) return set_error(SRU_ERR_BAD_ARG, "steps must be 0 to 1000, got %d", steps);
    if (!(eps >= 0.0)) return set_error(SRU_ERR_BAD_ARG, "eps must not be negative");
    if (grad_dtype != SRU_F32 && grad_dtype != SRU_F16 && grad_dtype != SRU_BF16)
        return set_error(SRU_ERR_UNSUPPORTED, "orthogonalize: the matrix must be float32, float16 or bfloat16, got %d", grad_dtype);
    if (out_dtype != SRU_F16 && out_dtype != SRU_BF16)
        return set_error(SRU_ERR_UNSUPPORTED, "orthogonalize: the result is float16 or bfloat16, got %d", out_dtype);
    if (batch == 0 || rows == 0 || cols == 0) return 0;
    if (!out || !grad) return set_error(SRU_ERR_BAD_ARG, "orthogonalize: a required pointer is null");
    if (stride_col != 1 && stride_row != 1) return set_error(SRU_ERR_BAD_ARG, "orthogonalize: rows or columns must be contiguous");
    const bool pairs = out_dtype == SRU_F16;
    const NsPlan p = ns_plan(batch, rows, cols, pairs);
    if (!workspace || workspace_bytes < p.total() || reinterpret_cast<uintptr_t>(workspace) % 256)
        return set_error(SRU_ERR_WORKSPACE, "256-byte aligned workspace of %zu bytes needed, %zu given", p.total(), workspace_bytes);
    if (int rc = ensure_context()) return rc;
    int dev = 0, sms = 0;
    SRUB_CUDA_CHECK(cudaGetDevice(&dev));
    SRUB_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    int *err = device_error_flag();
    if (!err) return set_error(SRU_ERR_CUDA, "device error flag unavailable");
    cudaStream_t st = static_cast<cudaStream_t>(stream);

    char *ws = static_cast<char *>(workspace);
    double *part = reinterpret_cast<double *>(ws);
    __half *x[2] = {reinterpret_cast<__half *>(ws + p.part_bytes), reinterpret_cast<__half *>(ws + p.part_bytes + p.x_bytes)};
    __half *a_buf = reinterpret_cast<__half *>(ws + p.part_bytes + 2 * p.x_bytes);
    __half *m_buf = reinterpret_cast<__half *>(ws + p.part_bytes + 2 * p.x_bytes + p.a_bytes);
    float *fix = reinterpret_cast<float *>(ws + p.part_bytes + 2 * p.x_bytes + 2 * p.a_bytes);

    const bool tall = rows > cols;
    NsEdge e;
    memset(&e, 0, sizeof(e));
    e.src = grad; e.dst = x[0]; e.part = part;
    e.m = (int)p.m; e.n = (int)p.n;
    e.s_i = tall ? stride_col : stride_row; e.s_j = tall ? stride_row : stride_col; e.s_b = stride_batch;
    e.ldx = p.ldx; e.x_batch = p.m * p.ldx; e.x_lo = pairs ? batch * p.m * p.ldx : 0; e.eps = eps;
    const int k = iterate_exponent(steps, ca, cb, cc);
    e.up = std::ldexp(1.0f, k); e.down = std::ldexp(1.0f, -k);
    const float gram_by = e.down * e.down;
    const bool turned = e.s_j != 1;
    e.lines = turned ? p.n : p.m; e.len = turned ? p.m : p.n; e.pitch = turned ? e.s_j : e.s_i;
    const int64_t size = (int64_t)dtype_size(grad_dtype);
    e.wide = reinterpret_cast<uintptr_t>(grad) % 16 == 0 && e.pitch * size % 16 == 0 && (batch == 1 || e.s_b * size % 16 == 0);
    if (e.pitch == e.len || e.lines == 1) { e.len *= e.lines; e.lines = 1; e.pitch = 0; }       // one line
    const int unit = e.lines * ((e.len + 2047) / 2048) * batch < sms * 8 ? 512 : 2048;
    e.parts = (int)std::min<int64_t>((e.lines * ((e.len + unit - 1) / unit) + 7) / 8, kMaxParts);
    const dim3 norm_grid((unsigned)e.parts, (unsigned)batch);
    if (!pairs && p.m <= kSmallM && p.n <= kSmallN) {
        NsSmall a;
        memset(&a, 0, sizeof(a));
        a.e = e; a.e.dst = out;
        a.o_i = tall ? 1 : cols; a.o_j = tall ? cols : 1; a.o_b = rows * cols;
        a.steps = steps; a.ca = (float)ca; a.cb = (float)cb; a.cc = (float)cc; a.gram_by = gram_by; a.err = err;
        a.out_wide = cols % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
        return grad_dtype == SRU_F32 ? ns_small<float>(a, batch, st) : grad_dtype == SRU_F16 ? ns_small<__half>(a, batch, st)
                                                                                          : ns_small<__nv_bfloat16>(a, batch, st);
    }
    auto begin = [&](auto t) -> int {
        using T = decltype(t);
        if (unit == 512) ns_norm_kernel<T, 512><<<norm_grid, 256, 0, st>>>(e);
        else ns_norm_kernel<T, 2048><<<norm_grid, 256, 0, st>>>(e);
        SRUB_LAUNCHED();
        if (turned) {
            const dim3 grid((unsigned)((p.ldx + 63) / 64), (unsigned)((p.m + 63) / 64), (unsigned)batch);
            return launch_early(grid, ns_first_turned_kernel<T>, e, st);
        } else {
            const dim3 grid((unsigned)std::min<int64_t>((p.m * p.ldx / 8 + 255) / 256, sms * 8), (unsigned)batch);
            return launch_early(grid, ns_first_rows_kernel<T>, e, st);
        }
    };
    if (int rc = grad_dtype == SRU_F32 ? begin(float()) : grad_dtype == SRU_F16 ? begin(__half()) : begin(__nv_bfloat16())) return rc;

    // The last product writes the caller's matrix itself where its rows are 16-byte aligned (a cluster's turned one, always).
    const int ctas = steps > 0 && !pairs ? choose_cluster(p.m, p.n, batch, sms) : 0;
    const bool aligned = steps > 0 && cols % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0, direct = aligned || (ctas && tall);
    NsMaps xm[2], am, mm, om;
    if (aligned)
        if (int rc = ns_maps(&om, out, cols, rows, batch, cols)) return rc;
    if (steps > 0) {
        int rc = ns_maps(&am, a_buf, p.m, p.m, p.parts * batch, p.ldm);
        if (!rc) rc = ns_maps(&mm, m_buf, p.m, p.m, p.parts * batch, p.ldm);
        for (int i = 0; i < 2 && !rc; ++i) rc = ns_maps(&xm[i], x[i], p.n, p.m, p.parts * batch, p.ldx);
        if (rc) return rc;
    }
    if (ctas) {
        NsCluster g;
        memset(&g, 0, sizeof(g));
        g.m = (int)p.m; g.n = (int)p.n; g.steps = steps;
        g.ca = (float)ca; g.cb = (float)cb; g.cc = (float)cc;
        g.x0 = x[0]; g.x1 = x[1]; g.a = a_buf; g.mm = m_buf; g.ldx = p.ldx; g.ldm = p.ldm;
        g.out = direct ? out : nullptr; g.turned = tall; g.turned_wide = aligned; g.err = err;
        g.gram_by = gram_by; g.out_by = e.down; g.fix = fix; g.fix_pitch = (int)p.fix_pitch;
        if (int rc = ns_cluster(xm[0], xm[1], am, mm, g, batch, ctas, st)) return rc;
    }
    for (int s = 0; s < steps && !ctas; ++s) {
        const int cur = s & 1;
        NsArgs g;
        memset(&g, 0, sizeof(g));
        g.batch = (int)batch; g.err = err;
        g.ca = (float)ca; g.cb = (float)cb; g.cc = (float)cc; g.fix = fix; g.fix_pitch = (int)p.fix_pitch;
        const NsMaps *to = s == steps - 1 && direct ? &om : nullptr;
        const int rc = pairs ? ns_step<true>(xm[cur], xm[cur ^ 1], am, mm, to, a_buf, p, g, gram_by, e.down, tall, sms, st)
                             : ns_step<false>(xm[cur], xm[cur ^ 1], am, mm, to, a_buf, p, g, gram_by, e.down, tall, sms, st);
        if (rc) return rc;
    }
    if (direct) return 0;
    const dim3 tile_grid((unsigned)((p.ldx + 31) / 32), (unsigned)((p.m + 31) / 32), (unsigned)batch);
    e.src = x[steps & 1]; e.dst = out;
    e.s_i = tall ? 1 : cols; e.s_j = tall ? cols : 1; e.s_b = rows * cols;
    if (out_dtype == SRU_F16) ns_last_kernel<__half><<<tile_grid, 256, 0, st>>>(e);
    else ns_last_kernel<__nv_bfloat16><<<tile_grid, 256, 0, st>>>(e);
    SRUB_LAUNCHED();
    return 0;
}

}  // extern "C"
