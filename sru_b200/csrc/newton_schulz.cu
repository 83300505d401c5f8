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
// the start and about 1.2 later, |M| below 10), so fp16's eleven bits are worth more than bf16's range: on
// gradients with a decaying spectrum the result is 1.2e-3 off the exact steps against 1.0e-2 with bf16 iterates.
//
// The products run on pairs of SMs (cta_group::2, 256 x BN tiles) in a persistent grid over (matrix, tile).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "tcgen05.cuh"

namespace srub {

namespace {

constexpr int kBK = 64;
constexpr int kABytes = 128 * kBK * 2;          // a CTA's 128 rows of the first operand per stage
constexpr int kNsThreads = 192;
constexpr int kMaxParts = 128;                  // partial sums of squares per matrix

enum { kPlain = 0, kCombine = 1 };

struct NsArgs {
    __half *c;                      // product; rows ldc apart, matrices c_batch apart
    const __half *d;                // kCombine: A, laid out as c
    int64_t ldc, c_batch;
    int M, N, K, batch, tiles_m, tiles_n;
    int symmetric;                  // only tiles that reach the diagonal or lie right of it; the others are mirrored
    int per_matrix;                 // tiles computed per matrix
    float ca, cb, cc;
    int *err;
};

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar & 0xFEFFFFFFu), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Unit -> matrix and tile.  A symmetric product keeps, of 256-row block i, the 128-column tiles from 2 i on.
__device__ __forceinline__ void ns_unit(const NsArgs &g, int unit, int *z, int *mb, int *nb) {
    *z = unit / g.per_matrix;
    int t = unit - *z * g.per_matrix;
    if (g.symmetric) {
        int i = 0, left = g.tiles_n;
        while (t >= left) { t -= left; left -= 2; ++i; }
        *mb = i;
        *nb = 2 * i + t;
    } else {
        *mb = t / g.tiles_n;
        *nb = t - *mb * g.tiles_n;
    }
}

template <int BN> struct NsShape {
    static constexpr int kBBytes = BN / 2 * kBK * 2;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kStages = BN == 128 ? 8 : 6;
    static constexpr int kSmem = kStages * kStageBytes + 1024 + 256;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// BMN: the second operand is stored (K, N) (MN-major), else (N, K).
template <int BN, bool BMN, int MODE>
__global__ void __launch_bounds__(kNsThreads, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const NsArgs g) {
    using S = NsShape<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kStages * S::kStageBytes);
    const uint32_t bar_full = smem_u32(bars);                 // in the leader: loads of both CTAs
    const uint32_t bar_empty = bar_full + 8 * S::kStages;
    const uint32_t bar_tfull = bar_empty + 8 * S::kStages;    // [2]
    const uint32_t bar_tempty = bar_tfull + 16;               // [2] in the leader
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S::kStages + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int nunits = g.per_matrix * g.batch;
    const int nkb = (g.K + kBK - 1) / kBK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(bar_tfull + 8 * i, 1); mbar_init(bar_tempty + 8 * i, 8); }
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

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int unit = pair; unit < nunits && ok; unit += npairs) {
                int z, mb, nb;
                ns_unit(g, unit, &z, &mb, &nb);
                const int m0 = mb * 256 + (int)rank * 128, n0 = nb * BN + (int)rank * (BN / 2);
                for (int kb = 0; kb < nkb; ++kb) {
                    if (!mbar_wait_bounded(bar_empty + 8 * stage, phase ^ 1)) { atomicExch(g.err, 31); ok = false; break; }
                    const uint32_t full = bar_full + 8 * stage;
                    if (rank == 0) mbar_arrive_expect_tx(full, 2 * S::kStageBytes);
                    const uint32_t sa = smem_u32(smem + stage * S::kStageBytes), sb = sa + kABytes;
                    tma_load_3d_pair(sa, &map_a, full, kb * kBK, m0, z);
                    if (!BMN) {
                        tma_load_3d_pair(sb, &map_b, full, kb * kBK, n0, z);
                    } else {
#pragma unroll
                        for (int j = 0; j < BN / 128; ++j) tma_load_3d_pair(sb + j * 8192, &map_b, full, n0 + j * 64, kb * kBK, z);
                    }
                    if (++stage == S::kStages) { stage = 0; phase ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            // instruction descriptor: float32 accumulator, fp16 operands, second operand's major, N / 8, M / 16
            constexpr uint32_t idesc = (1u << 4) | ((BMN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((256u >> 4) << 24);
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
                        tc_mma_pair(tmem_base + acc * BN, make_desc(sa + k16 * 32, 16, 1024),
                                    make_desc(sb + k16 * b_step, b_lbo, 1024), idesc, (kb | k16) ? 1u : 0u);
                    tc_commit_pair(bar_empty + 8 * stage);
                    if (++stage == S::kStages) { stage = 0; phase ^= 1; }
                }
                if (ok) tc_commit_pair(bar_tfull + 8 * acc);
            }
        }
    } else {
        const int q = warp & 3;                 // TMEM lane quarter: 32 of the CTA's 128 rows
        const uint32_t tempty_leader = map_to_cta(bar_tempty, 0);
        int it = 0;
        for (int unit = pair; unit < nunits; unit += npairs, ++it) {
            int z, mb, nb;
            ns_unit(g, unit, &z, &mb, &nb);
            const int acc = it & 1;
            if (!mbar_wait_bounded(bar_tfull + 8 * acc, (it >> 1) & 1)) { if (lane == 0) atomicExch(g.err, 34); break; }
            tc_fence_after();
            const int row = mb * 256 + (int)rank * 128 + q * 32 + lane;
            const bool mirror = g.symmetric && 2 * mb < (nb & ~1);      // the transposed tile is computed by nobody
            __half *c = g.c + (int64_t)z * g.c_batch;
            const __half *d = MODE == kCombine ? g.d + (int64_t)z * g.c_batch : nullptr;
#pragma unroll 1
            for (int cc = 0; cc < BN / 32; ++cc) {
                const int col0 = nb * BN + cc * 32;
                if (col0 >= g.N) break;
                uint32_t r[32];
                tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN + cc * 32, r);
                tmem_ld_wait();
                // rows are padded to 8 elements: a group of 8 that starts inside the matrix is inside its row
#pragma unroll
                for (int j0 = 0; j0 < 32; j0 += 8) {
                    const bool in = row < g.M && col0 + j0 < g.N;
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r[j0 + j]);
                    if (MODE == kCombine && in) {
                        const Pack<__half, 8> a = *reinterpret_cast<const Pack<__half, 8> *>(d + row * g.ldc + col0 + j0);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            v[j] = fmaf(g.cc, v[j], fmaf(g.cb, __half2float(a.v[j]), row == col0 + j0 + j ? g.ca : 0.0f));
                    }
                    if (in) store8<__half>(c + row * g.ldc + col0 + j0, v);
                    if (g.symmetric) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) r[j0 + j] = __float_as_uint(v[j]);
                    }
                }
                if (mirror) {
                    // element (row, col) again at (col, row): lanes hold consecutive rows; two rows to a 4-byte store,
                    // even lanes store column k, odd lanes column k + 1
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const float mine = __uint_as_float(lane & 1 ? r[k + 1] : r[k]);
                        const float give = __uint_as_float(lane & 1 ? r[k] : r[k + 1]);
                        const float got = __shfl_xor_sync(0xffffffffu, give, 1);
                        const int col = col0 + k + (lane & 1);
                        const __half2 two = lane & 1 ? __floats2half2_rn(got, mine) : __floats2half2_rn(mine, got);
                        if (col < g.N && (row & ~1) < g.M) *reinterpret_cast<__half2 *>(c + col * g.ldc + (row & ~1)) = two;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty_leader + 8 * acc);
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc2(tmem_base, 2 * BN);
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
    double eps;
};

// Partial sums of squares in 64 bits (squares of the extremes of bf16 leave float32's range); one warp per line along
// the contiguous direction.
template <typename T> __global__ void __launch_bounds__(256) ns_norm_kernel(const NsEdge e) {
    __shared__ double s[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool across = e.s_j != 1;                       // lines run along i
    const int lines = across ? e.n : e.m, len = across ? e.m : e.n;
    const int64_t pitch = across ? e.s_j : e.s_i;
    const T *g = static_cast<const T *>(e.src) + blockIdx.y * e.s_b;
    double sum = 0.0;
    for (int l = blockIdx.x * 8 + warp; l < lines; l += gridDim.x * 8) {
        const T *p = g + l * pitch;
        for (int k = lane; k < len; k += 32) {
            const double v = (double)Cvt<T>::to_f(p[k]);
            sum = fma(v, v, sum);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) sum += s[w];
        e.part[(int64_t)blockIdx.y * e.parts + blockIdx.x] = sum;
    }
}

// X_0 in fp16, tiles of 32 x 32 through shared memory: the source is read along its contiguous direction.
template <typename T> __global__ void __launch_bounds__(256) ns_first_kernel(const NsEdge e) {
    __shared__ float tile[32][33];
    __shared__ float scale;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    if (ty == 0) {
        double sum = 0.0;
        for (int p = tx; p < e.parts; p += 32) sum += e.part[(int64_t)blockIdx.z * e.parts + p];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (tx == 0) scale = (float)(1.0 / (sqrt(sum) + e.eps));
    }
    __syncthreads();
    const T *g = static_cast<const T *>(e.src) + blockIdx.z * e.s_b;
    __half *x = static_cast<__half *>(e.dst) + blockIdx.z * e.x_batch;
    const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;
    const bool across = e.s_j != 1;
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
        const int i = i0 + (across ? tx : ty + k), j = j0 + (across ? ty + k : tx);
        const float v = (i < e.m && j < e.n) ? Cvt<T>::to_f(g[i * e.s_i + j * e.s_j]) * scale : 0.0f;
        if (across) tile[tx][ty + k] = v;
        else tile[ty + k][tx] = v;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
        const int i = i0 + ty + k, j = j0 + tx;
        if (i < e.m && j < e.ldx) x[i * e.ldx + j] = __float2half_rn(tile[ty + k][tx]);
    }
}

// The last iterate into the caller's contiguous matrix and type.
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
        const float v = (i < e.m && j < e.n) ? __half2float(x[i * e.ldx + j]) : 0.0f;
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

// ---- host side ------------------------------------------------------------------------------------------------------
struct NsPlan {
    int64_t m, n, batch, ldx, ldm;
    size_t part_bytes, x_bytes, a_bytes;      // each rounded to 256
    size_t total() const { return part_bytes + 2 * x_bytes + 2 * a_bytes; }
};

NsPlan ns_plan(int64_t batch, int64_t rows, int64_t cols) {
    auto round = [](size_t v) { return (v + 255) / 256 * 256; };
    NsPlan p;
    p.m = std::min(rows, cols); p.n = std::max(rows, cols); p.batch = batch;
    p.ldx = (p.n + 7) / 8 * 8; p.ldm = (p.m + 7) / 8 * 8;
    p.part_bytes = round((size_t)batch * kMaxParts * sizeof(double));
    p.x_bytes = round((size_t)batch * p.m * p.ldx * 2);
    p.a_bytes = round((size_t)batch * p.m * p.ldm * 2);
    return p;
}

// (inner, rows, batch) fp16 matrices; boxes of 64 x box_rows elements, 128-byte swizzle; outside reads as zero.
int ns_map(CUtensorMap *map, const void *base, int64_t inner, int64_t rows, int64_t batch, int64_t ld, int box_rows) {
    auto fn = get_encode_fn();
    if (!fn) return set_error(SRU_ERR_CUDA, "cuTensorMapEncodeTiled entry point not found");
    cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)batch};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(ld * rows) * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(SRU_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return 0;
}

template <int BN, bool BMN, int MODE>
int ns_product(const CUtensorMap &map_a, const CUtensorMap &map_b, NsArgs g, int sms, cudaStream_t st) {
    auto kernel = ns_product_kernel<BN, BMN, MODE>;
    static bool attr_set[64] = {false};
    int dev = 0;
    SRUB_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        SRUB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NsShape<BN>::kSmem));
        attr_set[dev] = true;
    }
    g.tiles_m = (g.M + 255) / 256;
    g.tiles_n = (g.N + BN - 1) / BN;
    int64_t per = 0;
    if (g.symmetric) for (int i = 0; i < g.tiles_m; ++i) per += g.tiles_n - 2 * i;
    else per = (int64_t)g.tiles_m * g.tiles_n;
    if (per * g.batch > 0x7fffffff) return set_error(SRU_ERR_UNSUPPORTED, "orthogonalize: too many tiles");
    g.per_matrix = (int)per;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(2u * (unsigned)std::min<int64_t>(per * g.batch, sms / 2), 1, 1);
    cfg.blockDim = dim3(kNsThreads, 1, 1);
    cfg.dynamicSmemBytes = NsShape<BN>::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SRUB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, g));
    return 0;
}

}  // namespace

}  // namespace srub

using namespace srub;

extern "C" {

size_t sru_b200_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols) {
    if (batch < 1 || rows < 1 || cols < 1) return 0;
    return ns_plan(batch, rows, cols).total();
}

int sru_b200_orthogonalize(void *out, const void *grad, int64_t batch, int64_t rows, int64_t cols, int64_t stride_batch,
                           int64_t stride_row, int64_t stride_col, int steps, double a, double b, double c, double eps,
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
    const NsPlan p = ns_plan(batch, rows, cols);
    if (!workspace || workspace_bytes < p.total() || reinterpret_cast<uintptr_t>(workspace) % 256)
        return set_error(SRU_ERR_WORKSPACE, "256-byte aligned workspace of %zu bytes needed, %zu given", p.total(), workspace_bytes);
    if (int rc = ensure_context()) return rc;
    int dev = 0, sms = 148;
    SRUB_CUDA_CHECK(cudaGetDevice(&dev));
    SRUB_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    int *err = device_error_flag();
    if (!err) return set_error(SRU_ERR_CUDA, "device error flag unavailable");
    cudaStream_t st = static_cast<cudaStream_t>(stream);

    char *ws = static_cast<char *>(workspace);
    double *part = reinterpret_cast<double *>(ws);
    __half *x[2] = {reinterpret_cast<__half *>(ws + p.part_bytes), reinterpret_cast<__half *>(ws + p.part_bytes + p.x_bytes)};
    __half *am = reinterpret_cast<__half *>(ws + p.part_bytes + 2 * p.x_bytes);
    __half *mm = reinterpret_cast<__half *>(ws + p.part_bytes + 2 * p.x_bytes + p.a_bytes);

    const bool tall = rows > cols;
    NsEdge e;
    memset(&e, 0, sizeof(e));
    e.src = grad; e.dst = x[0]; e.part = part;
    e.m = (int)p.m; e.n = (int)p.n;
    e.s_i = tall ? stride_col : stride_row; e.s_j = tall ? stride_row : stride_col; e.s_b = stride_batch;
    e.ldx = p.ldx; e.x_batch = p.m * p.ldx; e.eps = eps;
    const int64_t lines = e.s_j != 1 ? p.n : p.m;
    e.parts = (int)std::min<int64_t>((lines + 7) / 8, kMaxParts);
    const dim3 norm_grid((unsigned)e.parts, (unsigned)batch);
    const dim3 tile_grid((unsigned)((p.ldx + 31) / 32), (unsigned)((p.m + 31) / 32), (unsigned)batch);
    auto begin = [&](auto t) {
        using T = decltype(t);
        ns_norm_kernel<T><<<norm_grid, 256, 0, st>>>(e);
        ns_first_kernel<T><<<tile_grid, 256, 0, st>>>(e);
    };
    if (grad_dtype == SRU_F32) begin(float());
    else if (grad_dtype == SRU_F16) begin(__half());
    else begin(__nv_bfloat16());
    SRUB_CUDA_CHECK(cudaGetLastError());

    CUtensorMap xa[2], xb[2], aa, ab, ma;             // as first operand (128-row boxes), as second (64)
    int rc = 0;
    for (int i = 0; i < 2 && steps > 0; ++i) {
        if ((rc = ns_map(&xa[i], x[i], p.n, p.m, batch, p.ldx, 128))) return rc;
        if ((rc = ns_map(&xb[i], x[i], p.n, p.m, batch, p.ldx, 64))) return rc;
    }
    if (steps > 0) {
        if ((rc = ns_map(&aa, am, p.m, p.m, batch, p.ldm, 128))) return rc;
        if ((rc = ns_map(&ab, am, p.m, p.m, batch, p.ldm, 64))) return rc;
        if ((rc = ns_map(&ma, mm, p.m, p.m, batch, p.ldm, 128))) return rc;
    }
    for (int s = 0; s < steps; ++s) {
        const int cur = s & 1;
        NsArgs g;
        memset(&g, 0, sizeof(g));
        g.batch = (int)batch; g.err = err;
        g.c = am; g.ldc = p.ldm; g.c_batch = p.m * p.ldm;
        g.M = (int)p.m; g.N = (int)p.m; g.K = (int)p.n; g.symmetric = 1;
        if ((rc = ns_product<128, false, kPlain>(xa[cur], xb[cur], g, sms, st))) return rc;
        g.c = mm; g.d = am; g.K = (int)p.m;
        g.ca = (float)a; g.cb = (float)b; g.cc = (float)c;
        if ((rc = ns_product<128, false, kCombine>(aa, ab, g, sms, st))) return rc;
        g.c = x[cur ^ 1]; g.d = nullptr; g.ldc = p.ldx; g.c_batch = p.m * p.ldx;
        g.N = (int)p.n; g.symmetric = 0;
        if ((rc = ns_product<256, true, kPlain>(ma, xb[cur], g, sms, st))) return rc;
    }
    e.src = x[steps & 1]; e.dst = out;
    e.s_i = tall ? 1 : cols; e.s_j = tall ? cols : 1; e.s_b = rows * cols;
    if (out_dtype == SRU_F16) ns_last_kernel<__half><<<tile_grid, 256, 0, st>>>(e);
    else ns_last_kernel<__nv_bfloat16><<<tile_grid, 256, 0, st>>>(e);
    SRUB_CUDA_CHECK(cudaGetLastError());
    return 0;
}

}  // extern "C"
