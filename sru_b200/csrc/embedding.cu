// Scaled lookup in a table of token vectors, and its gradient.
//
//   forward    y[n, :] = scale * W[token_n, :]
//   backward   dW[v, :] = scale * sum over {n : token_n = v} of dy[n, :],   0 for tokens that do not occur
//
// Both are bound by HBM: the rows read and written, and for the gradient the dense dW.
//
// The gradient is formed by sorted tokens, so that it needs no floating-point atomics and repeated calls give identical
// bits: a stable radix sort of (token, position) by one cluster of sixteen CTAs, then sums over tiles of kTile sorted
// positions.  Token frequencies are uneven (one word may be a twentieth of all positions), so the unit of work is a
// tile of positions, not a token: a run of equal tokens inside a tile goes straight to dW; a run that crosses tiles
// leaves one float32 partial row per tile, and a last kernel adds those up in order.
//
// A token outside the table reads nothing: its row of y is zero, it adds nothing to the gradient, and the device error
// flag is raised (sru_b200_check_device_error).
#include <algorithm>
#include <cstring>

#include "common.cuh"

namespace srub {

namespace {

constexpr int kSortCtas = 16, kSortWarps = 16, kBins = 256;
constexpr int kTile = 32;             // sorted positions per tile: one per lane of the warp that reads their keys

struct EmbArgs {
    const void *tokens, *src;         // src: table (forward) or dy (backward)
    void *dst;                        // y (forward) or dW (backward)
    float *part;                      // backward: (tiles, 2, d): sums of a tile's first and last run where they cross it
    uint2 *sorted, *spare;            // (token, position)
    int64_t n, v, ld;
    int64_t padding;
    int d;
    int passes;
    float scale;
    int dst_size;                     // bytes of an element of dW
    bool fill16;                      // rows of dW are 16-byte aligned
    int *err;
};

template <typename TK> __device__ __forceinline__ int64_t token_at(const void *tokens, int64_t i) {
    return static_cast<int64_t>(static_cast<const TK *>(tokens)[i]);
}

// ---- forward ----------------------------------------------------------------------------------------------------
// y taken as one line of groups of VEC elements, REP groups per thread, neighbouring threads on neighbouring groups: every
// store instruction fills whole lines whatever the row length (a warp per block of a row left most lanes idle in the last
// block of a row: 520 floats 18.5 us for 32768 rows, 68 MB).
template <typename TK, typename TI, typename TO, int VEC, int REP>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const EmbArgs a, uint32_t groups_per_row, uint32_t step_rows, uint32_t step_groups) {
    const int64_t total = a.n * groups_per_row;
    const int64_t g0 = (int64_t)blockIdx.x * (256 * REP) + threadIdx.x;
    // row and group within it, by one division; 256 groups on are step_rows rows and step_groups groups
    uint32_t row = total <= 0xffffffffll ? (uint32_t)g0 / groups_per_row : (uint32_t)(g0 / groups_per_row);
    uint32_t col = (uint32_t)(g0 - (int64_t)row * groups_per_row);
    const uint32_t n = (uint32_t)a.n, ld = (uint32_t)a.ld;      // all below 2^31
    const uint64_t v = (uint64_t)a.v;
    Pack<TI, VEC> in[REP];
    bool bad = false;
#pragma unroll
    for (int r = 0; r < REP; ++r) {
        memset(&in[r], 0, sizeof(in[r]));
        if (row < n) {
            const uint64_t t = (uint64_t)token_at<TK>(a.tokens, row);       // a negative one is a large one
            if (t < v) in[r] = *reinterpret_cast<const Pack<TI, VEC> *>(static_cast<const TI *>(a.src) + (uint64_t)(uint32_t)t * ld + col * VEC);
            else bad = true;
        }
        row += step_rows;
        col += step_groups;
        if (col >= groups_per_row) { col -= groups_per_row; ++row; }
    }
#pragma unroll
    for (int r = 0; r < REP; ++r) {
        const int64_t g = g0 + r * 256;
        Pack<TO, VEC> out;
#pragma unroll
        for (int k = 0; k < VEC; ++k) out.v[k] = Cvt<TO>::from_f(Cvt<TI>::to_f(in[r].v[k]) * a.scale);
        if (g < total) *reinterpret_cast<Pack<TO, VEC> *>(static_cast<TO *>(a.dst) + g * VEC) = out;
    }
    if (bad) atomicExch(a.err, kSiteToken);
}

// ---- sort -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t rank, uint32_t v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}

// Key of position i: the token, or v (behind all tokens) where the position adds nothing to the gradient.
template <typename TK> __device__ __forceinline__ uint32_t key_at(const EmbArgs &a, int64_t i) {
    const int64_t t = token_at<TK>(a.tokens, i);
    if (t < 0 || t >= a.v) { atomicExch(a.err, kSiteToken); return (uint32_t)a.v; }
    return (uint32_t)(t == a.padding ? a.v : t);
}

// Stable radix sort, 8 bits a pass, by ONE cluster: every warp owns a contiguous part of the positions and a histogram of
// its own; counts become starting offsets by a prefix over (digit, CTA, warp), the CTAs' totals travelling through
// distributed shared memory; then every warp writes its entries in order.  Counts are integers: no order matters.
// Bound by latency up to some 16000 positions (13 us in two passes), then by the scattered 8-byte writes of its SMs: sixteen
// CTAs of 16 warps instead of eight of 32 took the whole gradient of 65536 tokens from 78 to 70 us.
constexpr int kHeld = 8;              // entries per lane that stay in registers between counting and writing
struct SortShared {
    uint32_t hist[kSortWarps][kBins];
    uint32_t totals[kSortCtas][kBins];
    uint32_t offs[kBins];
    uint32_t warp_sum[8];
};

template <typename TK> __device__ __forceinline__ void sort_tokens(const EmbArgs &a, SortShared &sh) {
    auto &hist = sh.hist;
    auto &totals = sh.totals;
    auto &offs = sh.offs;
    auto &warp_sum = sh.warp_sum;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int64_t per = ((a.n + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps) + 31) / 32 * 32;
    const int64_t i0 = min(a.n, ((int64_t)rank * kSortWarps + warp) * per), i1 = min(a.n, i0 + per);

    cluster_barrier();       // every CTA has started before another writes to its shared memory
    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = 8 * pass;
        // the last pass ends in a.sorted
        uint2 *out = ((a.passes - pass) & 1) ? a.sorted : a.spare;
        const uint2 *in = ((a.passes - pass) & 1) ? a.spare : a.sorted;
        auto entry = [&](int64_t i) -> uint2 {
            if (pass == 0) return make_uint2(key_at<TK>(a, i), (uint32_t)i);
            return __ldcg(in + i);         // written by other SMs of the cluster: past L1
        };
        const bool held = per <= 32 * kHeld;        // the same for all warps
        uint2 mine[kHeld];
        if (held) {
#pragma unroll
            for (int h = 0; h < kHeld; ++h) {
                const int64_t i = i0 + h * 32 + lane;
                mine[h] = i < i1 ? entry(i) : make_uint2(0u, 0u);
            }
        }
        for (int k = lane; k < kBins; k += 32) hist[warp][k] = 0;
        __syncwarp();
        if (held) {
#pragma unroll
            for (int h = 0; h < kHeld; ++h)
                if (i0 + h * 32 + lane < i1) atomicAdd(&hist[warp][(mine[h].x >> shift) & 255u], 1u);
        } else {
            for (int64_t i = i0 + lane; i < i1; i += 32) atomicAdd(&hist[warp][(entry(i).x >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (threadIdx.x < kBins) {
            uint32_t s = 0;
#pragma unroll 8
            for (int w = 0; w < kSortWarps; ++w) {
                const uint32_t c = hist[w][threadIdx.x];
                hist[w][threadIdx.x] = s;
                s += c;
            }
            for (uint32_t r = 0; r < kSortCtas; ++r) store_cluster(smem_u32(&totals[rank][threadIdx.x]), r, s);
        }
        cluster_barrier();
        uint32_t all = 0, below = 0, incl = 0;
        if (threadIdx.x < kBins) {
#pragma unroll
            for (uint32_t r = 0; r < kSortCtas; ++r) {
                const uint32_t c = totals[r][threadIdx.x];
                below += r < rank ? c : 0u;
                all += c;
            }
            incl = all;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            if (lane == 31) warp_sum[warp] = incl;
        }
        __syncthreads();
        if (threadIdx.x < kBins) {
            uint32_t base = incl - all;
            for (int w = 0; w < warp; ++w) base += warp_sum[w];
            offs[threadIdx.x] = base + below;
        }
        __syncthreads();
        auto write = [&](bool on, uint2 e) {
            const uint32_t digit = (e.x >> shift) & 255u;
            const unsigned same = __match_any_sync(0xffffffffu, on ? digit : 256u + lane);
            const uint32_t at = on ? hist[warp][digit] : 0u;
            __syncwarp();
            if (on) {
                if ((same >> lane) == 1u) hist[warp][digit] = at + __popc(same);     // the last lane with this digit
                out[offs[digit] + at + __popc(same & ((1u << lane) - 1u))] = e;
            }
            __syncwarp();
        };
        if (held) {
#pragma unroll
            for (int h = 0; h < kHeld; ++h)
                if (i0 + h * 32 < i1) write(i0 + h * 32 + lane < i1, mine[h]);
        } else {
            for (int64_t i = i0; i < i1; i += 32) {
                const bool on = i + lane < i1;
                write(on, on ? entry(i + lane) : make_uint2(0u, 0u));
            }
        }
        __threadfence();
        cluster_barrier();
    }
}

template <typename TK>
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortWarps * 32)
embedding_sort_kernel(const EmbArgs a) {
    __shared__ SortShared sh;
    early_next_kernel();
    sort_tokens<TK>(a, sh);
}

// Zeros in those of the rows [block * kFillRows, ...) of dW whose token does not occur, which a bisection of the sorted
// positions tells for every row.  (Zeros everywhere before the sums, in the sort's launch or as a memory set, write the rows
// that occur twice and leave L2 full of lines that the sums then have to push out: 133 and 121 us for 16384 tokens over
// 50000 x 2048 floats.)
constexpr int kFillRows = 64;
__device__ __forceinline__ void fill_row(const EmbArgs &a, int64_t row, int64_t row_bytes, int lane) {
    char *p = static_cast<char *>(a.dst) + row * row_bytes;
    if (a.fill16) {
        for (int64_t c = lane * 16; c < row_bytes; c += 512) __stcs(reinterpret_cast<uint4 *>(p + c), make_uint4(0, 0, 0, 0));
    } else {
        for (int64_t c = lane * 2; c < row_bytes; c += 64) *reinterpret_cast<uint16_t *>(p + c) = 0;
    }
}
__device__ __forceinline__ void fill_absent(const EmbArgs &a, int64_t block) {
    __shared__ bool present[kFillRows];
    const int64_t r0 = block * kFillRows;
    const int rows = (int)min((int64_t)kFillRows, a.v - r0);
    if (threadIdx.x < rows) {
        const uint32_t row = (uint32_t)(r0 + threadIdx.x);
        int64_t lo = 0, hi = a.n;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (a.sorted[mid].x < row) lo = mid + 1;
            else hi = mid;
        }
        present[threadIdx.x] = lo < a.n && a.sorted[lo].x == row;
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row_bytes = (int64_t)a.d * a.dst_size;
    for (int k = warp; k < rows; k += blockDim.x >> 5) {
        if (!present[k]) fill_row(a, r0 + k, row_bytes, lane);
    }
}

// ---- sums over sorted positions ---------------------------------------------------------------------------------
// Columns of this lane: c0 + r * 32 * VEC + k, r < REP, k < VEC.
template <typename TO, int VEC, int REP>
__device__ __forceinline__ void store_sum(TO *row, int c0, int d, const float (&acc)[REP][VEC], float scale) {
#pragma unroll
    for (int r = 0; r < REP; ++r) {
        const int c = c0 + r * 32 * VEC;
        if (c >= d) continue;
        Pack<TO, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = Cvt<TO>::from_f(acc[r][k] * scale);
        *reinterpret_cast<Pack<TO, VEC> *>(row + c) = o;
    }
}

// Unit w: a tile of positions, a block of columns.  (Sorted positions past L1: the kernel that sorted them may be this one.)
template <typename TI, typename TO, int VEC, int REP>
__device__ __forceinline__ void sum_unit(const EmbArgs &a, int64_t w, int blocks_per_row) {
    const int lane = threadIdx.x & 31;
    const int64_t tile = w / blocks_per_row, i0 = tile * kTile;
    const int c0 = (int)(w - tile * blocks_per_row) * (32 * VEC * REP) + lane * VEC;
    const uint32_t none = (uint32_t)a.v;                // key of positions that add nothing
    const uint2 mine = (i0 + lane < a.n) ? __ldcg(a.sorted + i0 + lane) : make_uint2(none, 0u);
    const uint32_t before = i0 > 0 ? __ldcg(&a.sorted[i0 - 1].x) : none;
    const uint32_t after = i0 + kTile < a.n ? __ldcg(&a.sorted[i0 + kTile].x) : none;
    // sorted: the positions that count come first, and a bit says where a run ends (the tile's end ends them all)
    const int count = __popc(__ballot_sync(0xffffffffu, mine.x != none));
    const uint32_t next_key = __shfl_down_sync(0xffffffffu, mine.x, 1);
    const unsigned ends = __ballot_sync(0xffffffffu, lane == kTile - 1 || next_key != mine.x);
    const TI *src = static_cast<const TI *>(a.src) + c0;
    float acc[REP][VEC];
#pragma unroll
    for (int r = 0; r < REP; ++r)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[r][k] = 0.0f;
    bool whole_head = true;                             // the current run reaches back to the tile's first entry
    constexpr int G = 8;                                // rows requested together
    for (int e0 = 0; e0 < count; e0 += G) {
        Pack<TI, VEC> in[G][REP];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const TI *row = src + (int64_t)__shfl_sync(0xffffffffu, mine.y, e0 + g) * a.d;
#pragma unroll
            for (int r = 0; r < REP; ++r) {
                if (e0 + g < count && c0 + r * 32 * VEC < a.d) in[g][r] = *reinterpret_cast<const Pack<TI, VEC> *>(row + r * 32 * VEC);
                else memset(&in[g][r], 0, sizeof(in[g][r]));
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int e = e0 + g;
#pragma unroll
            for (int r = 0; r < REP; ++r)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[r][k] += Cvt<TI>::to_f(in[g][r].v[k]);
            if (!((ends >> e) & 1u) || e >= count) continue;
            const uint32_t key = __shfl_sync(0xffffffffu, mine.x, e);
            if (whole_head && key == before)
                store_sum<float, VEC, REP>(a.part + (tile * 2) * a.d, c0, a.d, acc, 1.0f);
            else if (e == kTile - 1 && after == key)
                store_sum<float, VEC, REP>(a.part + (tile * 2 + 1) * a.d, c0, a.d, acc, 1.0f);
            else
                store_sum<TO, VEC, REP>(static_cast<TO *>(a.dst) + (int64_t)key * a.d, c0, a.d, acc, a.scale);
#pragma unroll
            for (int r = 0; r < REP; ++r)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[r][k] = 0.0f;
            whole_head = false;
        }
    }
}

// The grid's first CTAs fill the rows of absent tokens: they search, then write, while the others wait for their rows.
template <typename TI, typename TO, int VEC, int REP>
__global__ void __launch_bounds__(128) embedding_sum_kernel(const EmbArgs a, int blocks_per_row, unsigned fill_ctas) {
    early_next_kernel();
    previous_kernel_done();
    if (blockIdx.x < fill_ctas) {
        fill_absent(a, blockIdx.x);
        return;
    }
    const int64_t tiles = (a.n + kTile - 1) / kTile, units = tiles * blocks_per_row, step = (int64_t)(gridDim.x - fill_ctas) * 4;
    for (int64_t w = (int64_t)(blockIdx.x - fill_ctas) * 4 + (threadIdx.x >> 5); w < units; w += step) sum_unit<TI, TO, VEC, REP>(a, w, blocks_per_row);
}

// Key of the run that starts in this tile and goes on behind it; v: there is none.
__device__ __forceinline__ uint32_t run_from(const EmbArgs &a, int64_t tile) {
    const int64_t i0 = tile * kTile, i1 = i0 + kTile;
    const uint32_t none = (uint32_t)a.v;
    if (i1 >= a.n) return none;
    const uint32_t key = __ldcg(&a.sorted[i1 - 1].x), next = __ldcg(&a.sorted[i1].x), first = __ldcg(&a.sorted[i0].x);
    const uint32_t before = i0 > 0 ? __ldcg(&a.sorted[i0 - 1].x) : none;
    return next != key || (first == key && before == key) ? none : key;
}
// The first tile behind `tile` that its last run does not reach; by a whole warp.
__device__ __forceinline__ int64_t run_end(const EmbArgs &a, int64_t tile, uint32_t key) {
    const int lane = threadIdx.x & 31;
    const int64_t tiles = (a.n + kTile - 1) / kTile;
    // tiles that the run reaches behind this one: the first 32, then by bisection in 32 parts
    int64_t lo = tile + 1, hi = tiles;          // the run covers the start of every tile below lo, of none from hi on
    const unsigned m = __ballot_sync(0xffffffffu, lo + lane < hi && __ldcg(&a.sorted[(lo + lane) * kTile].x) == key);
    if (m != 0xffffffffu) {
        lo += __ffs(~m) - 1;
    } else {
        for (lo += 32; lo < hi;) {
            const int64_t step = (hi - lo + 31) / 32, u = lo + lane * step;
            const unsigned c = __ballot_sync(0xffffffffu, u < hi && __ldcg(&a.sorted[u * kTile].x) == key);
            const int covered = c == 0xffffffffu ? 32 : __ffs(~c) - 1;
            if (covered == 0) break;
            const int64_t last = lo + (covered - 1) * step;     // the last probed tile inside the run
            hi = min(hi, last + step);
            lo = last + 1;
        }
    }
    return lo;
}

// Runs that cross tiles: of the tile in which the run starts, a CTA per block of columns adds the tiles' partial rows, the
// tiles in four contiguous parts, one warp each, then the parts in order: the order is fixed by the tokens alone.
template <typename TO, int VEC, int REP>
__global__ void __launch_bounds__(128) embedding_join_kernel(const EmbArgs a) {
    __shared__ float parts[3][32 * VEC * REP];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t tile = blockIdx.x;
    previous_kernel_done();
    const uint32_t key = run_from(a, tile);
    if (key == (uint32_t)a.v) return;
    const int64_t lo = run_end(a, tile, key);
    const int64_t count = lo - (tile + 1), per = (count + 3) / 4, q0 = min(count, warp * per), q1 = min(count, q0 + per);
    const int c0 = blockIdx.y * (32 * VEC * REP) + lane * VEC;
    float acc[REP][VEC];
#pragma unroll
    for (int r = 0; r < REP; ++r)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[r][k] = 0.0f;
    constexpr int G = 8;                        // rows requested together
    auto add_rows = [&](int64_t row, int64_t step, int n) {
        Pack<float, VEC> in[G][REP];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int r = 0; r < REP; ++r) {
                const int c = c0 + r * 32 * VEC;
                if (g < n && c < a.d) in[g][r] = *reinterpret_cast<const Pack<float, VEC> *>(a.part + (row + g * step) * a.d + c);
                else memset(&in[g][r], 0, sizeof(in[g][r]));
            }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int r = 0; r < REP; ++r)
#pragma unroll
                for (int k = 0; k < VEC; ++k) acc[r][k] += in[g][r].v[k];
    };
    if (warp == 0) add_rows(tile * 2 + 1, 0, 1);
    for (int64_t q = q0; q < q1; q += G) add_rows((tile + 1 + q) * 2, 2, (int)min((int64_t)G, q1 - q));
    if (warp > 0)
#pragma unroll
        for (int r = 0; r < REP; ++r)
#pragma unroll
            for (int k = 0; k < VEC; ++k) parts[warp - 1][(r * 32 + lane) * VEC + k] = acc[r][k];
    __syncthreads();
    if (warp > 0) return;
    for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int r = 0; r < REP; ++r)
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[r][k] += parts[w][(r * 32 + lane) * VEC + k];
    store_sum<TO, VEC, REP>(static_cast<TO *>(a.dst) + (int64_t)key * a.d, c0, a.d, acc, a.scale);
}

// A small gradient in one launch: the cluster that sorts also sums, fills the absent rows and joins the runs, a warp for each of
// their units.
template <typename TK, typename TI, typename TO, int VEC, int REP>
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortWarps * 32)
embedding_small_kernel(const EmbArgs a, int blocks_per_row) {
    __shared__ SortShared sh;
    sort_tokens<TK>(a, sh);
    const int lane = threadIdx.x & 31;
    const int64_t me = (int64_t)cluster_rank() * kSortWarps + (threadIdx.x >> 5), warps = kSortCtas * kSortWarps;
    const int64_t tiles = (a.n + kTile - 1) / kTile, units = tiles * blocks_per_row, row_bytes = (int64_t)a.d * a.dst_size;
    for (int64_t w = me; w < units; w += warps) sum_unit<TI, TO, VEC, REP>(a, w, blocks_per_row);
    for (int64_t r0 = (warps - 1 - me) * 32; r0 < a.v; r0 += warps * 32) {     // from the other end: the last warps have fewer units
        const int64_t row = r0 + lane;
        int64_t lo = 0, hi = a.n;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (__ldcg(&a.sorted[mid].x) < (uint32_t)row) lo = mid + 1;
            else hi = mid;
        }
        const bool here = lo < a.n && __ldcg(&a.sorted[lo].x) == (uint32_t)row;
        for (unsigned absent = __ballot_sync(0xffffffffu, row < a.v && !here); absent; absent &= absent - 1)
            fill_row(a, r0 + __ffs(absent) - 1, row_bytes, lane);
    }
    __threadfence();
    cluster_barrier();
    for (int64_t w = me; w < units; w += warps) {
        const int64_t tile = w / blocks_per_row;
        const uint32_t key = run_from(a, tile);
        if (key == (uint32_t)a.v) continue;
        const int c0 = (int)(w - tile * blocks_per_row) * (32 * VEC * REP) + lane * VEC;
        const int64_t end = run_end(a, tile, key);
        float acc[REP][VEC];
#pragma unroll
        for (int r = 0; r < REP; ++r)
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[r][k] = 0.0f;
        constexpr int G = 8;                    // rows requested together
        for (int64_t q0 = tile; q0 < end; q0 += G) {
            float in[G][REP][VEC];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int r = 0; r < REP; ++r) {
                    const int64_t q = q0 + g;
                    const int c = c0 + r * 32 * VEC;
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        in[g][r][k] = q < end && c < a.d ? __ldcg(a.part + (q == tile ? q * 2 + 1 : q * 2) * a.d + c + k) : 0.0f;
                }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int r = 0; r < REP; ++r)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) acc[r][k] += in[g][r][k];
        }
        store_sum<TO, VEC, REP>(static_cast<TO *>(a.dst) + (int64_t)key * a.d, c0, a.d, acc, a.scale);
    }
}

int check_embedding(int64_t n, int64_t v, int64_t d, int64_t ld, int token_bytes, int table_dtype, int y_dtype) {
    if (n < 0 || v < 1 || d < 1 || ld < d || ld > 0x7fffffff || n > 0x7fffffff || v > 0x7fffffff || d > (1 << 24))
        return set_error(SRU_ERR_BAD_ARG, "bad sizes: %lld tokens, table (%lld, %lld) with row stride %lld", (long long)n,
                         (long long)v, (long long)d, (long long)ld);
    if (token_bytes != 4 && token_bytes != 8) return set_error(SRU_ERR_BAD_ARG, "tokens must be 4 or 8 bytes wide");
    const bool t16 = table_dtype == SRU_F16 || table_dtype == SRU_BF16, y16 = y_dtype == SRU_F16 || y_dtype == SRU_BF16;
    if (!(table_dtype == y_dtype && (t16 || table_dtype == SRU_F32)) && !(table_dtype == SRU_F32 && y16))
        return set_error(SRU_ERR_UNSUPPORTED, "embedding: y must have the table's type (float32, float16, bfloat16) or be "
                         "16-bit over a float32 table, got %d over %d", y_dtype, table_dtype);
    return 0;
}

bool aligned16(const void *p, int64_t row_bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row_bytes % 16 == 0; }

template <typename TK, typename TI, typename TO> int launch_forward(const EmbArgs &a, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(TO);
    const bool wide = aligned16(a.src, a.ld * sizeof(TI)) && aligned16(a.dst, a.d * sizeof(TO));
    auto go = [&](auto vec, auto rep) -> int {
        constexpr int V = decltype(vec)::value, R = decltype(rep)::value;
        const int64_t blocks = (a.n * (a.d / V) + 256 * R - 1) / (256 * R);
        if (blocks > 0x7fffffff) return set_error(SRU_ERR_UNSUPPORTED, "embedding: n * hidden too large");
        const uint32_t groups = a.d / V;
        embedding_fwd_kernel<TK, TI, TO, V, R><<<(unsigned)blocks, 256, 0, st>>>(a, groups, 256 / groups, 256 % groups);
        SRUB_LAUNCHED();
        return 0;
    };
    if (!wide) return go(std::integral_constant<int, 1>(), std::integral_constant<int, 8>());
    // a few rows: one group per thread, so that they reach all SMs
    if (a.n * (a.d / VEC) < kSms * 2048) return go(std::integral_constant<int, VEC>(), std::integral_constant<int, 1>());
    return go(std::integral_constant<int, VEC>(), std::integral_constant<int, 2>());
}

template <typename TK> int launch_sort(const EmbArgs &a, cudaStream_t st) {
    static bool attr_set[64] = {false};
    int dev = 0;
    SRUB_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        SRUB_CUDA_CHECK(cudaFuncSetAttribute(embedding_sort_kernel<TK>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        attr_set[dev] = true;
    }
    embedding_sort_kernel<TK><<<kSortCtas, kSortWarps * 32, 0, st>>>(a);
    SRUB_LAUNCHED();
    return 0;
}

// One launch for a gradient of at most 1 MB and 2048 tokens, which sixteen SMs move about as fast as all: three launches / one, us with the host's
// share and of the GPU alone: 64 tokens over 100 x 64 20 / 12 and 8.8 / 9.3, 500 over 200 x 64 (0.2 MB) 20 / 12 and 11.0 / 11.3, 500
// over 1000 x 256 (1.5 MB) 19 / 19 and 14.6 / 17.7, 4000 over 4000 x 256 (8 MB) 19 / 25 and 16.5 / 22.2.
// A run is joined by one warp there, so that few tiles are wanted.
bool is_small(const EmbArgs &a, int64_t src_size) { return a.n <= 64 * kTile && (a.n * src_size + a.v * a.dst_size) * a.d <= (1 << 20); }

template <typename TK, typename TI, typename TO> int launch_backward(const EmbArgs &a, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(TI);
    const bool wide = aligned16(a.src, a.d * sizeof(TI)) && aligned16(a.dst, a.d * sizeof(TO));
    auto go = [&](auto vec, auto rep) -> int {
        constexpr int V = decltype(vec)::value, R = decltype(rep)::value;
        const int per_row = (a.d + 32 * V * R - 1) / (32 * V * R);
        if (per_row > 65535) return set_error(SRU_ERR_UNSUPPORTED, "embedding: hidden too large");
        if (is_small(a, sizeof(TI))) {
            auto kernel = embedding_small_kernel<TK, TI, TO, V, R>;
            static bool attr_set[64] = {false};
            int dev = 0;
            SRUB_CUDA_CHECK(cudaGetDevice(&dev));
            if (dev >= 0 && dev < 64 && !attr_set[dev]) {
                SRUB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
                attr_set[dev] = true;
            }
            kernel<<<kSortCtas, kSortWarps * 32, 0, st>>>(a, per_row);
            SRUB_LAUNCHED();
            return 0;
        }
        if (int rc = launch_sort<TK>(a, st)) return rc;
        const int64_t units = (a.n + kTile - 1) / kTile * per_row;
        const int64_t sums = std::min<int64_t>((units + 3) / 4, kSms * 64), fill = (a.v + kFillRows - 1) / kFillRows;
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        cudaLaunchAttribute early = early_launch();
        cfg.attrs = &early; cfg.numAttrs = 1; cfg.stream = st;
        cfg.blockDim = dim3(128);
        cfg.gridDim = dim3((unsigned)(sums + fill));
        SRUB_LAUNCH(&cfg, embedding_sum_kernel<TI, TO, V, R>, a, per_row, (unsigned)fill);
        cfg.gridDim = dim3((unsigned)((a.n + kTile - 1) / kTile), per_row);
        SRUB_LAUNCH(&cfg, embedding_join_kernel<TO, V, R>, a);
        return 0;
    };
    if (wide) return go(std::integral_constant<int, VEC>(), std::integral_constant<int, 1>());
    return go(std::integral_constant<int, 1>(), std::integral_constant<int, 4>());
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t sort_bytes(int64_t n) { return round256((size_t)n * sizeof(uint2)); }

}  // namespace

}  // namespace srub

using namespace srub;

extern "C" {

int sru_b200_embedding_forward(void *y, const void *tokens, const void *table, int64_t n, int64_t vocabulary,
                               int64_t hidden, int64_t table_stride, double scale, int token_bytes, int table_dtype,
                               int y_dtype, void *stream) {
    int rc = check_embedding(n, vocabulary, hidden, table_stride, token_bytes, table_dtype, y_dtype);
    if (rc) return rc;
    if (n == 0) return 0;
    if (!y || !tokens || !table) return set_error(SRU_ERR_BAD_ARG, "embedding: a required pointer is null");
    EmbArgs a;
    memset(&a, 0, sizeof(a));
    a.tokens = tokens; a.src = table; a.dst = y;
    a.n = n; a.v = vocabulary; a.d = (int)hidden; a.ld = table_stride; a.scale = (float)scale;
    a.err = device_error_flag();
    if (!a.err) return set_error(SRU_ERR_CUDA, "device error flag unavailable");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto tk) -> int {
        using TK = decltype(tk);
        if (table_dtype == SRU_F32 && y_dtype == SRU_F32) return launch_forward<TK, float, float>(a, st);
        if (table_dtype == SRU_F32 && y_dtype == SRU_F16) return launch_forward<TK, float, __half>(a, st);
        if (table_dtype == SRU_F32) return launch_forward<TK, float, __nv_bfloat16>(a, st);
        if (table_dtype == SRU_F16) return launch_forward<TK, __half, __half>(a, st);
        return launch_forward<TK, __nv_bfloat16, __nv_bfloat16>(a, st);
    };
    return token_bytes == 4 ? go(int32_t()) : go(int64_t());
}

size_t sru_b200_embedding_backward_workspace_bytes(int64_t n, int64_t vocabulary, int64_t hidden) {
    (void)vocabulary;
    if (n < 1 || hidden < 1) return 0;
    return 2 * sort_bytes(n) + (size_t)((n + kTile - 1) / kTile) * 2 * (size_t)hidden * sizeof(float);
}

int sru_b200_embedding_backward(void *grad_table, const void *tokens, const void *grad_y, int64_t n, int64_t vocabulary,
                                int64_t hidden, int64_t padding_idx, double scale, int token_bytes, int table_dtype,
                                int y_dtype, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = check_embedding(n, vocabulary, hidden, hidden, token_bytes, table_dtype, y_dtype);
    if (rc) return rc;
    if (!grad_table || (n > 0 && (!tokens || !grad_y))) return set_error(SRU_ERR_BAD_ARG, "embedding: a required pointer is null");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t need = sru_b200_embedding_backward_workspace_bytes(n, vocabulary, hidden);
    if (n > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
        return set_error(SRU_ERR_WORKSPACE, "16-byte aligned workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    if (n == 0) {
        SRUB_CUDA_CHECK(cudaMemsetAsync(grad_table, 0, (size_t)vocabulary * hidden * dtype_size(table_dtype), st));
        return 0;
    }
    EmbArgs a;
    memset(&a, 0, sizeof(a));
    char *ws = static_cast<char *>(workspace);
    a.tokens = tokens; a.src = grad_y; a.dst = grad_table;
    a.sorted = reinterpret_cast<uint2 *>(ws);
    a.spare = reinterpret_cast<uint2 *>(ws + sort_bytes(n));
    a.part = reinterpret_cast<float *>(ws + 2 * sort_bytes(n));
    a.n = n; a.v = vocabulary; a.d = (int)hidden; a.padding = padding_idx < 0 ? -1 : padding_idx; a.scale = (float)scale;
    a.passes = 1;
    while (a.passes < 4 && (vocabulary >> (8 * a.passes)) != 0) ++a.passes;     // the largest key is `vocabulary`
    a.err = device_error_flag();
    if (!a.err) return set_error(SRU_ERR_CUDA, "device error flag unavailable");
    a.dst_size = (int)dtype_size(table_dtype);
    a.fill16 = aligned16(grad_table, hidden * a.dst_size);
    auto go = [&](auto tk) -> int {
        using TK = decltype(tk);
        if (table_dtype == SRU_F32 && y_dtype == SRU_F32) return launch_backward<TK, float, float>(a, st);
        if (table_dtype == SRU_F32 && y_dtype == SRU_F16) return launch_backward<TK, __half, float>(a, st);
        if (table_dtype == SRU_F32) return launch_backward<TK, __nv_bfloat16, float>(a, st);
        if (table_dtype == SRU_F16) return launch_backward<TK, __half, __half>(a, st);
        return launch_backward<TK, __nv_bfloat16, __nv_bfloat16>(a, st);
    };
    return token_bytes == 4 ? go(int32_t()) : go(int64_t());
}

}  // extern "C"
