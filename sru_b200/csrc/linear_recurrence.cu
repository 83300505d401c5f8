// The gated linear recurrence: SRU's state update with a gate that does not look at the state,
//
//   f_t = sigmoid(g_t + bias),   c_t = f_t c_{t-1} + (1 - f_t) x_t,   h_t = c_t      (0 at padded positions, c carried)
//
// over u (L, B, d, 2) holding the pairs (x, g), gate index innermost as in the SRU's U.  Backward, with dc_t the whole
// gradient of c_t:
//
//   dc_t = grad_h_t + f_{t+1} dc_{t+1},   dx_t = (1 - f_t) dc_t,   dg_t = dc_t (c_{t-1} - x_t) f_t (1 - f_t),
//   dbias = sum over t, b of dg,          dc_0 = f_first dc_first.
//
// HBM-bound: 3 elements per column-step forward, 5 backward.  A lane owns V = 2 adjacent columns of one sequence (1 where
// sizes or alignment forbid pairs) and walks time in chunks of kT steps; the next chunk's loads are issued before the current chunk is worked on.  The forward
// pass leaves the float32 state in front of every chunk (kT = 8: half a byte per column-step); the backward
// pass recomputes the states of a chunk from it, which is cheaper than reading a saved history (2 or 4 bytes) and
// exact in the 16-bit types, whose rounded h would enter c_{t-1} - x_t.
//
// Arithmetic is float32 throughout.  With e = 2^(-(g + bias) log2 e), f = 1 / (1 + e) and 1 - f = e f: both keep their
// relative accuracy however close to 0 or 1 the gate is.
#include <algorithm>
#include <cstring>

#include "f32x2.cuh"
#include "tcgen05.cuh"

namespace srub {

namespace {

constexpr int kT = 8;           // steps per chunk, and between two saved states

// Slices of time per column: warps of a CTA, times CTAs of a cluster.
struct Slices {
    int warps, ranks;
    int count() const { return warps * ranks; }
};

struct LinRecArgs {
    void *h;                    // forward: (L, B, d); backward: grad_u (L, B, d, 2)
    float *last;                // forward: c_last (B, d); backward: grad of c0 (B, d); may be NULL
    float *states;              // (chunks, B, d): state in front of each chunk; forward may have NULL
    float *bias_part;           // backward: (parts, d) partial sums of grad_bias, or NULL
    const void *u;
    const float *bias, *first;  // first: c0 (forward), grad of c_last (backward); may be NULL
    const void *grad_h;         // backward; may be NULL
    const uint8_t *mask;        // (L, B) bytes or NULL
    int64_t L, B;
    int64_t u_t, u_b, gh_t, gh_b;   // strides in elements (time strides signed: a reversed scan starts at the end)
    int64_t h_t, m_t;               // signed time strides of h / grad_u's column unit and of the mask
    int d, groups;                  // groups: warps' worth of columns per sequence
    int *err;
};

// ---- V float32 values, one per column of a lane; pairs go through the two-lane instructions -------------------------
template <int V> struct Num;
template <> struct Num<1> {
    float a;
    __device__ __forceinline__ float get(int) const { return a; }
};
template <> struct Num<2> {
    F2 a;
    __device__ __forceinline__ float get(int v) const {
        float lo, hi;
        f2_split(a, lo, hi);
        return v ? hi : lo;
    }
};
__device__ __forceinline__ Num<1> num(const float (&v)[1]) { return Num<1>{v[0]}; }
__device__ __forceinline__ Num<2> num(const float (&v)[2]) { return Num<2>{f2_make(v[0], v[1])}; }
template <int V> __device__ __forceinline__ Num<V> all(float x) {
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = x;
    return num(v);
}
__device__ __forceinline__ Num<1> fma(Num<1> a, Num<1> b, Num<1> c) { return {fmaf(a.a, b.a, c.a)}; }
__device__ __forceinline__ Num<1> mul(Num<1> a, Num<1> b) { return {a.a * b.a}; }
__device__ __forceinline__ Num<1> add(Num<1> a, Num<1> b) { return {a.a + b.a}; }
__device__ __forceinline__ Num<1> sub(Num<1> a, Num<1> b) { return {a.a - b.a}; }
__device__ __forceinline__ Num<2> fma(Num<2> a, Num<2> b, Num<2> c) { return {f2_fma(a.a, b.a, c.a)}; }
__device__ __forceinline__ Num<2> mul(Num<2> a, Num<2> b) { return {f2_mul(a.a, b.a)}; }
__device__ __forceinline__ Num<2> add(Num<2> a, Num<2> b) { return {f2_add(a.a, b.a)}; }
__device__ __forceinline__ Num<2> sub(Num<2> a, Num<2> b) { return {f2_sub(a.a, b.a)}; }
__device__ __forceinline__ Num<1> pick(bool first, Num<1> a, Num<1> b) { return first ? a : b; }
__device__ __forceinline__ Num<2> pick(bool first, Num<2> a, Num<2> b) { return {f2_select(first, a.a, b.a)}; }

template <typename TT> __device__ __forceinline__ Pack<TT, 2> pack2(float a, float b) {
    Pack<TT, 2> r;
    r.v[0] = Cvt<TT>::from_f(a);
    r.v[1] = Cvt<TT>::from_f(b);
    return r;
}
template <> __device__ __forceinline__ Pack<__half, 2> pack2<__half>(float a, float b) {
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const Pack<__half, 2> *>(&t);
}
template <> __device__ __forceinline__ Pack<__nv_bfloat16, 2> pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const Pack<__nv_bfloat16, 2> *>(&t);
}
template <typename TT> __device__ __forceinline__ Pack<TT, 1> rounded(Num<1> a) {
    Pack<TT, 1> r;
    r.v[0] = Cvt<TT>::from_f(a.a);
    return r;
}
template <typename TT> __device__ __forceinline__ Pack<TT, 2> rounded(Num<2> a) { return pack2<TT>(a.get(0), a.get(1)); }
template <typename TT> __device__ __forceinline__ Num<1> widened(const Pack<TT, 1> &p) { return {Cvt<TT>::to_f(p.v[0])}; }
template <typename TT> __device__ __forceinline__ Num<2> widened(const Pack<TT, 2> &p) {
    return {f2_make(Cvt<TT>::to_f(p.v[0]), Cvt<TT>::to_f(p.v[1]))};
}
// the pairs (x, g) of V columns
template <typename TT, int V> __device__ __forceinline__ void unpair(const Pack<TT, 2 * V> &p, Num<V> *x, Num<V> *g) {
    float a[V], b[V];
#pragma unroll
    for (int v = 0; v < V; ++v) { a[v] = Cvt<TT>::to_f(p.v[2 * v]); b[v] = Cvt<TT>::to_f(p.v[2 * v + 1]); }
    *x = num(a);
    *g = num(b);
}

__device__ __forceinline__ float min_nan(float a, float b) {     // NaN if either is
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// f and 1 - f from the gate's logit; nb = -bias * log2(e).  The exponential stays at most 2^126, so that e f is finite.
template <int V> __device__ __forceinline__ void gate(Num<V> g, Num<V> nb, Num<V> *f, Num<V> *keep) {
    const Num<V> z = fma(g, all<V>(kNegLog2e), nb);
    float e[V], r[V];
#pragma unroll
    for (int v = 0; v < V; ++v) e[v] = ex2_approx(min_nan(z.get(v), 126.0f));
    const Num<V> en = num(e), den = add(en, all<V>(1.0f));
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = rcp_approx(den.get(v));
    *f = num(r);
    *keep = mul(en, *f);
}

// T steps of a strided stream of N elements per lane and step; of a chunk that sticks out, steps from `n` on are zero and
// not read.
template <typename TT, int N, int T>
__device__ __forceinline__ void load_steps(Pack<TT, N> (&r)[T], const TT *p, int64_t stride, int64_t n) {
    if (n >= T) {
#pragma unroll
        for (int i = 0; i < T; ++i, p += stride) r[i] = *reinterpret_cast<const Pack<TT, N> *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < T; ++i, p += stride) {
            if (i < n) r[i] = *reinterpret_cast<const Pack<TT, N> *>(p);
            else memset(&r[i], 0, sizeof(r[i]));
        }
    }
}

// Padding of a chunk.  The whole warp works on one sequence, so the flags are uniform; lane i fetches step i's byte one
// round ahead, and the flags are formed when the round begins (formed at once, they would wait for the bytes: 34 -> 43 us for
// 1000 x 24 x 1024).  Bit i: step i is padded or lies behind the end.  0 is the common case, and takes the paths without
// selects.
template <int T> __device__ __forceinline__ uint8_t load_pad(const uint8_t *mask, int64_t stride, int64_t n, int lane, const uint8_t *any) {
    // an address for every lane, so that nothing but pad_flags depends on the byte
    return mask ? *(lane < T && lane < n ? mask + lane * stride : any) : (uint8_t)0;
}
template <int T> __device__ __forceinline__ unsigned pad_flags(const uint8_t *mask, uint8_t pad, int64_t n, int lane) {
    if (!mask) return n >= T ? 0u : (n <= 0 ? 0xffffffffu : 0xffffffffu << n) & (uint32_t)((1ull << T) - 1);
    return __ballot_sync(0xffffffffu, lane < T && (lane >= n || pad != 0));
}

// Where a warp stands: its sequence and columns, and which of the interleaved slices of time it works on.  Slices are the
// warps of a CTA and the CTAs of a cluster; chunk k of a column belongs to slice k mod slices.  Lanes behind the last
// column repeat it (they load and store the same values), so that no access needs a predicate.
struct Place {
    int lane, warp, warps;          // of the CTA
    uint32_t rank, ranks;           // of the cluster
    int64_t b, col;
    int j, shift;                   // first column; its place behind the first column of lane 0
};

// With a ring and without slices the CTA's warps stand side by side on 64-column groups of one sequence, and its last warp
// is not one of `warps`: it asks for the copies.
constexpr int kSide = 2;
template <int V, bool SPLIT, bool RING> __device__ __forceinline__ bool find_place(const LinRecArgs &a, Place *p) {
    p->lane = threadIdx.x & 31;
    p->warp = threadIdx.x >> 5;
    p->warps = (blockDim.x >> 5) - (RING && !SPLIT ? 1 : 0);
    p->rank = 0; p->ranks = 1;
    int j0;
    if (SPLIT || RING) {
        if (SPLIT) {
            asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(p->rank));
            asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(p->ranks));
        }
        const int64_t unit = blockIdx.x / p->ranks;
        const int units = SPLIT ? a.groups : (a.groups + kSide - 1) / kSide;        // of a sequence
        p->b = unit / units;
        j0 = (int)(unit - p->b * units) * (SPLIT ? 1 : kSide) * 32 * V;
        if (!SPLIT) p->warps = min(p->warps, (a.d - j0 + 32 * V - 1) / (32 * V));
        if (!SPLIT && p->warp < p->warps) j0 += p->warp * 32 * V;
    } else {
        const int64_t wid = (int64_t)blockIdx.x * p->warps + p->warp;
        p->b = wid / a.groups;
        j0 = (int)(wid - p->b * a.groups) * 32 * V;
    }
    p->j = min(j0 + p->lane * V, a.d - V);
    p->shift = p->j - j0;
    p->col = p->b * a.d + p->j;
    return p->b < a.B;
}

template <int V> __device__ __forceinline__ Num<V> load_small(const float *p, int64_t at) {
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = p ? p[at + k] : 0.0f;
    return num(v);
}
template <int V> __device__ __forceinline__ void store_small(float *p, int64_t at, Num<V> v) {
#pragma unroll
    for (int k = 0; k < V; ++k) p[at + k] = v.get(k);
}
template <int V> __device__ __forceinline__ Num<V> load_state(const float *p) {
    return widened<float>(*reinterpret_cast<const Pack<float, V> *>(p));
}
template <int V> __device__ __forceinline__ void store_state(float *p, Num<V> v) {
    *reinterpret_cast<Pack<float, V> *>(p) = rounded<float>(v);
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The affine maps s -> P s + C of all slices' chunks, exchanged: returns the value in front of this warp's chunk and moves
// *carry behind the last one.  `BACK`: the slices follow each other from the last to the first.  One buffer is written while
// the other may still be read, so one barrier per round is enough.
//
// Between the CTAs of a cluster the CTA's map travels as asynchronous stores that count their bytes on an mbarrier of the
// receiver.  A cluster barrier in their place has to wait until this round's stores of h are performed: 5300 cycles an
// exchange of eight CTAs against 1200 within one.
constexpr int kMaxWarps = 8, kMaxRanks = 8;
template <int V> struct Map { Num<V> P, C; };
template <int V> struct Exchange {
    Map<V> warp[2][kMaxWarps][32];
    Map<V> cta[2][kMaxRanks][32];
    uint64_t arrived[2];
    Patience patience;              // of the whole CTA, here and not in registers, which are short in the float32 backward pass
    uint8_t pad[111];
};
static_assert(sizeof(Exchange<1>) % 128 == 0 && sizeof(Exchange<2>) % 128 == 0, "the ring's boxes lie behind it");

__device__ __forceinline__ void store_async(uint32_t addr, uint32_t bar, Map<1> m) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];"
                 ::"r"(addr), "r"(__float_as_uint(m.P.a)), "r"(__float_as_uint(m.C.a)), "r"(bar) : "memory");
}
__device__ __forceinline__ void store_async(uint32_t addr, uint32_t bar, Map<2> m) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];"
                 ::"r"(addr), "l"(m.P.a.v), "l"(m.C.a.v), "r"(bar) : "memory");
}

// Barriers of a cluster's exchange; no CTA writes to another's shared memory before that one is through here.
template <int V> __device__ __forceinline__ void exchange_start(Exchange<V> &x, const Place &p) {
    if (p.ranks == 1) return;
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&x.arrived[0]), 1);
        mbar_init(smem_u32(&x.arrived[1]), 1);
        x.patience.gone = false;
        fence_mbar_init();
    }
    __syncthreads();
    cluster_sync();
}

// The gates of some ten closed steps multiply to less than the smallest float32, although no gate is 0 (gate() keeps f at
// 2^-126 and above), and 0 * inf would make NaN of an infinite state that a walk step by step keeps.  So a map's P stays at
// the smallest float32, which is as far off as rounding it to 0.
template <int V> __device__ __forceinline__ Num<V> not_zero(Num<V> P) {
    float r[V];
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = fmaxf(P.get(v), __int_as_float(1));
    return num(r);
}
// The smallest float32 in the columns where s is infinite, 0 in the others; false: there are none in the warp.
template <int V> __device__ __forceinline__ bool at_inf(Num<V> s, Num<V> *tiny) {
    float r[V];
    bool any = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const bool inf = fabsf(s.get(v)) == __int_as_float(0x7f800000);
        r[v] = inf ? __int_as_float(1) : 0.0f;
        any |= inf;
    }
    *tiny = num(r);
    return __any_sync(0xffffffffu, any);
}

// A wait that gives up raises the device error flag; from then on a warp waits for no more stages of its ring, and a CTA for no
// more messages of its cluster, but both keep taking part in the barriers.
__device__ __forceinline__ void wait_for(uint32_t bar, uint32_t parity, Patience &patience, int *err, int site) {
    patience.wait([&]() { return mbar_wait_bounded(bar, parity); }, [&]() { atomicExch(err, site); });
}

// refill() is called when all warps of the CTA have read their chunks.
template <int V, bool BACK, typename Refill>
__device__ __forceinline__ Num<V> exchange(Exchange<V> &x, int64_t round, const Place &p, Map<V> own, Num<V> *carry, int *err, Refill refill) {
    const int buf = (int)(round & 1);
    x.warp[buf][p.warp][p.lane] = {not_zero(own.P), own.C};
    __syncthreads();
    refill();
    Num<V> start = *carry;
    if (p.ranks > 1) {
        const uint32_t bar = smem_u32(&x.arrived[buf]);
        if (p.warp == 0) {
            if (p.lane == 0) mbar_arrive_expect_tx(bar, p.ranks * 32 * (uint32_t)sizeof(Map<V>));
            Map<V> t{all<V>(1.0f), all<V>(0.0f)};
#pragma unroll
            for (int k = 0; k < kMaxWarps; ++k) {
                if (k >= p.warps) break;
                const Map<V> m = x.warp[buf][BACK ? p.warps - 1 - k : k][p.lane];
                t.C = fma(m.P, t.C, m.C);
                t.P = not_zero(mul(t.P, m.P));
            }
            const uint32_t here = smem_u32(&x.cta[buf][p.rank][p.lane]);
            for (uint32_t r = 0; r < p.ranks; ++r) {
                uint32_t there, there_bar;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(r));
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there_bar) : "r"(bar), "r"(r));
                store_async(there, there_bar, t);
            }
        }
        wait_for(bar, (uint32_t)(round >> 1) & 1u, x.patience, err, 42);
        Num<V> s = *carry;
#pragma unroll
        for (int k = 0; k < kMaxRanks; ++k) {
            if (k >= (int)p.ranks) break;
            const int r = BACK ? (int)p.ranks - 1 - k : k;
            start = pick(r == (int)p.rank, s, start);
            const Map<V> m = x.cta[buf][r][p.lane];
            s = fma(m.P, s, m.C);
        }
        *carry = s;
    }
    Num<V> s = start, mine = start;
#pragma unroll
    for (int k = 0; k < kMaxWarps; ++k) {
        if (k >= p.warps) break;
        const int w = BACK ? p.warps - 1 - k : k;
        mine = pick(w == p.warp, s, mine);
        const Map<V> m = x.warp[buf][w][p.lane];
        s = fma(m.P, s, m.C);
    }
    if (p.ranks == 1) *carry = s;
    return mine;
}

// ---- how a chunk gets to its lanes ----------------------------------------------------------------------------------
// Ring: the chunks that a CTA's warps work on in one round are neighbours (in time with slices, in columns without), so ONE
// box per tensor brings them all, DEPTH rounds ahead, into a stage of shared memory.  Issued by the scanning warps, each for
// its own chunk, the requests cost them 340 cycles a round forward and 490 backward, a tenth and a quarter of their time.
// Without slices a warp of its own asks for the boxes.  With slices the last warp does, behind the exchange's barrier, when
// all have read the stage; a ninth warp would leave the others 96 registers each.  This needs 16-byte aligned rows.
// Without a ring (other layouts, and a few steps, where setting it up costs more) a warp loads its next chunk to registers
// while it works on the current one.
template <typename TT> struct Cut {
    static constexpr int kFwdT = sizeof(TT) == 2 ? 16 : 8;      // steps of a slice's chunk, forward, with a ring
    static constexpr int kFwdDepth = 3;
    static constexpr int kBwdDepth = sizeof(TT) == 2 ? 3 : 2;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
template <typename P> __device__ __forceinline__ P load_shared(uint32_t addr) {
    P p;
    if constexpr (sizeof(P) == 16) {
        uint4 v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
        memcpy(&p, &v, 16);
    } else if constexpr (sizeof(P) == 8) {
        uint2 v;
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
        memcpy(&p, &v, 8);
    } else {
        uint32_t v;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
        memcpy(&p, &v, 4);
    }
    return p;
}

// full: the stage's bytes are there; empty: all scanning warps have read it.
template <int DEPTH> struct Ring {
    uint32_t data, bars, bytes;
    int stage = 0;
    uint32_t phase = 0;
    Patience patience;
    __device__ __forceinline__ void start(uint32_t data_, uint32_t bars_, uint32_t bytes_, int readers) {
        data = data_; bars = bars_; bytes = bytes_;
        if (threadIdx.x == 0) {
            for (int s = 0; s < DEPTH; ++s) {
                mbar_init(bars + 8 * s, 1);
                mbar_init(bars + 8 * (DEPTH + s), readers);
            }
            fence_mbar_init();
        }
        __syncthreads();
    }
    __device__ __forceinline__ uint32_t at() const { return data + stage * bytes; }
    __device__ __forceinline__ uint32_t full() const { return bars + 8 * stage; }
    __device__ __forceinline__ uint32_t empty() const { return bars + 8 * (DEPTH + stage); }
    __device__ __forceinline__ void next() { if (++stage == DEPTH) { stage = 0; phase ^= 1; } }
    __device__ __forceinline__ void read(int lane) {       // this warp has read the stage
        __syncwarp();
        if (lane == 0) mbar_arrive(empty());
    }
};

constexpr int kBarBytes = 128;
template <int V> constexpr size_t ring_shared(size_t stage, int depth, bool split) {
    return (split ? sizeof(Exchange<V>) : 0) + kBarBytes + stage * depth;
}

// ---- forward --------------------------------------------------------------------------------------------------------
// A chunk scanned from 0 in registers, with the products of f: the state after step i is C[i] + P[i] c_in, whatever c_in
// turns out to be.  CLEAN: no step is padded.
template <typename TT, int V, int T, bool CLEAN, typename In>
__device__ __forceinline__ void scan_local(In in, Num<V> nb, unsigned flags, Num<V> (&C)[T], Num<V> (&P)[T]) {
    Num<V> lc = all<V>(0.0f), lp = all<V>(1.0f);
#pragma unroll
    for (int i = 0; i < T; ++i) {
        Num<V> x, g, f, keep;
        unpair<TT, V>(in(i), &x, &g);
        gate<V>(g, nb, &f, &keep);
        const bool pad = !CLEAN && ((flags >> i) & 1u);
        const Num<V> n = fma(f, lc, mul(keep, x));
        lc = CLEAN ? n : pick(pad, lc, n);
        lp = CLEAN ? mul(lp, f) : pick(pad, lp, mul(lp, f));
        C[i] = lc;
        P[i] = lp;
    }
}

template <typename TT, int V, int T, bool SPLIT, bool RING>
__global__ void __launch_bounds__(SPLIT ? 256 : RING ? 96 : 64, SPLIT ? 2 : RING ? 5 : 6)
linear_recurrence_fwd_kernel(const __grid_constant__ CUtensorMap map_u, const LinRecArgs a) {
    extern __shared__ __align__(128) uint8_t shared[];
    Exchange<V> *x = reinterpret_cast<Exchange<V> *>(shared);
    Place p;
    if (!find_place<V, SPLIT, RING>(a, &p)) return;
    const Num<V> nb = mul(load_small<V>(a.bias, p.j), all<V>(kNegLog2e));
    Num<V> carry = load_small<V>(a.first, p.col);
    const int slices = SPLIT ? p.warps * (int)p.ranks : 1;
    const int slice = SPLIT ? (int)p.rank * p.warps + p.warp : 0;
    const int64_t round = (int64_t)slices * T;
    int64_t left = a.L - (int64_t)slice * T;        // steps from the start of this warp's chunk to the end
    const TT *u = static_cast<const TT *>(a.u) + p.b * a.u_b + 2 * p.j + (int64_t)slice * T * a.u_t;
    TT *h = static_cast<TT *>(a.h) + p.col + (int64_t)slice * T * a.h_t;
    const uint8_t *mask = a.mask ? a.mask + p.b + (int64_t)slice * T * a.m_t : nullptr;
    const int64_t states_t = a.B * a.d;
    float *states = a.states ? a.states + (int64_t)slice * (T / kT) * states_t + p.col : nullptr;

    constexpr int DEPTH = Cut<TT>::kFwdDepth;
    constexpr uint32_t kRow = (SPLIT ? 1 : kSide) * 32 * V * 2 * sizeof(TT);       // of the box
    const int steps = SPLIT ? p.warps * T : T;
    const bool back = a.h_t < 0;                    // time runs backwards: the box's rows as well
    Ring<DEPTH> ring;
    int64_t box_left = a.L - (int64_t)p.rank * steps;           // steps from the box's first to the end
    auto ask = [&](int64_t n, uint32_t to, uint32_t bar) {
        if (n <= 0) return;                         // behind the end: the box's turn never comes
        mbar_arrive_expect_tx(bar, steps * kRow);
        tma_load_3d(to, &map_u, bar, 2 * (p.j - p.shift), (int)p.b, (int)(back ? n - steps : a.L - n));
    };
    if constexpr (RING) {
        const uint32_t base = smem_u32(shared) + (SPLIT ? (uint32_t)sizeof(Exchange<V>) : 0u);
        ring.start(base + kBarBytes, base, steps * kRow, p.warps);
        if (!SPLIT && p.warp >= p.warps) {          // the warp that asks (and, beside the last columns, one without any)
            if (p.lane == 0 && p.warp == kSide) {
                for (int64_t n = a.L, turn = 0; n > 0; n -= round, ++turn) {
                    if (turn >= DEPTH) wait_for(ring.empty(), ring.phase ^ 1, ring.patience, a.err, 41);
                    if (ring.patience.gone) break;
                    ask(n, ring.at(), ring.full());
                    ring.next();
                }
            }
            return;
        }
        if (SPLIT && threadIdx.x == 0)
            for (int s = 0; s < DEPTH; ++s) ask(box_left - s * round, ring.data + s * ring.bytes, ring.bars + 8 * s);
    }
    constexpr unsigned kAll = (unsigned)((1ull << T) - 1);
    Pack<TT, 2 * V> next[RING ? 1 : T];
    uint8_t next_pad;
    if constexpr (!RING) load_steps<TT, 2 * V, T>(next, u, a.u_t, left);
    next_pad = load_pad<T>(mask, a.m_t, left, p.lane, a.mask + p.b);
    if (SPLIT) exchange_start(*x, p);
    int64_t turn = 0;
    for (int64_t r0 = 0; r0 < a.L; r0 += round, ++turn, left -= round) {
        const unsigned flags = pad_flags<T>(mask, next_pad, left, p.lane);
        if (r0 + round < a.L) {
            if (mask) mask += round * a.m_t;
            next_pad = load_pad<T>(mask, a.m_t, left - round, p.lane, a.mask + p.b);
        }
        Pack<TT, 2 * V> cur[RING ? 1 : T];
        uint32_t row = 0;
        int32_t row_step = 0;
        if constexpr (RING) {
            if (box_left > 0) wait_for(ring.full(), ring.phase, ring.patience, a.err, 41);
            const int first = SPLIT ? p.warp * T : 0;
            row = ring.at() + (p.shift + (SPLIT ? 0 : p.warp * 32 * V)) * 2 * sizeof(TT) + (back ? steps - 1 - first : first) * kRow;
            row_step = back ? -(int32_t)kRow : (int32_t)kRow;
        } else {
#pragma unroll
            for (int i = 0; i < T; ++i) cur[i] = next[i];
            if (r0 + round < a.L) {
                u += round * a.u_t;
                load_steps<TT, 2 * V, T>(next, u, a.u_t, left - round);
            }
        }
        auto in = [&](int i) -> Pack<TT, 2 * V> {
            if constexpr (RING) return load_shared<Pack<TT, 2 * V>>(row + i * row_step);
            else return cur[i];
        };
        auto refill = [&]() {
            if (RING && threadIdx.x == (p.warps - 1) * 32 && !ring.patience.gone) ask(box_left - DEPTH * round, ring.at(), ring.full());
        };
        if constexpr (SPLIT) {
            Num<V> C[T], P[T];
            if (flags == 0) {
                scan_local<TT, V, T, true>(in, nb, flags, C, P);
            } else if (flags == kAll) {             // nothing but padding
#pragma unroll
                for (int i = 0; i < T; ++i) { C[i] = all<V>(0.0f); P[i] = all<V>(1.0f); }
            } else {
                scan_local<TT, V, T, false>(in, nb, flags, C, P);
            }
            const Num<V> c = exchange<V, false>(*x, turn, p, Map<V>{P[T - 1], C[T - 1]}, &carry, a.err, refill);
            Num<V> tiny;
            if (at_inf(c, &tiny)) {
#pragma unroll
                for (int i = 0; i < T; ++i) P[i] = add(P[i], tiny);     // the other columns keep their bits
            }
            if (states) {
#pragma unroll
                for (int i = 0; i < T; i += kT)
                    if (i < left) store_state<V>(states + (i / kT) * states_t, i ? fma(P[i - 1], c, C[i - 1]) : c);
            }
            TT *q = h;
            if (flags == 0) {
#pragma unroll
                for (int i = 0; i < T; ++i, q += a.h_t)
                    *reinterpret_cast<Pack<TT, V> *>(q) = rounded<TT>(fma(P[i], c, C[i]));
            } else {
#pragma unroll
                for (int i = 0; i < T; ++i, q += a.h_t)
                    if (i < left)
                        *reinterpret_cast<Pack<TT, V> *>(q) = rounded<TT>(pick((flags >> i) & 1u, all<V>(0.0f), fma(P[i], c, C[i])));
            }
        } else {
            TT *q = h;
            auto walk = [&](auto clean) {
                constexpr bool CLEAN = decltype(clean)::value;
#pragma unroll
                for (int i = 0; i < T; ++i, q += a.h_t) {
                    if (i % kT == 0 && states && (CLEAN || i < left)) store_state<V>(states + (i / kT) * states_t, carry);
                    Num<V> xi, g, f, keep;
                    unpair<TT, V>(in(i), &xi, &g);
                    gate<V>(g, nb, &f, &keep);
                    const bool pad = !CLEAN && ((flags >> i) & 1u);
                    const Num<V> n = fma(f, carry, mul(keep, xi));
                    carry = CLEAN ? n : pick(pad, carry, n);
                    if (CLEAN || i < left)
                        *reinterpret_cast<Pack<TT, V> *>(q) = rounded<TT>(CLEAN ? n : pick(pad, all<V>(0.0f), n));
                }
            };
            if (flags == 0) walk(std::true_type());
            else walk(std::false_type());
            if (RING) ring.read(p.lane);
        }
        if (RING) ring.next();
        box_left -= round;
        h += round * a.h_t;
        if (states) states += (int64_t)slices * (T / kT) * states_t;
    }
    if (SPLIT && p.ranks > 1) cluster_sync();       // a CTA's last message has arrived before its sender or receiver is gone
    if (slice == 0 && a.last) store_small<V>(a.last, p.col, carry);
}

// ---- backward -------------------------------------------------------------------------------------------------------
template <typename TT, int V, bool SPLIT, bool RING>
__global__ void __launch_bounds__(SPLIT ? 256 : RING ? 96 : 64, SPLIT ? 2 : RING ? 5 : 6)
linear_recurrence_bwd_kernel(const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_g,
                             const __grid_constant__ CUtensorMap map_s, const LinRecArgs a) {
    extern __shared__ __align__(128) uint8_t shared[];
    Exchange<V> *x = reinterpret_cast<Exchange<V> *>(shared);
    constexpr int T = kT;
    Place p;
    if (!find_place<V, SPLIT, RING>(a, &p)) return;
    const Num<V> nb = mul(load_small<V>(a.bias, p.j), all<V>(kNegLog2e));
    Num<V> carry = load_small<V>(a.first, p.col), db = all<V>(0.0f);
    const int slices = SPLIT ? p.warps * (int)p.ranks : 1;
    const int slice = SPLIT ? (int)p.rank * p.warps + p.warp : 0;
    const int64_t round = (int64_t)slices * T;
    const int64_t r_top = (a.L - 1) / round * round, t_top = r_top + (int64_t)slice * T;
    int64_t left = a.L - t_top;
    const TT *u = static_cast<const TT *>(a.u) + p.b * a.u_b + 2 * p.j + t_top * a.u_t;
    const TT *gh = a.grad_h ? static_cast<const TT *>(a.grad_h) + p.b * a.gh_b + p.j + t_top * a.gh_t : nullptr;
    TT *gu = static_cast<TT *>(a.h) + 2 * (p.col + t_top * a.h_t);
    const uint8_t *mask = a.mask ? a.mask + p.b + t_top * a.m_t : nullptr;
    const int64_t states_t = a.B * a.d;
    const float *states = a.states + (t_top / T) * states_t + p.col;

    constexpr int DEPTH = Cut<TT>::kBwdDepth;
    constexpr uint32_t kCols = (SPLIT ? 1 : kSide) * 32 * V, kRowU = kCols * 2 * sizeof(TT), kRowG = kCols * sizeof(TT), kRowS = kCols * 4;
    const int chunks = SPLIT ? p.warps : 1, steps = chunks * T;     // of a box
    const uint32_t g_at = steps * kRowU, s_at = g_at + steps * kRowG, stage_bytes = s_at + chunks * kRowS;
    const bool back = a.h_t < 0;
    Ring<DEPTH> ring;
    int64_t box_left = a.L - (r_top + (int64_t)p.rank * steps);      // steps from the box's first to the end
    auto ask = [&](int64_t n, uint32_t to, uint32_t bar) {
        if (n > a.L) return;                        // in front of the start
        if (n <= 0) { mbar_arrive(bar); return; }   // behind the end (first round only): the stage's turn passes empty
        const int t = (int)(back ? n - steps : a.L - n), j0 = p.j - p.shift;
        mbar_arrive_expect_tx(bar, gh ? stage_bytes : stage_bytes - steps * kRowG);
        tma_load_3d(to, &map_u, bar, 2 * j0, (int)p.b, t);
        if (gh) tma_load_3d(to + g_at, &map_g, bar, j0, (int)p.b, t);
        tma_load_3d(to + s_at, &map_s, bar, j0, (int)p.b, (int)((a.L - n) / T));
    };
    if constexpr (RING) {
        const uint32_t base = smem_u32(shared) + (SPLIT ? (uint32_t)sizeof(Exchange<V>) : 0u);
        ring.start(base + kBarBytes, base, stage_bytes, p.warps);
        if (!SPLIT && p.warp >= p.warps) {
            if (p.lane == 0 && p.warp == kSide) {
                for (int64_t n = box_left, turn = 0; n <= a.L; n += round, ++turn) {
                    if (turn >= DEPTH) wait_for(ring.empty(), ring.phase ^ 1, ring.patience, a.err, 41);
                    if (ring.patience.gone) break;
                    ask(n, ring.at(), ring.full());
                    ring.next();
                }
            }
            return;
        }
        if (SPLIT && threadIdx.x == 0)
            for (int s = 0; s < DEPTH; ++s) ask(box_left + s * round, ring.data + s * ring.bytes, ring.bars + 8 * s);
    }
    constexpr unsigned kAll = (1u << T) - 1u;
    Pack<TT, 2 * V> next_u[RING ? 1 : T];
    Pack<TT, V> next_g[RING ? 1 : T];
    Num<V> next_c = all<V>(0.0f);
    uint8_t next_pad;
    auto fetch = [&](int64_t n) {
        if constexpr (!RING) {
            if (n > 0) next_c = load_state<V>(states);
            load_steps<TT, 2 * V, T>(next_u, u, a.u_t, n);
            if (gh) load_steps<TT, V, T>(next_g, gh, a.gh_t, n);
            else memset(&next_g, 0, sizeof(next_g));
        }
        next_pad = load_pad<T>(mask, a.m_t, n, p.lane, a.mask + p.b);
    };
    fetch(left);
    if (SPLIT) exchange_start(*x, p);
    int64_t turn = 0;
    for (int64_t r0 = r_top; r0 >= 0; r0 -= round, ++turn, left += round) {
        const unsigned flags = pad_flags<T>(mask, next_pad, left, p.lane);
        Num<V> c = next_c;
        Num<V> f[T], keep[T], w[T];      // w = (c_{t-1} - x) f (1 - f)
        Pack<TT, V> g[T];
        Pack<TT, 2 * V> cur[RING ? 1 : T];
        uint32_t row = 0;
        int32_t row_step = 0;
        if constexpr (!RING) {
#pragma unroll
            for (int i = 0; i < T; ++i) { cur[i] = next_u[i]; g[i] = next_g[i]; }
        }
        if (r0 > 0) {
            if constexpr (!RING) {
                u -= round * a.u_t;
                if (gh) gh -= round * a.gh_t;
            }
            if (mask) mask -= round * a.m_t;
            states -= (int64_t)slices * states_t;
            fetch(left + round);
        }
        if constexpr (RING) {
            wait_for(ring.full(), ring.phase, ring.patience, a.err, 41);
            const int first = SPLIT ? p.warp * T : 0, cols = p.shift + (SPLIT ? 0 : p.warp * 32 * V);
            const int at = back ? steps - 1 - first : first;
            row = ring.at() + cols * 2 * sizeof(TT) + at * kRowU;
            row_step = back ? -(int32_t)kRowU : (int32_t)kRowU;
            c = widened<float>(load_shared<Pack<float, V>>(ring.at() + s_at + (SPLIT ? p.warp : 0) * kRowS + cols * 4));
            uint32_t grow = ring.at() + g_at + cols * sizeof(TT) + at * kRowG;
#pragma unroll
            for (int i = 0; i < T; ++i, grow += row_step / 2) {
                if (gh) g[i] = load_shared<Pack<TT, V>>(grow);
                else memset(&g[i], 0, sizeof(g[i]));
            }
        }
        auto in = [&](int i) -> Pack<TT, 2 * V> {
            if constexpr (RING) return load_shared<Pack<TT, 2 * V>>(row + i * row_step);
            else return cur[i];
        };
        const Num<V> zero = all<V>(0.0f), one = all<V>(1.0f);
        Map<V> own{one, zero};
        auto recompute = [&](auto clean) {
            constexpr bool CLEAN = decltype(clean)::value;
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const bool pad = !CLEAN && ((flags >> i) & 1u);
                Num<V> xi, gi, fi, ki;
                unpair<TT, V>(in(i), &xi, &gi);
                gate<V>(gi, nb, &fi, &ki);
                const Num<V> wi = mul(mul(sub(c, xi), fi), ki), ci = fma(fi, c, mul(ki, xi));
                w[i] = CLEAN ? wi : pick(pad, zero, wi);
                c = CLEAN ? ci : pick(pad, c, ci);
                f[i] = CLEAN ? fi : pick(pad, one, fi);
                keep[i] = CLEAN ? ki : pick(pad, zero, ki);
            }
            if constexpr (SPLIT) {
#pragma unroll
                for (int i = T - 1; i >= 0; --i) {
                    const bool pad = !CLEAN && ((flags >> i) & 1u);
                    const Num<V> s = add(own.C, widened<TT>(g[i]));
                    own.C = mul(f[i], CLEAN ? s : pick(pad, own.C, s));
                    own.P = mul(own.P, f[i]);
                }
            }
        };
        if (flags == 0) {
            recompute(std::true_type());
        } else if (flags == kAll) {                 // nothing but padding
#pragma unroll
            for (int i = 0; i < T; ++i) { f[i] = one; keep[i] = zero; w[i] = zero; }
        } else {
            recompute(std::false_type());
        }
        Num<V> dc = carry;
        if constexpr (SPLIT) {
            dc = exchange<V, true>(*x, turn, p, own, &carry, a.err, [&]() {
                if (RING && threadIdx.x == (p.warps - 1) * 32 && !ring.patience.gone) ask(box_left + DEPTH * round, ring.at(), ring.full());
            });
        } else if constexpr (RING) {
            ring.read(p.lane);
        }
        if (RING) ring.next();
        box_left += round;
        auto finish = [&](auto clean) {
            constexpr bool CLEAN = decltype(clean)::value;
            TT *q = gu + 2 * (T - 1) * a.h_t;
#pragma unroll
            for (int i = T - 1; i >= 0; --i, q -= 2 * a.h_t) {
                const bool pad = !CLEAN && ((flags >> i) & 1u);
                const Num<V> s = add(dc, widened<TT>(g[i]));
                const Num<V> total = CLEAN ? s : pick(pad, dc, s);
                Num<V> dx = mul(keep[i], total), dg = mul(w[i], total);
                if (!CLEAN) { dx = pick(pad, zero, dx); dg = pick(pad, zero, dg); }
                db = add(db, dg);
                dc = mul(f[i], total);
                Pack<TT, 2 * V> out;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const Pack<TT, 2> o = pack2<TT>(dx.get(v), dg.get(v));
                    out.v[2 * v] = o.v[0];
                    out.v[2 * v + 1] = o.v[1];
                }
                if (CLEAN || i < left) *reinterpret_cast<Pack<TT, 2 * V> *>(q) = out;
            }
        };
        if (flags == 0) finish(std::true_type());
        else finish(std::false_type());
        if (!SPLIT) carry = dc;
        gu -= 2 * round * a.h_t;
    }
    if (SPLIT && p.ranks > 1) cluster_sync();
    if (a.last && slice == 0) store_small<V>(a.last, p.col, carry);
    if (a.bias_part) store_small<V>(a.bias_part, (p.b * slices + slice) * a.d + p.j, db);
}

// grad_bias[j] = sum over the parts in a fixed order: 8 slices of the parts per column, then the slices.
__global__ void __launch_bounds__(256)
linear_recurrence_bias_kernel(float *__restrict__ out, const float *__restrict__ part, int64_t parts, int d) {
    __shared__ float s[8][32];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int j = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (j < d)
        for (int64_t p = slice; p < parts; p += 8) v += part[p * d + j];
    s[slice][lane] = v;
    __syncthreads();
    if (slice == 0 && j < d) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += s[k][lane];
        out[j] = t;
    }
}

int check_sizes(int64_t L, int64_t B, int64_t d, int dtype) {
    if (L < 0 || B < 0 || d < 1 || d > (1 << 28))
        return set_error(SRU_ERR_BAD_ARG, "bad sizes L=%lld B=%lld d=%lld", (long long)L, (long long)B, (long long)d);
    if (dtype != SRU_F32 && dtype != SRU_F16 && dtype != SRU_BF16)
        return set_error(SRU_ERR_UNSUPPORTED, "linear recurrence: dtype must be float32, float16 or bfloat16, got %d", dtype);
    return 0;
}

// Moves the bases to the last time step and turns the time strides round: the kernels then run a reversed scan as is.
void reverse_time(LinRecArgs *a, size_t size, int units) {
    const int64_t n = a->L - 1;
    a->u = static_cast<const char *>(a->u) + n * a->u_t * (int64_t)size;
    a->h = static_cast<char *>(a->h) + n * a->h_t * (int64_t)size * units;
    if (a->grad_h) a->grad_h = static_cast<const char *>(a->grad_h) + n * a->gh_t * (int64_t)size;
    if (a->mask) a->mask += n * a->m_t;
    a->u_t = -a->u_t; a->h_t = -a->h_t; a->gh_t = -a->gh_t; a->m_t = -a->m_t;
}

Slices choose_slices(int64_t L, int64_t B, int64_t d, int dtype, bool backward) {
    const int64_t columns = (d + 63) / 64 * B;              // warps that one walk over time takes
    int64_t want = option(OPT_LINREC_SLICES, 0);
    // One walk takes about 70 ns a step forward and 120 backward however few columns there are, which is what HBM needs
    // for some 70 000 columns: with 1024 warps of columns (512 x 32 x 2048) one walk takes 37 / 63 us, four slices 44 / 68.
    // With fewer, slices fill the GPU with up to 14 warps an SM, all it holds at their register count, and four at least:
    // 640 warps (2048 x 40 x 1024) 110 / 216 us in two slices, 99 / 193 in four; 384 (4096 x 24 x 1024) 112 / 219 in four, 121 /
    // 226 in eight; 256 (8192 x 16 x 1024) 166 / 341 in four, 148 / 281 in eight, 181 / 344 in sixteen; 32 (65536 x 2048) 2410 in
    // one walk and 193 in 64.
    if (want <= 0) {
        want = columns < kSms * 6 ? 4 : 1;
        if (want > 1)
            while (want < 64 && columns * want * 2 <= kSms * 14) want *= 2;
    }
    // two CTAs an SM: eight warps' float32 stages of the backward pass would leave room for one (4096 x 4 x 512 in 64 slices
    // 75 us, in 56 of seven warps 49)
    const int most = dtype == SRU_F32 && backward ? kMaxWarps - 1 : kMaxWarps;
    want = std::min<int64_t>(std::min<int64_t>(want, most * kMaxRanks), (L + kT - 1) / kT);
    Slices s;
    s.ranks = (int)((want + most - 1) / most);
    s.warps = (int)((want + s.ranks - 1) / s.ranks);
    return s;
}

// Boxes of `cols` elements, one sequence and `steps` steps; outside reads as zero.
template <typename TT>
int make_box(CUtensorMap *map, const void *base, int64_t inner, int64_t B, int64_t L, int64_t s_b, int64_t s_t, int cols, int steps) {
    auto fn = get_encode_fn();
    if (!fn) return set_error(SRU_ERR_CUDA, "cuTensorMapEncodeTiled entry point not found");
    const CUtensorMapDataType type = sizeof(TT) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : std::is_same<TT, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)B, (cuuint64_t)L};
    cuuint64_t strides[2] = {(cuuint64_t)s_b * sizeof(TT), (cuuint64_t)s_t * sizeof(TT)};
    cuuint32_t box[3] = {(cuuint32_t)cols, 1, (cuuint32_t)steps}, estr[3] = {1, 1, 1};
    CUresult r = fn(map, type, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(SRU_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return 0;
}

struct Maps { CUtensorMap u, g, s; };

template <typename TT, int V, bool SPLIT, bool RING>
int launch(LinRecArgs a, const Slices &s, const Maps &maps, bool backward, cudaStream_t st) {
    // a slice's chunk is the same with and without a ring, and with it the order of all roundings: bits do not depend on layout
    constexpr int T = SPLIT || RING ? Cut<TT>::kFwdT : 2 * kT;
    constexpr size_t kRow = (SPLIT ? 1 : kSide) * 32 * V * 2 * sizeof(TT);
    auto fwd = linear_recurrence_fwd_kernel<TT, V, T, SPLIT, RING>;
    auto bwd = linear_recurrence_bwd_kernel<TT, V, SPLIT, RING>;
    a.groups = (a.d + 32 * V - 1) / (32 * V);
    const int64_t columns = (int64_t)a.groups * a.B;
    const int warps = SPLIT ? s.warps : kSide;
    const int64_t blocks = SPLIT ? columns * s.ranks : RING ? (int64_t)((a.groups + kSide - 1) / kSide) * a.B : (columns + kSide - 1) / kSide;
    if (blocks > 0x7fffffff) return set_error(SRU_ERR_UNSUPPORTED, "linear recurrence: batch * hidden too large");
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.stream = st;
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3(32 * (warps + (RING && !SPLIT ? 1 : 0)), 1, 1);
    cfg.dynamicSmemBytes = SPLIT ? sizeof(Exchange<V>) : 0;
    if (RING) {
        auto fwd_bytes = [&](int n) { return ring_shared<V>(n * T * kRow, Cut<TT>::kFwdDepth, SPLIT); };
        auto bwd_bytes = [&](int n) { return ring_shared<V>(n * (kT * kRow * 3 / 2 + kRow / (2 * sizeof(TT)) * 4), Cut<TT>::kBwdDepth, SPLIT); };
        static bool attr_set[64] = {false};
        int dev = 0;
        SRUB_CUDA_CHECK(cudaGetDevice(&dev));
        if (dev >= 0 && dev < 64 && !attr_set[dev]) {
            SRUB_CUDA_CHECK(cudaFuncSetAttribute(fwd, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fwd_bytes(SPLIT ? kMaxWarps : 1)));
            SRUB_CUDA_CHECK(cudaFuncSetAttribute(bwd, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bwd_bytes(SPLIT ? kMaxWarps : 1)));
            attr_set[dev] = true;
        }
        cfg.dynamicSmemBytes = backward ? bwd_bytes(SPLIT ? warps : 1) : fwd_bytes(SPLIT ? warps : 1);
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s.ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = SPLIT ? 1 : 0;
    if (backward) SRUB_LAUNCH(&cfg, bwd, maps.u, maps.g, maps.s, a);
    else SRUB_LAUNCH(&cfg, fwd, maps.u, a);
    return 0;
}

// Two columns per lane and a ring where all rows are 16-byte aligned and pairs of columns aligned to their size.
bool ring_fits(const LinRecArgs &a, int64_t size, bool backward) {
    auto at = [](const void *p, int64_t unit) { return reinterpret_cast<uintptr_t>(p) % unit == 0; };
    auto rows = [&](const void *p, int64_t t, int64_t b) {
        return at(p, 16) && t > 0 && t * size % 16 == 0 && (a.B == 1 || (b > 0 && b * size % 16 == 0));
    };
    if (a.L < 2 * kT || a.d % 4 || a.L > 0x7fffffff - 1024 || a.B > 0x7fffffff || !at(a.states, 16)) return false;
    if (!at(a.h, (backward ? 4 : 2) * size) || !rows(a.u, a.u_t, a.u_b)) return false;
    return !a.grad_h || rows(a.grad_h, a.gh_t, a.gh_b);
}

template <typename TT> int launch_typed(LinRecArgs a, const Slices &s, bool reverse, bool backward, cudaStream_t st) {
    Maps maps;
    memset(&maps, 0, sizeof(maps));
    const bool ring = ring_fits(a, sizeof(TT), backward), split = s.count() > 1;
    if (ring) {
        if (int rc = ensure_context()) return rc;
        const bool one = a.B == 1;       // the stride of a single sequence is never taken
        const int cols = split ? 64 : 64 * kSide, chunks = split ? s.warps : 1;
        const int steps = chunks * (backward ? kT : Cut<TT>::kFwdT);
        int rc = make_box<TT>(&maps.u, a.u, 2 * a.d, a.B, a.L, one ? a.u_t : a.u_b, a.u_t, 2 * cols, steps);
        if (!rc && a.grad_h) rc = make_box<TT>(&maps.g, a.grad_h, a.d, a.B, a.L, one ? a.gh_t : a.gh_b, a.gh_t, cols, steps);
        if (!rc && backward)
            rc = make_box<float>(&maps.s, a.states, a.d, a.B, (a.L + kT - 1) / kT, a.d, a.B * a.d, cols, chunks);
        if (rc) return rc;
    }
    a.err = device_error_flag();
    if (!a.err) return set_error(SRU_ERR_CUDA, "device error flag unavailable");
    if (reverse) reverse_time(&a, sizeof(TT), backward ? 2 : 1);
    if (ring) return split ? launch<TT, 2, true, true>(a, s, maps, backward, st) : launch<TT, 2, false, true>(a, s, maps, backward, st);
    return split ? launch<TT, 1, true, false>(a, s, maps, backward, st) : launch<TT, 1, false, false>(a, s, maps, backward, st);
}

int dispatch(const LinRecArgs &a, const Slices &s, int dtype, bool reverse, bool backward, cudaStream_t st) {
    switch (dtype) {
        case SRU_F16: return launch_typed<__half>(a, s, reverse, backward, st);
        case SRU_BF16: return launch_typed<__nv_bfloat16>(a, s, reverse, backward, st);
        default: return launch_typed<float>(a, s, reverse, backward, st);
    }
}

}  // namespace

}  // namespace srub

using namespace srub;

extern "C" {

size_t sru_b200_linear_recurrence_states_bytes(int64_t length, int64_t batch, int64_t hidden) {
    if (length < 1 || batch < 1 || hidden < 1) return 0;
    return (size_t)((length + kT - 1) / kT) * (size_t)batch * (size_t)hidden * sizeof(float);
}

int sru_b200_linear_recurrence_forward(void *h, float *c_last, void *states, const void *u, const float *bias,
                                       const float *c_init, const uint8_t *mask_pad, int64_t length, int64_t batch,
                                       int64_t hidden, int64_t u_stride_t, int64_t u_stride_b, int reverse, int dtype,
                                       void *stream) {
    int rc = check_sizes(length, batch, hidden, dtype);
    if (rc) return rc;
    if (length == 0 || batch == 0) return 0;
    if (!h || !u) return set_error(SRU_ERR_BAD_ARG, "linear recurrence: h and u must not be null");
    const size_t size = dtype_size(dtype);
    if ((reinterpret_cast<uintptr_t>(u) % (2 * size)) || u_stride_t % 2 || u_stride_b % 2)
        return set_error(SRU_ERR_BAD_ARG, "linear recurrence: the pairs of u must be aligned to their size");
    if (reinterpret_cast<uintptr_t>(states) % sizeof(float))
        return set_error(SRU_ERR_BAD_ARG, "linear recurrence: states must be aligned to 4 bytes");
    LinRecArgs a;
    memset(&a, 0, sizeof(a));
    a.h = h; a.last = c_last; a.states = static_cast<float *>(states);
    a.u = u; a.bias = bias; a.first = c_init; a.mask = mask_pad;
    a.L = length; a.B = batch; a.d = (int)hidden;
    a.u_t = u_stride_t; a.u_b = u_stride_b;
    a.h_t = batch * hidden; a.m_t = batch;
    return dispatch(a, choose_slices(length, batch, hidden, dtype, false), dtype, reverse != 0, false, static_cast<cudaStream_t>(stream));
}

size_t sru_b200_linear_recurrence_backward_workspace_bytes(int64_t length, int64_t batch, int64_t hidden, int dtype) {
    if (length < 1 || batch < 1 || hidden < 1) return 0;
    return (size_t)batch * choose_slices(length, batch, hidden, dtype, true).count() * (size_t)hidden * sizeof(float);
}

int sru_b200_linear_recurrence_backward(void *grad_u, float *grad_bias, float *grad_init, const void *u,
                                        const float *bias, const void *states, const uint8_t *mask_pad,
                                        const void *grad_h, const float *grad_last, int64_t length, int64_t batch,
                                        int64_t hidden, int64_t u_stride_t, int64_t u_stride_b, int64_t gh_stride_t,
                                        int64_t gh_stride_b, int reverse, int dtype, void *workspace,
                                        size_t workspace_bytes, void *stream) {
    int rc = check_sizes(length, batch, hidden, dtype);
    if (rc) return rc;
    if (length == 0 || batch == 0) return 0;
    if (!grad_u || !u || !states) return set_error(SRU_ERR_BAD_ARG, "linear recurrence: a required pointer is null");
    const size_t size = dtype_size(dtype);
    if ((reinterpret_cast<uintptr_t>(u) % (2 * size)) || u_stride_t % 2 || u_stride_b % 2)
        return set_error(SRU_ERR_BAD_ARG, "linear recurrence: the pairs of u must be aligned to their size");
    if (reinterpret_cast<uintptr_t>(grad_u) % (2 * size))
        return set_error(SRU_ERR_BAD_ARG, "linear recurrence: the pairs of grad_u must be aligned to their size");
    if (reinterpret_cast<uintptr_t>(states) % sizeof(float))
        return set_error(SRU_ERR_BAD_ARG, "linear recurrence: states must be aligned to 4 bytes");
    const Slices s = choose_slices(length, batch, hidden, dtype, true);
    if (grad_bias) {
        const size_t need = (size_t)batch * s.count() * (size_t)hidden * sizeof(float);
        if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % sizeof(float))
            return set_error(SRU_ERR_WORKSPACE, "4-byte aligned workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    }
    LinRecArgs a;
    memset(&a, 0, sizeof(a));
    a.h = grad_u; a.last = grad_init; a.states = const_cast<float *>(static_cast<const float *>(states));
    a.bias_part = grad_bias ? static_cast<float *>(workspace) : nullptr;
    a.u = u; a.bias = bias; a.first = grad_last; a.grad_h = grad_h; a.mask = mask_pad;
    a.L = length; a.B = batch; a.d = (int)hidden;
    a.u_t = u_stride_t; a.u_b = u_stride_b; a.gh_t = gh_stride_t; a.gh_b = gh_stride_b;
    a.h_t = batch * hidden; a.m_t = batch;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rc = dispatch(a, s, dtype, reverse != 0, true, st);
    if (rc || !grad_bias) return rc;
    linear_recurrence_bias_kernel<<<(unsigned)((hidden + 31) / 32), 256, 0, st>>>(grad_bias, a.bias_part,
                                                                                   batch * s.count(), (int)hidden);
    SRUB_LAUNCHED();
    return 0;
}

}  // extern "C"
