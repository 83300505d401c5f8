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
// HBM-bound: 3 elements per column-step forward, 5 backward.  A lane owns V adjacent columns of one sequence and walks
// time in chunks of kT steps; the next chunk's loads are issued before the current chunk is worked on.  The forward
// pass leaves the float32 state in front of every chunk (kT = 16: a quarter of a byte per column-step); the backward
// pass recomputes the states of a chunk from it, which is cheaper than reading a saved history (2 or 4 bytes) and
// exact in the 16-bit types, whose rounded h would enter c_{t-1} - x_t.
//
// Arithmetic is float32 throughout.  With e = 2^(-(g + bias) log2 e), f = 1 / (1 + e) and 1 - f = e f: both keep their
// relative accuracy however close to 0 or 1 the gate is.
#include <algorithm>
#include <cstring>

#include "common.cuh"

namespace srub {

namespace {

constexpr int kT = 16;          // steps per chunk, and between two saved states

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
};

__device__ __forceinline__ float min_nan(float a, float b) {     // NaN if either is
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// One step's pair of u, as loaded.
template <typename TT> struct PairLoad {
    Pack<TT, 2> p;
    __device__ __forceinline__ float x() const { return Cvt<TT>::to_f(p.v[0]); }
    __device__ __forceinline__ float g() const { return Cvt<TT>::to_f(p.v[1]); }
};

template <typename P> __device__ __forceinline__ P zero_pack() {
    P p;
    memset(&p, 0, sizeof(P));
    return p;
}

// T steps of a strided stream of N elements per lane and step; steps from `n` on are left zero and not read.
template <typename TT, int N, int T>
__device__ __forceinline__ void load_steps(Pack<TT, N> (&r)[T], const TT *p, int64_t stride, int64_t n, bool on) {
    if (on && n >= T) {
#pragma unroll
        for (int i = 0; i < T; ++i) r[i] = *reinterpret_cast<const Pack<TT, N> *>(p + i * stride);
    } else {
#pragma unroll
        for (int i = 0; i < T; ++i)
            r[i] = (on && i < n) ? *reinterpret_cast<const Pack<TT, N> *>(p + i * stride) : zero_pack<Pack<TT, N>>();
    }
}

// Bit i: step i of the chunk is padded or lies behind the end.  The whole warp works on one sequence, so the flags are
// uniform; lane i fetches step i's byte.
template <int T> __device__ __forceinline__ unsigned load_flags(const uint8_t *mask, int64_t stride, int64_t n, int lane) {
    bool pad = lane >= n;
    if (mask && lane < T && lane < n) pad = mask[lane * stride] != 0;
    return __ballot_sync(0xffffffffu, pad);
}

// f and 1 - f from the gate's logit; nb = -bias * log2(e)
__device__ __forceinline__ void gate(float g, float nb, float *f, float *keep) {
    const float e = ex2_approx(min_nan(fmaf(g, kNegLog2e, nb), 126.0f));    // at most 2^126, so that e * f stays finite
    *f = rcp_approx(1.0f + e);
    *keep = e * *f;
}

// Where a warp stands: its sequence and column, and which of the `slices` interleaved parts of time it works on.  Slices are
// the warps of a CTA and the CTAs of a cluster; chunk k of a column belongs to slice k mod slices.
struct Place {
    int lane, warp, warps;          // of the CTA
    uint32_t rank, ranks;           // of the cluster
    int64_t b, col;
    int j;
    bool on;
};

template <bool SPLIT> __device__ __forceinline__ bool find_place(const LinRecArgs &a, Place *p) {
    p->lane = threadIdx.x & 31;
    p->warp = threadIdx.x >> 5;
    p->warps = blockDim.x >> 5;
    p->rank = 0; p->ranks = 1;
    int64_t wid;
    if (SPLIT) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(p->rank));
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(p->ranks));
        wid = blockIdx.x / p->ranks;
    } else {
        wid = (int64_t)blockIdx.x * p->warps + p->warp;
    }
    p->b = wid / a.groups;
    p->j = (int)(wid - p->b * a.groups) * 32 + p->lane;
    p->on = p->j < a.d;
    p->col = p->b * a.d + p->j;
    return p->b < a.B;
}

// The affine maps s -> P s + C of all slices' chunks, exchanged: returns the value in front of this warp's chunk and moves
// *carry behind the last one.  `back`: the slices follow each other from the last to the first.  One buffer is written while
// the other may still be read, so one barrier per round is enough.
constexpr int kMaxWarps = 8, kMaxRanks = 8;
struct Exchange {
    float2 warp[2][kMaxWarps][32];
    float2 cta[2][kMaxRanks][32];
};

__device__ __forceinline__ float exchange(Exchange &x, int buf, const Place &p, float P, float C, bool back, float *carry) {
    x.warp[buf][p.warp][p.lane] = make_float2(P, C);
    __syncthreads();
    float start = *carry;
    if (p.ranks > 1) {
        if (p.warp == 0) {
            float tp = 1.0f, tc = 0.0f;
            for (int k = 0; k < p.warps; ++k) {
                const float2 m = x.warp[buf][back ? p.warps - 1 - k : k][p.lane];
                tc = fmaf(m.x, tc, m.y);
                tp *= m.x;
            }
            const uint32_t here = smem_u32(&x.cta[buf][p.rank][p.lane]);
            for (uint32_t r = 0; r < p.ranks; ++r) {
                uint32_t there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(r));
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(tp), "f"(tc) : "memory");
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        float s = *carry;
        for (uint32_t k = 0; k < p.ranks; ++k) {
            const uint32_t r = back ? p.ranks - 1 - k : k;
            if (r == p.rank) start = s;
            const float2 m = x.cta[buf][r][p.lane];
            s = fmaf(m.x, s, m.y);
        }
        *carry = s;
    }
    float s = start, mine = start;
    for (int k = 0; k < p.warps; ++k) {
        const int w = back ? p.warps - 1 - k : k;
        if (w == p.warp) mine = s;
        const float2 m = x.warp[buf][w][p.lane];
        s = fmaf(m.x, s, m.y);
    }
    if (p.ranks == 1) *carry = s;
    return mine;
}

// No CTA of a cluster writes to another's shared memory before that one has started.
__device__ __forceinline__ void cluster_started(const Place &p) {
    if (p.ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// SPLIT: the slices' chunks are scanned locally, c_t = C_t + P_t c_in, and finished once c_in is known.
template <typename TT, int T, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 256 : 64, SPLIT ? 3 : 8)
linear_recurrence_fwd_kernel(const LinRecArgs a) {
    __shared__ Exchange x[1];
    Place p;
    if (!find_place<SPLIT>(a, &p)) return;
    const TT *u = static_cast<const TT *>(a.u) + p.b * a.u_b + 2 * p.j;
    TT *h = static_cast<TT *>(a.h) + p.col;
    const uint8_t *mask = a.mask ? a.mask + p.b : nullptr;
    const float nb = (p.on && a.bias) ? a.bias[p.j] * kNegLog2e : 0.0f;
    float carry = (p.on && a.first) ? a.first[p.col] : 0.0f;
    const int slices = SPLIT ? p.warps * (int)p.ranks : 1;
    const int slice = SPLIT ? (int)p.rank * p.warps + p.warp : 0;
    const int64_t round = (int64_t)slices * T;
    Pack<TT, 2> next[T];
    unsigned next_flags;
    auto fetch = [&](int64_t t0) {
        load_steps<TT, 2, T>(next, u + t0 * a.u_t, a.u_t, a.L - t0, p.on);
        next_flags = load_flags<T>(mask ? mask + t0 * a.m_t : nullptr, a.m_t, a.L - t0, p.lane);
    };
    fetch((int64_t)slice * T);
    if (SPLIT) cluster_started(p);
    int buf = 0;
    for (int64_t r0 = 0; r0 < a.L; r0 += round, buf ^= 1) {
        const int64_t t0 = r0 + (int64_t)slice * T;
        PairLoad<TT> cur[T];
#pragma unroll
        for (int i = 0; i < T; ++i) cur[i].p = next[i];
        const unsigned flags = next_flags;
        if (r0 + round < a.L) fetch(t0 + round);
        float c = carry;
        if (SPLIT) {
            float C[T], P[T];
            float lc = 0.0f, lp = 1.0f;
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const bool pad = (flags >> i) & 1u;
                float f, keep;
                gate(cur[i].g(), nb, &f, &keep);
                const float n = fmaf(f, lc, keep * cur[i].x());
                lc = pad ? lc : n;
                lp = pad ? lp : lp * f;
                C[i] = lc;
                P[i] = lp;
            }
            c = exchange(x[0], buf, p, lp, lc, false, &carry);
            if (a.states && p.on && t0 < a.L) a.states[(t0 / kT) * a.B * a.d + p.col] = c;
            if (p.on) {
#pragma unroll
                for (int i = 0; i < T; ++i)
                    if (t0 + i < a.L) h[(t0 + i) * a.h_t] = Cvt<TT>::from_f((flags >> i) & 1u ? 0.0f : fmaf(P[i], c, C[i]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < T; ++i) {
                if (i % kT == 0 && a.states && p.on && t0 + i < a.L) a.states[((t0 + i) / kT) * a.B * a.d + p.col] = c;
                const bool pad = (flags >> i) & 1u;
                float f, keep;
                gate(cur[i].g(), nb, &f, &keep);
                const float n = fmaf(f, c, keep * cur[i].x());
                c = pad ? c : n;
                if (p.on && t0 + i < a.L) h[(t0 + i) * a.h_t] = Cvt<TT>::from_f(pad ? 0.0f : n);
            }
            carry = c;
        }
    }
    if (slice == 0 && p.on && a.last) a.last[p.col] = carry;
}

template <typename TT, bool SPLIT>
__global__ void __launch_bounds__(SPLIT ? 256 : 64, SPLIT ? 2 : 8)
linear_recurrence_bwd_kernel(const LinRecArgs a) {
    __shared__ Exchange x[1];
    constexpr int T = kT;
    Place p;
    if (!find_place<SPLIT>(a, &p)) return;
    const TT *u = static_cast<const TT *>(a.u) + p.b * a.u_b + 2 * p.j;
    const TT *gh = a.grad_h ? static_cast<const TT *>(a.grad_h) + p.b * a.gh_b + p.j : nullptr;
    TT *gu = static_cast<TT *>(a.h) + 2 * p.col;
    const uint8_t *mask = a.mask ? a.mask + p.b : nullptr;
    const float nb = (p.on && a.bias) ? a.bias[p.j] * kNegLog2e : 0.0f;
    float carry = (p.on && a.first) ? a.first[p.col] : 0.0f, db = 0.0f;
    const int slices = SPLIT ? p.warps * (int)p.ranks : 1;
    const int slice = SPLIT ? (int)p.rank * p.warps + p.warp : 0;
    const int64_t round = (int64_t)slices * T;
    Pack<TT, 2> next_u[T];
    Pack<TT, 1> next_g[T];
    float next_c = 0.0f;
    unsigned next_flags;
    auto fetch = [&](int64_t t0) {
        if (p.on && t0 < a.L) next_c = a.states[(t0 / T) * a.B * a.d + p.col];
        load_steps<TT, 2, T>(next_u, u + t0 * a.u_t, a.u_t, a.L - t0, p.on);
        load_steps<TT, 1, T>(next_g, gh + t0 * a.gh_t, a.gh_t, a.L - t0, p.on && gh);
        next_flags = load_flags<T>(mask ? mask + t0 * a.m_t : nullptr, a.m_t, a.L - t0, p.lane);
    };
    const int64_t r_top = (a.L - 1) / round * round;
    fetch(r_top + (int64_t)slice * T);
    if (SPLIT) cluster_started(p);
    int buf = 0;
    for (int64_t r0 = r_top; r0 >= 0; r0 -= round, buf ^= 1) {
        const int64_t t0 = r0 + (int64_t)slice * T;
        float f[T], keep[T], w[T];      // w = (c_{t-1} - x) f (1 - f)
        Pack<TT, 1> g[T];
        const unsigned flags = next_flags;
        {
            PairLoad<TT> cur[T];
            float c = next_c;
#pragma unroll
            for (int i = 0; i < T; ++i) { cur[i].p = next_u[i]; g[i] = next_g[i]; }
            if (r0 > 0) fetch(t0 - round);
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const bool pad = (flags >> i) & 1u;
                const float xi = cur[i].x();
                float fi, ki;
                gate(cur[i].g(), nb, &fi, &ki);
                w[i] = pad ? 0.0f : (c - xi) * fi * ki;
                c = pad ? c : fmaf(fi, c, ki * xi);
                f[i] = pad ? 1.0f : fi;
                keep[i] = pad ? 0.0f : ki;
            }
        }
        float dc = carry;
        if (SPLIT) {
            float lc = 0.0f, lp = 1.0f;
#pragma unroll
            for (int i = T - 1; i >= 0; --i) {
                lc = f[i] * ((flags >> i) & 1u ? lc : lc + Cvt<TT>::to_f(g[i].v[0]));
                lp *= f[i];
            }
            dc = exchange(x[0], buf, p, lp, lc, true, &carry);
        }
#pragma unroll
        for (int i = T - 1; i >= 0; --i) {
            const bool pad = (flags >> i) & 1u;
            const float total = pad ? dc : dc + Cvt<TT>::to_f(g[i].v[0]);
            const float dg = pad ? 0.0f : w[i] * total;
            Pack<TT, 2> out;
            out.v[0] = Cvt<TT>::from_f(pad ? 0.0f : keep[i] * total);
            out.v[1] = Cvt<TT>::from_f(dg);
            db += dg;
            dc = f[i] * total;
            if (p.on && t0 + i < a.L) *reinterpret_cast<Pack<TT, 2> *>(gu + 2 * (t0 + i) * a.h_t) = out;
        }
        if (!SPLIT) carry = dc;
    }
    if (p.on) {
        if (a.last && slice == 0) a.last[p.col] = carry;
        if (a.bias_part) a.bias_part[(p.b * slices + slice) * a.d + p.j] = db;
    }
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

Slices choose_slices(int64_t L, int64_t B, int64_t d) {
    const int64_t columns = (d + 31) / 32 * B;              // warps that one walk over time takes
    int64_t want = option(OPT_LINREC_SLICES, 0);
    if (want <= 0) {
        want = 1;
        while (want < 64 && columns * want * 2 <= 148 * 24) want *= 2;
    }
    want = std::min<int64_t>(std::min<int64_t>(want, 64), (L + kT - 1) / kT);
    Slices s;
    s.ranks = (int)((want + kMaxWarps - 1) / kMaxWarps);
    s.warps = (int)((want + s.ranks - 1) / s.ranks);
    return s;
}

template <typename TT> int launch(const LinRecArgs &a0, const Slices &s, bool backward, cudaStream_t st) {
    LinRecArgs a = a0;
    a.groups = (a.d + 31) / 32;
    const int64_t columns = (int64_t)a.groups * a.B;
    if (columns * s.ranks > 0x7fffffff) return set_error(SRU_ERR_UNSUPPORTED, "linear recurrence: batch * hidden too large");
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s.ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    if (s.count() > 1) {
        cfg.gridDim = dim3((unsigned)(columns * s.ranks), 1, 1);
        cfg.blockDim = dim3(32 * s.warps, 1, 1);
        cfg.numAttrs = 1;
        if (backward) SRUB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, linear_recurrence_bwd_kernel<TT, true>, a));
        else SRUB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, linear_recurrence_fwd_kernel<TT, kT, true>, a));
    } else {
        cfg.gridDim = dim3((unsigned)((columns + 1) / 2), 1, 1);
        cfg.blockDim = dim3(64, 1, 1);
        if (backward) SRUB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, linear_recurrence_bwd_kernel<TT, false>, a));
        else SRUB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, linear_recurrence_fwd_kernel<TT, 2 * kT, false>, a));
    }
    return 0;
}

int dispatch(const LinRecArgs &a, const Slices &s, int dtype, bool backward, cudaStream_t st) {
    switch (dtype) {
        case SRU_F16: return launch<__half>(a, s, backward, st);
        case SRU_BF16: return launch<__nv_bfloat16>(a, s, backward, st);
        default: return launch<float>(a, s, backward, st);
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
    LinRecArgs a;
    memset(&a, 0, sizeof(a));
    a.h = h; a.last = c_last; a.states = static_cast<float *>(states);
    a.u = u; a.bias = bias; a.first = c_init; a.mask = mask_pad;
    a.L = length; a.B = batch; a.d = (int)hidden;
    a.u_t = u_stride_t; a.u_b = u_stride_b;
    a.h_t = batch * hidden; a.m_t = batch;
    if (reverse) reverse_time(&a, size, 1);
    return dispatch(a, choose_slices(length, batch, hidden), dtype, false, static_cast<cudaStream_t>(stream));
}

size_t sru_b200_linear_recurrence_backward_workspace_bytes(int64_t length, int64_t batch, int64_t hidden) {
    if (length < 1 || batch < 1 || hidden < 1) return 0;
    return (size_t)batch * choose_slices(length, batch, hidden).count() * (size_t)hidden * sizeof(float);
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
    const Slices s = choose_slices(length, batch, hidden);
    if (grad_bias) {
        const size_t need = (size_t)batch * s.count() * (size_t)hidden * sizeof(float);
        if (!workspace || workspace_bytes < need)
            return set_error(SRU_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    }
    LinRecArgs a;
    memset(&a, 0, sizeof(a));
    a.h = grad_u; a.last = grad_init; a.states = const_cast<float *>(static_cast<const float *>(states));
    a.bias_part = grad_bias ? static_cast<float *>(workspace) : nullptr;
    a.u = u; a.bias = bias; a.first = grad_last; a.grad_h = grad_h; a.mask = mask_pad;
    a.L = length; a.B = batch; a.d = (int)hidden;
    a.u_t = u_stride_t; a.u_b = u_stride_b; a.gh_t = gh_stride_t; a.gh_b = gh_stride_b;
    a.h_t = batch * hidden; a.m_t = batch;
    if (reverse) reverse_time(&a, size, 2);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rc = dispatch(a, s, dtype, true, st);
    if (rc || !grad_bias) return rc;
    linear_recurrence_bias_kernel<<<(unsigned)((hidden + 31) / 32), 256, 0, st>>>(grad_bias, a.bias_part,
                                                                                   batch * s.count(), (int)hidden);
    SRUB_CUDA_CHECK(cudaGetLastError());
    return 0;
}

}  // extern "C"
