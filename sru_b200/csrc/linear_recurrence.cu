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

// One step's V pairs of u, as loaded.
template <typename TT, int V> struct PairLoad {
    Pack<TT, 2 * V> p;
    __device__ __forceinline__ float x(int v) const { return Cvt<TT>::to_f(p.v[2 * v]); }
    __device__ __forceinline__ float g(int v) const { return Cvt<TT>::to_f(p.v[2 * v + 1]); }
};

template <typename P> __device__ __forceinline__ P zero_pack() {
    P p;
    memset(&p, 0, sizeof(P));
    return p;
}

// kT steps of a strided stream of N elements per lane and step; steps from `n` on are left zero and not read.
template <typename TT, int N>
__device__ __forceinline__ void load_steps(Pack<TT, N> (&r)[kT], const TT *p, int64_t stride, int n, bool on) {
    if (on && n >= kT) {
#pragma unroll
        for (int i = 0; i < kT; ++i) r[i] = *reinterpret_cast<const Pack<TT, N> *>(p + i * stride);
    } else {
#pragma unroll
        for (int i = 0; i < kT; ++i)
            r[i] = (on && i < n) ? *reinterpret_cast<const Pack<TT, N> *>(p + i * stride) : zero_pack<Pack<TT, N>>();
    }
}

// Bit i: step i of the chunk is padded or lies behind the end.  The whole warp works on one sequence, so the flags are
// uniform; lane i fetches step i's byte.
__device__ __forceinline__ unsigned load_flags(const uint8_t *mask, int64_t stride, int64_t n, int lane) {
    bool pad = lane >= n;
    if (mask && lane < kT && lane < n) pad = mask[lane * stride] != 0;
    return __ballot_sync(0xffffffffu, pad) & ((1u << kT) - 1u);
}

// f and 1 - f from the gate's logit; nb = -bias * log2(e)
__device__ __forceinline__ void gate(float g, float nb, float *f, float *keep) {
    const float e = ex2_approx(min_nan(fmaf(g, kNegLog2e, nb), 126.0f));    // at most 2^126, so that e * f stays finite
    *f = rcp_approx(1.0f + e);
    *keep = e * *f;
}

template <typename TT, int V>
__global__ void __launch_bounds__(64)
linear_recurrence_fwd_kernel(const LinRecArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t wid = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t b = wid / a.groups;
    if (b >= a.B) return;
    const int j = (int)(wid - b * a.groups) * 32 * V + lane * V;
    const bool on = j < a.d;
    const int64_t col = b * a.d + j;
    const TT *u = static_cast<const TT *>(a.u) + b * a.u_b + 2 * j;
    TT *h = static_cast<TT *>(a.h) + col;
    const uint8_t *mask = a.mask ? a.mask + b : nullptr;
    float nb[V], c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        nb[v] = (on && a.bias) ? a.bias[j + v] * kNegLog2e : 0.0f;
        c[v] = (on && a.first) ? a.first[col + v] : 0.0f;
    }
    Pack<TT, 2 * V> next[kT];
    unsigned next_flags;
    auto fetch = [&](int64_t t0) {
        load_steps<TT, 2 * V>(next, u + t0 * a.u_t, a.u_t, (int)min((int64_t)kT, a.L - t0), on);
        next_flags = load_flags(mask ? mask + t0 * a.m_t : nullptr, a.m_t, a.L - t0, lane);
    };
    fetch(0);
    for (int64_t t0 = 0; t0 < a.L; t0 += kT) {
        PairLoad<TT, V> cur[kT];
#pragma unroll
        for (int i = 0; i < kT; ++i) cur[i].p = next[i];
        const unsigned flags = next_flags;
        if (t0 + kT < a.L) fetch(t0 + kT);
        if (a.states && on) {
            Pack<float, V> s;
#pragma unroll
            for (int v = 0; v < V; ++v) s.v[v] = c[v];
            *reinterpret_cast<Pack<float, V> *>(a.states + (t0 / kT) * a.B * a.d + col) = s;
        }
#pragma unroll
        for (int i = 0; i < kT; ++i) {
            const bool pad = (flags >> i) & 1u;
            Pack<TT, V> out;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float f, keep;
                gate(cur[i].g(v), nb[v], &f, &keep);
                const float n = fmaf(f, c[v], keep * cur[i].x(v));
                c[v] = pad ? c[v] : n;
                out.v[v] = Cvt<TT>::from_f(pad ? 0.0f : n);
            }
            if (on && t0 + i < a.L) *reinterpret_cast<Pack<TT, V> *>(h + (t0 + i) * a.h_t) = out;
        }
    }
    if (on && a.last) {
#pragma unroll
        for (int v = 0; v < V; ++v) a.last[col + v] = c[v];
    }
}

template <typename TT, int V>
__global__ void __launch_bounds__(64)
linear_recurrence_bwd_kernel(const LinRecArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t wid = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t b = wid / a.groups;
    if (b >= a.B) return;
    const int j = (int)(wid - b * a.groups) * 32 * V + lane * V;
    const bool on = j < a.d;
    const int64_t col = b * a.d + j;
    const TT *u = static_cast<const TT *>(a.u) + b * a.u_b + 2 * j;
    const TT *gh = a.grad_h ? static_cast<const TT *>(a.grad_h) + b * a.gh_b + j : nullptr;
    TT *gu = static_cast<TT *>(a.h) + 2 * col;
    const uint8_t *mask = a.mask ? a.mask + b : nullptr;
    float nb[V], dc[V], db[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        nb[v] = (on && a.bias) ? a.bias[j + v] * kNegLog2e : 0.0f;
        dc[v] = (on && a.first) ? a.first[col + v] : 0.0f;
        db[v] = 0.0f;
    }
    Pack<TT, 2 * V> next_u[kT];
    Pack<TT, V> next_g[kT];
    Pack<float, V> next_c = zero_pack<Pack<float, V>>();
    unsigned next_flags;
    auto fetch = [&](int64_t t0) {
        const int n = (int)min((int64_t)kT, a.L - t0);
        if (on) next_c = *reinterpret_cast<const Pack<float, V> *>(a.states + (t0 / kT) * a.B * a.d + col);
        load_steps<TT, 2 * V>(next_u, u + t0 * a.u_t, a.u_t, n, on);
        load_steps<TT, V>(next_g, gh + t0 * a.gh_t, a.gh_t, n, on && gh);
        next_flags = load_flags(mask ? mask + t0 * a.m_t : nullptr, a.m_t, a.L - t0, lane);
    };
    const int64_t t_top = (a.L - 1) / kT * kT;
    fetch(t_top);
    for (int64_t t0 = t_top; t0 >= 0; t0 -= kT) {
        float f[kT][V], keep[kT][V], w[kT][V];      // w = (c_{t-1} - x) f (1 - f)
        Pack<TT, V> g[kT];
        const unsigned flags = next_flags;
        {
            PairLoad<TT, V> cur[kT];
            Pack<float, V> c = next_c;
#pragma unroll
            for (int i = 0; i < kT; ++i) { cur[i].p = next_u[i]; g[i] = next_g[i]; }
            if (t0 > 0) fetch(t0 - kT);
#pragma unroll
            for (int i = 0; i < kT; ++i) {
                const bool pad = (flags >> i) & 1u;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float x = cur[i].x(v);
                    float fi, ki;
                    gate(cur[i].g(v), nb[v], &fi, &ki);
                    w[i][v] = pad ? 0.0f : (c.v[v] - x) * fi * ki;
                    c.v[v] = pad ? c.v[v] : fmaf(fi, c.v[v], ki * x);
                    f[i][v] = pad ? 1.0f : fi;
                    keep[i][v] = pad ? 0.0f : ki;
                }
            }
        }
#pragma unroll
        for (int i = kT - 1; i >= 0; --i) {
            const bool pad = (flags >> i) & 1u;
            Pack<TT, 2 * V> out;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float total = pad ? dc[v] : dc[v] + Cvt<TT>::to_f(g[i].v[v]);
                const float dg = pad ? 0.0f : w[i][v] * total;
                out.v[2 * v] = Cvt<TT>::from_f(pad ? 0.0f : keep[i][v] * total);
                out.v[2 * v + 1] = Cvt<TT>::from_f(dg);
                db[v] += dg;
                dc[v] = f[i][v] * total;
            }
            if (on && t0 + i < a.L) *reinterpret_cast<Pack<TT, 2 * V> *>(gu + 2 * (t0 + i) * a.h_t) = out;
        }
    }
    if (on) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (a.last) a.last[col + v] = dc[v];
            if (a.bias_part) a.bias_part[b * a.d + j + v] = db[v];
        }
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

template <typename TT> int launch(const LinRecArgs &a0, bool backward, cudaStream_t st) {
    LinRecArgs a = a0;
    constexpr int V = 1;
    a.groups = (a.d + 32 * V - 1) / (32 * V);
    const int64_t warps = (int64_t)a.groups * a.B;
    const int64_t blocks = (warps + 1) / 2;
    if (blocks > 0x7fffffff) return set_error(SRU_ERR_UNSUPPORTED, "linear recurrence: batch * hidden too large");
    if (backward) linear_recurrence_bwd_kernel<TT, V><<<(unsigned)blocks, 64, 0, st>>>(a);
    else linear_recurrence_fwd_kernel<TT, V><<<(unsigned)blocks, 64, 0, st>>>(a);
    SRUB_CUDA_CHECK(cudaGetLastError());
    return 0;
}

int dispatch(const LinRecArgs &a, int dtype, bool backward, cudaStream_t st) {
    switch (dtype) {
        case SRU_F16: return launch<__half>(a, backward, st);
        case SRU_BF16: return launch<__nv_bfloat16>(a, backward, st);
        default: return launch<float>(a, backward, st);
    }
}

int64_t bias_parts(int64_t B) { return B; }

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
    return dispatch(a, dtype, false, static_cast<cudaStream_t>(stream));
}

size_t sru_b200_linear_recurrence_backward_workspace_bytes(int64_t length, int64_t batch, int64_t hidden) {
    if (length < 1 || batch < 1 || hidden < 1) return 0;
    return (size_t)bias_parts(batch) * (size_t)hidden * sizeof(float);
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
    if (grad_bias) {
        const size_t need = sru_b200_linear_recurrence_backward_workspace_bytes(length, batch, hidden);
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
    rc = dispatch(a, dtype, true, st);
    if (rc || !grad_bias) return rc;
    linear_recurrence_bias_kernel<<<(unsigned)((hidden + 31) / 32), 256, 0, st>>>(grad_bias, a.bias_part,
                                                                                   bias_parts(batch), (int)hidden);
    SRUB_CUDA_CHECK(cudaGetLastError());
    return 0;
}

}  // extern "C"
