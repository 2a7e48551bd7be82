/*
 * Gated linear recurrence (kmamba_b200.h): forward, backward, one step.
 *
 *   u = rate sigmoid(gate_r), rate = scale softplus(decay); a = e^-u
 *   b = sqrt(1 - a^2) sigmoid(gate_i) x;  h_t = a_t h_{t-1} + b_t
 *
 * Adjoint, with G_t = dy_t + a_{t+1} G_{t+1}:
 *   dx = G sqrt(1 - a^2) i,  dgate_i = G b (1 - i)
 *   u dL/du = G (kappa b - u a h_{t-1}),  kappa = u a^2 / (1 - a^2)
 *   dgate_r = u dL/du (1 - r),  ddecay = sigmoid(decay) / softplus(decay)
 *   sum_t u dL/du
 * (dL/du goes through a and through the root; u times the root's share is
 * kappa b, so nothing divides by a vanishing root: kappa -> 1/2 at u = 0.)
 *
 * One thread per (sequence, channel) walks the rows in order.
 */
#include <cuda_bf16.h>

#include "kmb_common.cuh"
#include "../kmb_internal.h"

namespace {

constexpr int kThreads = 128;
constexpr int kChunk = KMB_GLR_CHUNK;

__device__ __forceinline__ float ld(const float *p) { return *p; }
__device__ __forceinline__ float ld(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st(float *p, float v) { *p = v; }
__device__ __forceinline__ void st(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + expf(-v)); }
__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v + expf(-v) : log1pf(expf(v)); }
/* sigmoid / softplus: 1 where both vanish */
__device__ __forceinline__ float decay_ratio(float v) {
    return v < -15.f ? 1.f : sigmoid(v) / softplus(v);
}

struct Gates {
    float r, i, u, a, root, b;
};

__device__ __forceinline__ Gates gates(float x, float gr, float gi, float rate) {
    Gates g;
    g.r = sigmoid(gr);
    g.i = sigmoid(gi);
    g.u = rate * g.r;
    g.a = expf(-g.u);
    g.root = sqrtf(-expm1f(-2.f * g.u));
    g.b = g.root * g.i * x;
    return g;
}

/* rows [lo, hi) of a sequence, clamped into the tensors */
__device__ __forceinline__ void bounds(const KmbGLR &a, long b, long &lo, long &hi) {
    if (!a.offsets) {
        lo = 0;
        hi = a.L;
        return;
    }
    lo = a.offsets[b];
    hi = a.offsets[b + 1];
    lo = lo < 0 ? 0 : lo;
    hi = hi > a.L ? a.L : hi;
}

template <typename T>
__device__ __forceinline__ T *at(const KmbGLR &a, const KmbRows &r, long b, long t, long d) {
    return (T *)r.data + (a.offsets ? 0 : b * r.batch_stride) + t * r.row_stride + d;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_glr_fwd(KmbGLR a, float *ckpt, int write_y) {
    const long d = (long)blockIdx.x * kThreads + threadIdx.x, b = blockIdx.y;
    if (d >= a.D) return;
    const float rate = a.scale * softplus(a.decay[d]);
    long lo, hi;
    bounds(a, b, lo, hi);
    float h = a.h0 ? a.h0[b * a.D + d] : 0.f;
    const long chunks = (a.L + kChunk - 1) / kChunk;
    for (long t = lo; t < hi; ++t) {
        if (ckpt && t % kChunk == 0) ckpt[((a.offsets ? 0 : b * chunks) + t / kChunk) * a.D + d] = h;
        const Gates g = gates(ld(at<T>(a, a.x, b, t, d)), ld(at<T>(a, a.gate_r, b, t, d)),
                              ld(at<T>(a, a.gate_i, b, t, d)), rate);
        h = fmaf(g.a, h, g.b);
        if (write_y) st(at<T>(a, a.y, b, t, d), h);
    }
    if (write_y && a.h_last) a.h_last[b * a.D + d] = h;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_glr_bwd(KmbGLR a, const float *ckpt, float *part) {
    const long d = (long)blockIdx.x * kThreads + threadIdx.x, b = blockIdx.y;
    if (d >= a.D) return;
    const float rate = a.scale * softplus(a.decay[d]);
    long lo, hi;
    bounds(a, b, lo, hi);
    const float first = a.h0 ? a.h0[b * a.D + d] : 0.f;
    float carry = a.dh_last ? a.dh_last[b * a.D + d] : 0.f, sum = 0.f;
    const long chunks = (a.L + kChunk - 1) / kChunk;
    float hp[kChunk]; /* the state before each row of the chunk */
    for (long c = lo < hi ? (hi - 1) / kChunk : -1; c >= 0 && c * kChunk + kChunk > lo; --c) {
        const long t0 = c * kChunk > lo ? c * kChunk : lo;
        const long t1 = c * kChunk + kChunk < hi ? c * kChunk + kChunk : hi;
        float h = t0 == lo ? first : ckpt[((a.offsets ? 0 : b * chunks) + c) * a.D + d];
        for (long t = t0; t < t1; ++t) {
            hp[t - c * kChunk] = h;
            const Gates g = gates(ld(at<T>(a, a.x, b, t, d)), ld(at<T>(a, a.gate_r, b, t, d)),
                                  ld(at<T>(a, a.gate_i, b, t, d)), rate);
            h = fmaf(g.a, h, g.b);
        }
        for (long t = t1 - 1; t >= t0; --t) {
            const Gates g = gates(ld(at<T>(a, a.x, b, t, d)), ld(at<T>(a, a.gate_r, b, t, d)),
                                  ld(at<T>(a, a.gate_i, b, t, d)), rate);
            const float G = ld(at<T>(a, a.dy, b, t, d)) + carry;
            const float one = -expm1f(-2.f * g.u);
            const float kappa = g.u > 0.f ? g.u * g.a * g.a / one : 0.5f;
            const float udu = G * (kappa * g.b - g.u * g.a * hp[t - c * kChunk]);
            carry = g.a * G;
            sum += udu;
            st(at<T>(a, a.dx, b, t, d), G * g.root * g.i);
            st(at<T>(a, a.dgate_r, b, t, d), udu * (1.f - g.r));
            st(at<T>(a, a.dgate_i, b, t, d), G * g.b * (1.f - g.i));
        }
    }
    if (a.dh0) a.dh0[b * a.D + d] = carry;
    if (part) part[b * a.D + d] = sum;
}

__global__ void k_glr_ddecay(const float *part, long parts, long D, const float *decay, float *ddecay,
                             int acc) {
    const long d = (long)blockIdx.x * kThreads + threadIdx.x;
    if (d >= D) return;
    float s = 0.f;
    for (long p = 0; p < parts; ++p) s += part[p * D + d];
    s *= decay_ratio(decay[d]);
    ddecay[d] = acc ? ddecay[d] + s : s;
}

/* a row whose slot an earlier row names is left out */
template <typename T>
__global__ void __launch_bounds__(kThreads) k_glr_step(KmbGLRStep a) {
    const long k = blockIdx.y;
    const long slot = a.slots ? a.slots[k] : k;
    if (slot < 0 || slot >= a.n_states) return;
    int taken = 0;
    if (a.slots)
        for (long j = threadIdx.x; j < k; j += kThreads) taken |= a.slots[j] == slot;
    if (__syncthreads_or(taken)) return;
    const long d = (long)blockIdx.x * kThreads + threadIdx.x;
    if (d >= a.D) return;
    const Gates g = gates(ld((const T *)a.x.data + k * a.x.row_stride + d),
                          ld((const T *)a.gate_r.data + k * a.gate_r.row_stride + d),
                          ld((const T *)a.gate_i.data + k * a.gate_i.row_stride + d),
                          a.scale * softplus(a.decay[d]));
    float *s = a.state + slot * a.ld_state + d;
    const float h = fmaf(g.a, *s, g.b);
    *s = h;
    st((T *)a.y.data + k * a.y.row_stride + d, h);
}

int done(const char *what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, what);
}

dim3 grid_of(long D, long n) { return dim3((unsigned)((D + kThreads - 1) / kThreads), (unsigned)n); }

template <typename T>
int bwd(const KmbGLR *a, cudaStream_t s) {
    float *ws = (float *)a->workspace;
    float *part = a->ddecay ? ws : nullptr;
    float *ckpt = a->ckpt;
    if (!ckpt) {
        ckpt = ws + (a->ddecay ? a->batch * a->D : 0);
        if (a->batch && a->L) k_glr_fwd<T><<<grid_of(a->D, a->batch), kThreads, 0, s>>>(*a, ckpt, 0);
    }
    if (a->batch) k_glr_bwd<T><<<grid_of(a->D, a->batch), kThreads, 0, s>>>(*a, ckpt, part);
    if (a->ddecay)
        k_glr_ddecay<<<grid_of(a->D, 1), kThreads, 0, s>>>(part, a->batch, a->D, a->decay, a->ddecay,
                                                           a->accumulate);
    return done("glr: backward launch");
}

} // namespace

extern "C" size_t kmb_glr_scratch_bytes(const KmbGLR *a, int bwd) {
    if (!bwd) return 0;
    return 4 * ((a->ddecay ? (size_t)a->batch * a->D : 0) + (a->ckpt ? 0 : (size_t)kmb_glr_ckpt_elems(a)));
}

extern "C" int kmb_launch_glr_fwd(const KmbGLR *a, cudaStream_t s) {
    if (!a->batch) return KMB_OK;
    const dim3 g = grid_of(a->D, a->batch);
    if (a->type == KMB_BF16)
        k_glr_fwd<__nv_bfloat16><<<g, kThreads, 0, s>>>(*a, a->ckpt, 1);
    else
        k_glr_fwd<float><<<g, kThreads, 0, s>>>(*a, a->ckpt, 1);
    return done("glr: forward launch");
}

extern "C" int kmb_launch_glr_bwd(const KmbGLR *a, cudaStream_t s) {
    return a->type == KMB_BF16 ? bwd<__nv_bfloat16>(a, s) : bwd<float>(a, s);
}

extern "C" int kmb_launch_glr_step(const KmbGLRStep *a, cudaStream_t s) {
    const dim3 g = grid_of(a->D, a->rows);
    if (a->type == KMB_BF16)
        k_glr_step<__nv_bfloat16><<<g, kThreads, 0, s>>>(*a);
    else
        k_glr_step<float><<<g, kThreads, 0, s>>>(*a);
    return done("glr: step launch");
}
