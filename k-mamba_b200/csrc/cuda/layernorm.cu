/*
 * Layer norm, forward and backward (kmamba_b200.h).
 *
 * Per row of D values: mean = sum x / D, rstd = (sum (x - mean)^2 / D +
 * eps)^-1/2, y = (x - mean) rstd w + b.  With xhat = (x - mean) rstd and g =
 * dy w the adjoint is dx = rstd (g - avg g - xhat avg(g xhat)); the weight's
 * and bias' gradients are the column sums of dy xhat and dy.
 *
 * Memory bounds both: every tensor is to be read or written once.  A row
 * stays in the registers of a warp (D <= 256) or a CTA from its load to the
 * store, 8 values a thread, so the mean and the centred squares are two
 * passes over registers.  CTAs are resident for the whole call and walk the
 * rows: weight and bias are loaded once, the next row's loads are in flight
 * while a row is reduced, and in the backward every thread keeps the column
 * sums of its own 8 columns, written once at the end as one row of partial
 * sums a CTA, which a second kernel adds in a fixed order.
 */
#include <cuda_bf16.h>

#include "kmb_common.cuh"
#include "../kmb_internal.h"

namespace {

constexpr int kSMs = 148;
constexpr int kEpt = 8;        /* values of a thread */
constexpr int kGroup = 256;    /* widest row of a single warp */
constexpr int kGroups = 8;     /* such rows of a CTA */
constexpr int kSmall = 256;    /* threads up to which a thread has 80 registers, not 64 */
constexpr int kMaxD = 1024 * kEpt;
constexpr int kWideEpt = 32;   /* forward: values of a thread for wider rows */
constexpr int kWideD = 1024 * kWideEpt;
constexpr int kLoop = 512;     /* threads for rows that do not stay in registers */

__device__ __forceinline__ float ld(const float *p) { return *p; }
__device__ __forceinline__ float ld(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st(float *p, float v) { *p = v; }
__device__ __forceinline__ void st(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

/* V values in one access (V = 1: any alignment), kept as loaded. */
template <typename T, int V>
struct Vec;
template <>
struct Vec<float, 1> {
    float v;
    __device__ __forceinline__ void load(const float *p) { v = __ldcs(p); }
    __device__ __forceinline__ void get(float *f) const { f[0] = v; }
    static __device__ __forceinline__ void store(float *p, const float *f) { __stcs(p, f[0]); }
};
template <>
struct Vec<float, 4> {
    float4 v;
    __device__ __forceinline__ void load(const float *p) { v = __ldcs(reinterpret_cast<const float4 *>(p)); }
    __device__ __forceinline__ void get(float *f) const {
        f[0] = v.x;
        f[1] = v.y;
        f[2] = v.z;
        f[3] = v.w;
    }
    static __device__ __forceinline__ void store(float *p, const float *f) {
        __stcs(reinterpret_cast<float4 *>(p), make_float4(f[0], f[1], f[2], f[3]));
    }
};
__device__ __forceinline__ unsigned pack2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&h);
}
__device__ __forceinline__ void unpack2(unsigned u, float *f) {
    f[0] = __uint_as_float(u << 16);
    f[1] = __uint_as_float(u & 0xffff0000u);
}
template <>
struct Vec<__nv_bfloat16, 1> {
    unsigned short v;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
        v = __ldcs(reinterpret_cast<const unsigned short *>(p));
    }
    __device__ __forceinline__ void get(float *f) const { f[0] = __uint_as_float((unsigned)v << 16); }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *f) {
        __stcs(reinterpret_cast<unsigned short *>(p), (unsigned short)pack2(f[0], 0.f));
    }
};
template <>
struct Vec<__nv_bfloat16, 4> {
    uint2 v;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { v = __ldcs(reinterpret_cast<const uint2 *>(p)); }
    __device__ __forceinline__ void get(float *f) const {
        unpack2(v.x, f);
        unpack2(v.y, f + 2);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *f) {
        __stcs(reinterpret_cast<uint2 *>(p), make_uint2(pack2(f[0], f[1]), pack2(f[2], f[3])));
    }
};
template <>
struct Vec<__nv_bfloat16, 8> {
    uint4 v;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { v = __ldcs(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void get(float *f) const {
        unpack2(v.x, f);
        unpack2(v.y, f + 2);
        unpack2(v.z, f + 4);
        unpack2(v.w, f + 6);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *f) {
        __stcs(reinterpret_cast<uint4 *>(p), make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]),
                                                       pack2(f[4], f[5]), pack2(f[6], f[7])));
    }
};

/* Sums over the threads of a row: a warp, or with more than one warp a row
 * the whole CTA, through two slots in turn, so that one barrier a sum does. */
struct Reducer {
    float2 (*slot)[32];
    int warps; /* of a row */
    int turn;
    __device__ __forceinline__ Reducer(float2 (*s)[32], int w) : slot(s), warps(w), turn(0) {}
    __device__ __forceinline__ float2 two(float a, float b) {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            a += __shfl_xor_sync(~0u, a, o);
            b += __shfl_xor_sync(~0u, b, o);
        }
        if (warps == 1) return make_float2(a, b);
        const int lane = threadIdx.x % 32;
        if (lane == 0) slot[turn][threadIdx.x / 32] = make_float2(a, b);
        __syncthreads();
        float2 v = lane < warps ? slot[turn][lane] : make_float2(0.f, 0.f);
        turn ^= 1;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            v.x += __shfl_xor_sync(~0u, v.x, o);
            v.y += __shfl_xor_sync(~0u, v.y, o);
        }
        return v;
    }
    __device__ __forceinline__ float one(float a) { return two(a, 0.f).x; }
};

/* Sums of rows whose plain fp32 sums overflow are taken again on scaled
 * values: 2^-32 x for the mean (D < 2^31), 2^-80 (x - mean) for the squares.
 * A row with an infinity or a NaN stays what it is. */
constexpr float kDown = 0x1p-32f, kUp = 0x1p32f, kSqDown = 0x1p-80f;

/* each(f) calls f(value) for the thread's values of the row */
template <typename Each>
__device__ __forceinline__ void row_stats(Each each, Reducer &red, float n, float eps, float &mean,
                                          float &rstd) {
    float s = 0.f;
    each([&](float x) { s += x; });
    mean = red.one(s) / n;
    if (!isfinite(mean)) {
        s = 0.f;
        each([&](float x) { s = fmaf(x, kDown, s); });
        mean = red.one(s) / n * kUp;
    }
    s = 0.f;
    each([&](float x) { s = fmaf(x - mean, x - mean, s); });
    s = red.one(s);
    rstd = 1.f / sqrtf(s / n + eps);
    if (!isfinite(s)) {
        s = 0.f;
        each([&](float x) { s = fmaf((x - mean) * kSqDown, (x - mean) * kSqDown, s); });
        rstd = kSqDown / sqrtf(red.one(s) / n + eps * kSqDown * kSqDown);
    }
}

/* The thread's columns: vector k begins at col(k); all of a vector's
 * columns exist or none. */
template <int V>
struct Cols {
    int t, tpr, D;
    __device__ __forceinline__ int col(int k) const { return (t + k * tpr) * V; }
    __device__ __forceinline__ bool in(int k) const { return col(k) < D; }
};

template <int V, int NV>
__device__ __forceinline__ void load_cols(const Cols<V> &c, const float *p, float none, float *out) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) out[k * V + e] = p && c.in(k) ? p[c.col(k) + e] : none;
}

/* ------------------------------------------------------------------ */
/* forward                                                              */
/* ------------------------------------------------------------------ */

template <typename TX, typename TY, int V, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == kSmall ? 3 : 1) k_ln_fwd(const __grid_constant__ KmbLayerNorm a, int wpr) {
    __shared__ float2 slot[2][32];
    constexpr bool kKeep = V * NV <= kEpt; /* weight and bias in registers, next row ahead */
    const bool single = wpr == 1;
    const int groups = single ? (int)blockDim.x / 32 : 1;
    const Cols<V> c = {single ? (int)threadIdx.x % 32 : (int)threadIdx.x, wpr * 32, (int)a.D};
    Reducer red(slot, wpr);
    const long step = (long)gridDim.x * groups;
    long r = (long)blockIdx.x * groups + (single ? threadIdx.x / 32 : 0);
    const float n = (float)a.D;
    float w[kKeep ? V * NV : 1], b[kKeep ? V * NV : 1];
    if (kKeep) {
        load_cols<V, kKeep ? NV : 0>(c, a.weight, 1.f, w);
        load_cols<V, kKeep ? NV : 0>(c, a.bias, 0.f, b);
    }
    Vec<TX, V> raw[NV];
    const auto fetch = [&](long row) {
        const TX *x = (const TX *)a.x + row * a.ld_x;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (c.in(k)) raw[k].load(x + c.col(k));
    };
    if (r < a.rows) fetch(r);
    for (; r < a.rows; r += step) {
        float x[V * NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) raw[k].get(x + k * V);
        if (kKeep && r + step < a.rows) fetch(r + step);
        float mean, rstd;
        row_stats(
            [&](auto f) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
                    if (c.in(k))
#pragma unroll
                        for (int e = 0; e < V; ++e) f(x[k * V + e]);
            },
            red, n, a.eps, mean, rstd);
        TY *y = (TY *)a.y + r * a.ld_y;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (!c.in(k)) continue;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float wv = kKeep ? w[k * V + e] : a.weight ? a.weight[c.col(k) + e] : 1.f;
                const float bv = kKeep ? b[k * V + e] : a.bias ? a.bias[c.col(k) + e] : 0.f;
                o[e] = fmaf((x[k * V + e] - mean) * rstd, wv, bv);
            }
            Vec<TY, V>::store(y + c.col(k), o);
        }
        if (c.t == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
        if (!kKeep && r + step < a.rows) fetch(r + step);
    }
}

/* rows wider than a CTA's registers: read again for each pass, from L2 */
template <typename TX, typename TY>
__global__ void __launch_bounds__(kLoop) k_ln_fwd_loop(const __grid_constant__ KmbLayerNorm a) {
    __shared__ float2 slot[2][32];
    Reducer red(slot, kLoop / 32);
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const TX *x = (const TX *)a.x + r * a.ld_x;
        TY *y = (TY *)a.y + r * a.ld_y;
        float mean, rstd;
        row_stats(
            [&](auto f) {
                for (long j = threadIdx.x; j < a.D; j += kLoop) f(ld(x + j));
            },
            red, (float)a.D, a.eps, mean, rstd);
        for (long j = threadIdx.x; j < a.D; j += kLoop)
            st(y + j, fmaf((ld(x + j) - mean) * rstd, a.weight ? a.weight[j] : 1.f, a.bias ? a.bias[j] : 0.f));
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

/* ------------------------------------------------------------------ */
/* backward                                                             */
/* ------------------------------------------------------------------ */

template <typename TX, typename TY, int V, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == kSmall ? 3 : 1) k_ln_bwd(const __grid_constant__ KmbLayerNorm a, int wpr, int sums) {
    static_assert(V * NV == kEpt, "8 values a thread");
    __shared__ float2 slot[2][32];
    __shared__ float fold[kGroups][kGroup];
    const bool single = wpr == 1;
    const int groups = single ? (int)blockDim.x / 32 : 1, warp = threadIdx.x / 32;
    const Cols<V> c = {single ? (int)threadIdx.x % 32 : (int)threadIdx.x, wpr * 32, (int)a.D};
    Reducer red(slot, wpr);
    const long step = (long)gridDim.x * groups;
    long r = (long)blockIdx.x * groups + (single ? warp : 0);
    const float n = (float)a.D, inv = 1.f / n;
    float w[kEpt], pw[kEpt], pb[kEpt];
    load_cols<V, NV>(c, a.weight, 1.f, w);
#pragma unroll
    for (int e = 0; e < kEpt; ++e) pw[e] = pb[e] = 0.f;
    Vec<TX, V> rx[NV];
    Vec<TY, V> rd[NV];
    float mean = 0.f, rstd = 0.f;
    const auto fetch = [&](long row) {
        const TX *x = (const TX *)a.x + row * a.ld_x;
        const TY *dy = (const TY *)a.dy + row * a.ld_dy;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (c.in(k)) {
                rx[k].load(x + c.col(k));
                rd[k].load(dy + c.col(k));
            }
        if (a.mean) {
            mean = a.mean[row];
            rstd = a.rstd[row];
        }
    };
    if (r < a.rows) fetch(r);
    for (; r < a.rows; r += step) {
        float h[kEpt], d[kEpt];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            rx[k].get(h + k * V);
            rd[k].get(d + k * V);
        }
        float m = mean, s = rstd;
        if (r + step < a.rows) fetch(r + step);
        Vec<TX, V> res[NV];
        if (a.dres) {
            const TX *p = (const TX *)a.dres + r * a.ld_dres;
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (c.in(k)) res[k].load(p + c.col(k));
        }
        if (!a.mean)
            row_stats(
                [&](auto f) {
#pragma unroll
                    for (int k = 0; k < NV; ++k)
                        if (c.in(k))
#pragma unroll
                            for (int e = 0; e < V; ++e) f(h[k * V + e]);
                },
                red, n, a.eps, m, s);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (c.in(k))
#pragma unroll
                for (int e = k * V; e < k * V + V; ++e) {
                    h[e] = (h[e] - m) * s;
                    pw[e] = fmaf(d[e], h[e], pw[e]);
                    pb[e] += d[e];
                    d[e] *= w[e];
                    s1 += d[e];
                    s2 = fmaf(d[e], h[e], s2);
                }
        const float2 t = red.two(s1, s2);
        s1 = t.x * inv;
        s2 = t.y * inv;
        TX *dx = (TX *)a.dx + r * a.ld_dx;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (c.in(k)) {
                float o[V], q[V];
                if (a.dres) res[k].get(q);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    o[e] = s * (d[k * V + e] - s1 - h[k * V + e] * s2);
                    if (a.dres) o[e] += q[e];
                }
                Vec<TX, V>::store(dx + c.col(k), o);
            }
    }
    if (!sums) return;
    float *part = (float *)a.workspace + (long)blockIdx.x * 2 * a.D;
    if (!single) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (c.in(k))
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    part[c.col(k) + e] = pw[k * V + e];
                    part[a.D + c.col(k) + e] = pb[k * V + e];
                }
        return;
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (c.in(k))
#pragma unroll
                for (int e = 0; e < V; ++e) fold[warp][c.col(k) + e] = which ? pb[k * V + e] : pw[k * V + e];
        __syncthreads();
        for (int j = threadIdx.x; j < a.D; j += blockDim.x) {
            float v = 0.f;
            for (int g = 0; g < groups; ++g) v += fold[g][j];
            part[which * a.D + j] = v;
        }
    }
}

/* wider rows: read a second time for dx, from L2; the column sums in
 * shared memory, or beyond its size in the CTA's row of the workspace, each
 * column one thread's */
template <typename TX, typename TY>
__global__ void __launch_bounds__(kLoop) k_ln_bwd_loop(const __grid_constant__ KmbLayerNorm a, int sums,
                                                       int in_shared) {
    extern __shared__ float cols[];
    __shared__ float2 slot[2][32];
    Reducer red(slot, kLoop / 32);
    float *part = (float *)a.workspace + (long)blockIdx.x * 2 * a.D;
    float *pw = in_shared ? cols : part, *pb = pw + a.D;
    if (sums)
        for (long j = threadIdx.x; j < a.D; j += kLoop) pw[j] = pb[j] = 0.f;
    const float inv = 1.f / (float)a.D;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const TX *x = (const TX *)a.x + r * a.ld_x;
        const TY *dy = (const TY *)a.dy + r * a.ld_dy;
        const TX *res = a.dres ? (const TX *)a.dres + r * a.ld_dres : nullptr;
        TX *dx = (TX *)a.dx + r * a.ld_dx;
        float mean, rstd;
        if (a.mean) {
            mean = a.mean[r];
            rstd = a.rstd[r];
        } else {
            row_stats(
                [&](auto f) {
                    for (long j = threadIdx.x; j < a.D; j += kLoop) f(ld(x + j));
                },
                red, (float)a.D, a.eps, mean, rstd);
        }
        float s1 = 0.f, s2 = 0.f;
        for (long j = threadIdx.x; j < a.D; j += kLoop) {
            const float h = (ld(x + j) - mean) * rstd, v = ld(dy + j);
            const float g = a.weight ? v * a.weight[j] : v;
            s1 += g;
            s2 = fmaf(g, h, s2);
            if (sums) {
                pw[j] = fmaf(v, h, pw[j]);
                pb[j] += v;
            }
        }
        const float2 t = red.two(s1, s2);
        s1 = t.x * inv;
        s2 = t.y * inv;
        for (long j = threadIdx.x; j < a.D; j += kLoop) {
            const float h = (ld(x + j) - mean) * rstd, v = ld(dy + j);
            const float g = a.weight ? v * a.weight[j] : v;
            const float d = rstd * (g - s1 - h * s2);
            st(dx + j, res ? d + ld(res + j) : d);
        }
    }
    if (sums && in_shared)
        for (long j = threadIdx.x; j < 2 * a.D; j += kLoop) part[j] = cols[j]; /* its own columns */
}

/* dweight, dbias from the rows of partial sums: 32 columns a CTA, 32 rows
 * of threads, joined in a fixed order */
__global__ void __launch_bounds__(1024) k_ln_sums(const float *part, long parts, long D, float *dw, float *db,
                                                  int acc) {
    __shared__ float s[32][33];
    const int tx = threadIdx.x, ty = threadIdx.y;
    const long j = (long)blockIdx.x * 32 + tx;
    float v = 0.f;
    if (j < 2 * D)
        for (long p = ty; p < parts; p += 32) v += part[p * 2 * D + j];
    s[ty][tx] = v;
    __syncthreads();
    v = s[tx][ty]; /* column ty, rows over the lanes */
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    const long k = (long)blockIdx.x * 32 + ty;
    if (tx || k >= 2 * D) return;
    float *to = k < D ? dw : db;
    if (!to) return;
    to += k < D ? k : k - D;
    *to = acc ? *to + v : v;
}

/* ------------------------------------------------------------------ */
/* launches                                                             */
/* ------------------------------------------------------------------ */

int warps_of(long D, int ept) { return (int)((D + 32 * ept - 1) / (32 * ept)); }

/* CTAs of the resident kernels: as many as the registers let an SM hold, no
 * more than there are rows (or groups of rows) */
long ctas(long rows, long D, int ept) {
    const int wpr = warps_of(D, ept), threads = wpr == 1 ? 32 * kGroups : 32 * wpr;
    const long need = wpr == 1 ? (rows + kGroups - 1) / kGroups : rows;
    const long most = (long)kSMs * (threads <= kSmall ? 3 * kSmall / threads : 1024 / threads);
    return need < most ? (need > 0 ? need : 1) : most;
}

bool aligned(const void *p, long ld, int type, int v) {
    const size_t es = type == KMB_BF16 ? 2 : 4;
    return !p || ((size_t)p / es % v == 0 && ld % v == 0);
}

int done() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, "layernorm: launch");
}

template <typename TX, typename TY, int V, int NV>
void run_fwd(const KmbLayerNorm *a, cudaStream_t s) {
    const int wpr = warps_of(a->D, V * NV), threads = wpr == 1 ? 32 * kGroups : 32 * wpr;
    const unsigned n = (unsigned)ctas(a->rows, a->D, V * NV);
    if (V * NV == kEpt && threads <= kSmall)
        k_ln_fwd<TX, TY, V, NV, V * NV == kEpt ? kSmall : 1024><<<n, threads, 0, s>>>(*a, wpr);
    else
        k_ln_fwd<TX, TY, V, NV, 1024><<<n, threads, 0, s>>>(*a, wpr);
}

template <typename TX, typename TY>
int fwd(const KmbLayerNorm *a, cudaStream_t s) {
    constexpr int V = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
    const bool vec = a->D % V == 0 && aligned(a->x, a->ld_x, a->x_type, V) && aligned(a->y, a->ld_y, a->y_type, V);
    if (a->D <= kMaxD)
        vec ? run_fwd<TX, TY, V, kEpt / V>(a, s) : run_fwd<TX, TY, 1, kEpt>(a, s);
    else if (a->D <= kWideD && vec)
        run_fwd<TX, TY, V, kWideEpt / V>(a, s);
    else
        k_ln_fwd_loop<TX, TY><<<(unsigned)(a->rows < 4 * kSMs ? a->rows : 4 * kSMs), kLoop, 0, s>>>(*a);
    return done();
}

template <typename TX, typename TY, int V, int NV>
void run_bwd(const KmbLayerNorm *a, int sums, cudaStream_t s) {
    const int wpr = warps_of(a->D, V * NV), threads = wpr == 1 ? 32 * kGroups : 32 * wpr;
    const unsigned n = (unsigned)ctas(a->rows, a->D, V * NV);
    if (threads <= kSmall)
        k_ln_bwd<TX, TY, V, NV, kSmall><<<n, threads, 0, s>>>(*a, wpr, sums);
    else
        k_ln_bwd<TX, TY, V, NV, 1024><<<n, threads, 0, s>>>(*a, wpr, sums);
}

constexpr size_t kColsShared = 200 * 1024; /* of the 227 KB an SM can give a CTA */

template <typename TX, typename TY>
int bwd(const KmbLayerNorm *a, cudaStream_t s) {
    constexpr int V = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
    const int sums = a->dweight || a->dbias;
    const long parts = kmb_layernorm_parts(a->rows, a->D);
    const bool vec = a->D % V == 0 && aligned(a->x, a->ld_x, a->x_type, V) &&
                     aligned(a->dy, a->ld_dy, a->y_type, V) && aligned(a->dx, a->ld_dx, a->x_type, V) &&
                     aligned(a->dres, a->ld_dres, a->x_type, V);
    if (a->rows && a->D <= kMaxD) {
        vec ? run_bwd<TX, TY, V, kEpt / V>(a, sums, s) : run_bwd<TX, TY, 1, kEpt>(a, sums, s);
    } else if (a->rows) {
        const size_t bytes = 8 * (size_t)a->D;
        const int shared = sums && bytes <= kColsShared;
        if (shared) {
            const cudaError_t e = cudaFuncSetAttribute(k_ln_bwd_loop<TX, TY>,
                                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       (int)kColsShared);
            if (e != cudaSuccess) return kmb_cuda_fail(e, "layernorm: shared memory");
        }
        k_ln_bwd_loop<TX, TY><<<(unsigned)parts, kLoop, shared ? bytes : 0, s>>>(*a, sums, shared);
    }
    if (sums)
        k_ln_sums<<<(unsigned)((2 * a->D + 31) / 32), dim3(32, 32), 0, s>>>(
            (const float *)a->workspace, a->rows ? parts : 0, a->D, a->dweight, a->dbias, a->accumulate);
    return done();
}

} // namespace

extern "C" long kmb_layernorm_parts(long rows, long D) {
    if (D <= kMaxD) return ctas(rows, D, kEpt);
    const long most = 8 * D <= (long)kColsShared ? kSMs : 4 * kSMs;
    return rows < most ? (rows > 0 ? rows : 1) : most;
}

extern "C" int kmb_launch_layernorm_fwd(const KmbLayerNorm *a, cudaStream_t s) {
    const int x16 = a->x_type == KMB_BF16, y16 = a->y_type == KMB_BF16;
    if (x16) return y16 ? fwd<__nv_bfloat16, __nv_bfloat16>(a, s) : fwd<__nv_bfloat16, float>(a, s);
    return y16 ? fwd<float, __nv_bfloat16>(a, s) : fwd<float, float>(a, s);
}

extern "C" int kmb_launch_layernorm_bwd(const KmbLayerNorm *a, cudaStream_t s) {
    const int x16 = a->x_type == KMB_BF16, y16 = a->y_type == KMB_BF16;
    if (x16) return y16 ? bwd<__nv_bfloat16, __nv_bfloat16>(a, s) : bwd<__nv_bfloat16, float>(a, s);
    return y16 ? bwd<float, __nv_bfloat16>(a, s) : bwd<float, float>(a, s);
}
