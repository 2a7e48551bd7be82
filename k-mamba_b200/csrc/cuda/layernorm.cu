/*
 * Layer norm, forward and backward (kmamba_b200.h).
 *
 * Per row of D values: mean = sum x / D, rstd = (sum (x - mean)^2 / D +
 * eps)^-1/2, y = (x - mean) rstd w + b.  With xhat = (x - mean) rstd and g =
 * dy w the adjoint is dx = rstd (g - avg g - xhat avg(g xhat)); the weight's
 * and bias' gradients are the column sums of dy xhat and dy.
 *
 * One CTA per row, each pass over the row read from memory again.
 */
#include <cuda_bf16.h>

#include "kmb_common.cuh"
#include "../kmb_internal.h"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float ld(const float *p) { return *p; }
__device__ __forceinline__ float ld(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st(float *p, float v) { *p = v; }
__device__ __forceinline__ void st(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

/* sum over the CTA, the same in every thread */
__device__ float cta_sum(float v) {
    __shared__ float part[kThreads / 32];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < kThreads / 32; ++i) s += part[i];
    return s;
}

/* Sums of rows whose plain fp32 sums overflow are taken again on scaled
 * values: 2^-32 x for the mean (D < 2^31), 2^-80 (x - mean) for the squares.
 * A row with an infinity or a NaN stays what it is. */
constexpr float kDown = 0x1p-32f, kUp = 0x1p32f, kSqDown = 0x1p-80f;

template <typename TX>
__device__ void row_stats(const TX *x, long D, float eps, float &mean, float &rstd) {
    float s = 0.f;
    for (long j = threadIdx.x; j < D; j += kThreads) s += ld(x + j);
    mean = cta_sum(s) / (float)D;
    if (!isfinite(mean)) {
        s = 0.f;
        for (long j = threadIdx.x; j < D; j += kThreads) s = fmaf(ld(x + j), kDown, s);
        mean = cta_sum(s) / (float)D * kUp;
    }
    s = 0.f;
    for (long j = threadIdx.x; j < D; j += kThreads) {
        const float c = ld(x + j) - mean;
        s = fmaf(c, c, s);
    }
    s = cta_sum(s);
    rstd = 1.f / sqrtf(s / (float)D + eps);
    if (!isfinite(s)) {
        s = 0.f;
        for (long j = threadIdx.x; j < D; j += kThreads) {
            const float c = (ld(x + j) - mean) * kSqDown;
            s = fmaf(c, c, s);
        }
        rstd = kSqDown / sqrtf(cta_sum(s) / (float)D + eps * kSqDown * kSqDown);
    }
}

template <typename TX, typename TY>
__global__ void __launch_bounds__(kThreads) k_ln_fwd(KmbLayerNorm a) {
    const long r = blockIdx.x;
    const TX *x = (const TX *)a.x + r * a.ld_x;
    TY *y = (TY *)a.y + r * a.ld_y;
    float mean, rstd;
    row_stats(x, a.D, a.eps, mean, rstd);
    for (long j = threadIdx.x; j < a.D; j += kThreads) {
        const float h = (ld(x + j) - mean) * rstd;
        st(y + j, fmaf(h, a.weight ? a.weight[j] : 1.f, a.bias ? a.bias[j] : 0.f));
    }
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[r] = mean;
        if (a.rstd) a.rstd[r] = rstd;
    }
}

/* CTAs take rows r, r + parts, ...; columns' sums go to the workspace rows
 * [part][dweight D | dbias D]: each column belongs to one thread */
template <typename TX, typename TY>
__global__ void __launch_bounds__(kThreads) k_ln_bwd(KmbLayerNorm a, int sums) {
    float *pw = (float *)a.workspace + (long)blockIdx.x * 2 * a.D, *pb = pw + a.D;
    if (sums)
        for (long j = threadIdx.x; j < a.D; j += kThreads) pw[j] = pb[j] = 0.f;
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
            row_stats(x, a.D, a.eps, mean, rstd);
        }
        float s1 = 0.f, s2 = 0.f;
        for (long j = threadIdx.x; j < a.D; j += kThreads) {
            const float h = (ld(x + j) - mean) * rstd, v = ld(dy + j);
            const float g = a.weight ? v * a.weight[j] : v;
            s1 += g;
            s2 = fmaf(g, h, s2);
            if (sums) {
                pw[j] = fmaf(v, h, pw[j]);
                pb[j] += v;
            }
        }
        s1 = cta_sum(s1) / (float)a.D;
        s2 = cta_sum(s2) / (float)a.D;
        for (long j = threadIdx.x; j < a.D; j += kThreads) {
            const float h = (ld(x + j) - mean) * rstd, v = ld(dy + j);
            const float g = a.weight ? v * a.weight[j] : v;
            const float d = rstd * (g - s1 - h * s2);
            st(dx + j, res ? d + ld(res + j) : d);
        }
    }
}

__global__ void k_ln_sums(const float *part, int parts, long D, float *dw, float *db, int acc) {
    const long j = (long)blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= D) return;
    float w = 0.f, b = 0.f;
    for (int p = 0; p < parts; ++p) {
        w += part[(long)p * 2 * D + j];
        b += part[(long)p * 2 * D + D + j];
    }
    if (dw) dw[j] = acc ? dw[j] + w : w;
    if (db) db[j] = acc ? db[j] + b : b;
}

template <typename TX, typename TY>
int fwd(const KmbLayerNorm *a, cudaStream_t s) {
    k_ln_fwd<TX, TY><<<(unsigned)a->rows, kThreads, 0, s>>>(*a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, "layernorm: launch");
}

template <typename TX, typename TY>
int bwd(const KmbLayerNorm *a, cudaStream_t s) {
    const int sums = a->dweight || a->dbias;
    const int parts = (int)kmb_layernorm_parts(a->rows, a->D);
    if (a->rows) k_ln_bwd<TX, TY><<<(unsigned)parts, kThreads, 0, s>>>(*a, sums);
    if (sums)
        k_ln_sums<<<(unsigned)((a->D + 255) / 256), 256, 0, s>>>(
            (const float *)a->workspace, a->rows ? parts : 0, a->D, a->dweight, a->dbias, a->accumulate);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, "layernorm: launch");
}

} // namespace

extern "C" long kmb_layernorm_parts(long rows, long D) {
    (void)D;
    return rows < 592 ? (rows > 0 ? rows : 1) : 592;
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
