/*
 * Layer norm, forward and backward (kmamba_b200.h).
 *
 * Per row of D values: mean = sum x / D, rstd = (sum (x - mean)^2 / D +
 * eps)^-1/2, y = (x - mean) rstd w + b.  With xhat = (x - mean) rstd and g =
 * dy w the adjoint is dx = rstd (g - avg g - xhat avg(g xhat)); the weight's
 * and bias' gradients are the column sums of dy xhat and dy.
 *
 * Memory bounds both: every tensor is to be read or written once.  A row
 * stays in the registers of a warp (up to 1024 values, 512 in the backward)
 * or a CTA from its load to the store, so the mean and the centred squares
 * are two passes over registers.  CTAs are resident for the whole call and
 * walk the rows.  In the backward every thread keeps the column sums of its
 * own columns, written once at the end as one row of partial sums a CTA,
 * which a second kernel adds in a fixed order (its launch is under way when
 * the first one's CTAs end; one launch of a cluster that adds its sums in
 * shared memory was no faster, 128 x 384 fp32 7.2 against 6.6 us, and slower
 * with more rows).
 *
 * Measured (B200, 6.56 TB/s copy): forward 262144 x 1024 fp32 -> bf16 246 us
 * (6.56 TB/s), 8192 x 8192 bf16 53 us (5.0 TB/s); backward with the residual
 * gradient, 262144 x 1024 fp32, 620 us (6.9 TB/s); backward 2048 x 8192 bf16
 * 37 us (2.7 TB/s: 14 rows a CTA, then the sums), 4096 x 1024 bf16 15.6 us;
 * 128 x 384 fp32 6.6 us (the launches); rows of odd width,
 * 16411 x 1537 bf16, 39 us (2.6 TB/s), where every value is a 2-byte access
 * to shared memory.
 */
#include <cuda_bf16.h>

#include "kmb_common.cuh"
#include "kmb_tma.cuh"
#include "../kmb_internal.h"

namespace {

constexpr int kSMs = 148;
constexpr int kWarps = 8;      /* warps of a CTA whose warps have their own rows */
constexpr int kStages = 8;     /* most stages of a ring */
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
    __device__ __forceinline__ void take(const float *p) { v = *p; }
    __device__ __forceinline__ void get(float *f) const { f[0] = v; }
    static __device__ __forceinline__ void store(float *p, const float *f) { __stcs(p, f[0]); }
};
template <>
struct Vec<float, 4> {
    float4 v;
    __device__ __forceinline__ void load(const float *p) { v = __ldcs(reinterpret_cast<const float4 *>(p)); }
    __device__ __forceinline__ void take(const float *p) { v = *reinterpret_cast<const float4 *>(p); }
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
    __device__ __forceinline__ void take(const __nv_bfloat16 *p) { v = *reinterpret_cast<const unsigned short *>(p); }
    __device__ __forceinline__ void get(float *f) const { f[0] = __uint_as_float((unsigned)v << 16); }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *f) {
        __stcs(reinterpret_cast<unsigned short *>(p), (unsigned short)pack2(f[0], 0.f));
    }
};
template <>
struct Vec<__nv_bfloat16, 4> {
    uint2 v;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { v = __ldcs(reinterpret_cast<const uint2 *>(p)); }
    __device__ __forceinline__ void take(const __nv_bfloat16 *p) { v = *reinterpret_cast<const uint2 *>(p); }
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
    __device__ __forceinline__ void take(const __nv_bfloat16 *p) { v = *reinterpret_cast<const uint4 *>(p); }
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

/* Sums over the threads of a row: L lanes, or with more than one warp a row
 * the whole CTA, through two slots in turn, so that one barrier a sum does. */
template <int L>
struct Reducer {
    float2 (*slot)[32];
    int warps; /* of a row */
    int turn;
    __device__ __forceinline__ Reducer(float2 (*s)[32], int w) : slot(s), warps(w), turn(0) {}
    template <bool TWO>
    __device__ __forceinline__ float2 sum(float a, float b) {
#pragma unroll
        for (int o = L / 2; o; o >>= 1) {
            a += __shfl_xor_sync(~0u, a, o);
            if (TWO) b += __shfl_xor_sync(~0u, b, o);
        }
        if (warps == 1) return make_float2(a, b);
        if (threadIdx.x % 32 == 0) slot[turn][threadIdx.x / 32] = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
        for (int w = 0; w < warps; ++w) {
            const float2 v = slot[turn][w];
            a += v.x;
            if (TWO) b += v.y;
        }
        turn ^= 1;
        return make_float2(a, b);
    }
    __device__ __forceinline__ float2 two(float a, float b) { return sum<true>(a, b); }
    __device__ __forceinline__ float one(float a) { return sum<false>(a, 0.f).x; }
    /* whether p holds for one of the rows that sum together: a warp's threads
     * have to take the same way to the next sum */
    __device__ __forceinline__ bool any(bool p) const { return L < 32 ? __any_sync(~0u, p) : p; }
};

/* Sums of rows whose plain fp32 sums overflow are taken again on scaled
 * values: 2^-32 x for the mean (D < 2^31), 2^-80 (x - mean) for the squares.
 * A row with an infinity or a NaN stays what it is. */
constexpr float kDown = 0x1p-32f, kUp = 0x1p32f, kSqDown = 0x1p-80f;

/* sum(f): the sum of f(pair) over the row's values, pairs of values */
template <typename Red, typename Sum>
__device__ __forceinline__ void row_stats(const Red &red, Sum sum, float inv, float eps, float &mean,
                                          float &rstd) {
    mean = sum([](float2 x) { return x; }) * inv;
    if (red.any(!isfinite(mean))) {
        const float t = sum([](float2 x) { return kmb_mul2(x, kmb_f2s(kDown)); }) * inv * kUp;
        if (!isfinite(mean)) mean = t;
    }
    const float2 m = kmb_f2s(-mean);
    const float s = sum([&](float2 x) {
        const float2 c = kmb_add2(x, m);
        return kmb_mul2(c, c);
    });
    rstd = rsqrtf(fmaf(s, inv, eps));
    if (red.any(!isfinite(s))) {
        const float t = sum([&](float2 x) {
            const float2 c = kmb_mul2(kmb_add2(x, m), kmb_f2s(kSqDown));
            return kmb_mul2(c, c);
        });
        if (!isfinite(s)) rstd = kSqDown * rsqrtf(fmaf(t, inv, eps * kSqDown * kSqDown));
    }
}

/* The thread's columns of a row: each block of L threads has L * EPT
 * columns in a row, EPT / V vectors a thread, a vector of the block's
 * threads side by side.  All of a vector's columns exist or none. */
template <int V, int EPT, int L>
struct Cols {
    static constexpr int NV = EPT / V;
    int base, left; /* the first column, columns from there to the row's end */
    bool full;      /* all columns of the block exist: asked once, not for each value */
    __device__ __forceinline__ Cols(int t, int D) : base((t / L) * L * EPT + (t % L) * V) {
        left = D - base;
        full = (t / L + 1) * L * EPT <= D;
    }
    static __device__ __forceinline__ constexpr int off(int k) { return k * (L * V); }
    __device__ __forceinline__ bool in(int k) const { return off(k) < left; }
    /* f(k) for the vectors that exist, else g(k) */
    template <typename F, typename G>
    __device__ __forceinline__ void each(F f, G g) const {
        if (full) {
#pragma unroll
            for (int k = 0; k < NV; ++k) f(k);
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (in(k)) f(k);
                else g(k);
            }
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        each(f, [](int) {});
    }
    /* a [D] vector, `none` where NULL or not there; vectors of 4 where its address allows */
    __device__ __forceinline__ void vector(const float *p, float none, float2 (&out)[EPT / 2]) const {
        float f[EPT];
#pragma unroll
        for (int e = 0; e < EPT; ++e) f[e] = none;
        if (p) {
            p += base;
            if (V >= 4 && ((size_t)p & 15) == 0)
                each([&](int k) {
#pragma unroll
                    for (int e = 0; e < V / 4; ++e)
                        *reinterpret_cast<float4 *>(f + k * V + 4 * e) =
                            *reinterpret_cast<const float4 *>(p + off(k) + 4 * e);
                });
            else
                each([&](int k) {
#pragma unroll
                    for (int e = 0; e < V; ++e) f[k * V + e] = p[off(k) + e];
                });
        }
#pragma unroll
        for (int e = 0; e < EPT / 2; ++e) out[e] = kmb_f2(f[2 * e], f[2 * e + 1]);
    }
    /* to a [D] vector whose address allows vectors of 4 (V >= 4) */
    __device__ __forceinline__ void columns(float *p, const float2 (&x)[EPT / 2]) const {
        p += base;
        each([&](int k) {
            if (V >= 4) {
#pragma unroll
                for (int e = 0; e < V / 4; ++e) {
                    const float2 l = x[(k * V + 4 * e) / 2], h = x[(k * V + 4 * e) / 2 + 1];
                    *reinterpret_cast<float4 *>(p + off(k) + 4 * e) = make_float4(l.x, l.y, h.x, h.y);
                }
            } else {
                p[off(k)] = k % 2 ? x[k / 2].y : x[k / 2].x;
            }
        });
    }
    template <typename T>
    static __device__ __forceinline__ void unpack(const Vec<T, V> (&raw)[NV], float2 (&x)[EPT / 2]) {
        float f[EPT];
#pragma unroll
        for (int k = 0; k < NV; ++k) raw[k].get(f + k * V);
#pragma unroll
        for (int e = 0; e < EPT / 2; ++e) x[e] = kmb_f2(f[2 * e], f[2 * e + 1]);
    }
    /* the row's values from shared memory (RING) or global memory; 0 where there are none */
    template <bool RING, typename T>
    __device__ __forceinline__ void fetch(const T *p, Vec<T, V> (&raw)[NV]) const {
        p += base;
        each([&](int k) { RING ? raw[k].take(p + off(k)) : raw[k].load(p + off(k)); },
             [&](int k) { raw[k] = Vec<T, V>{}; });
    }
    template <bool RING, typename T>
    __device__ __forceinline__ void load(const T *p, float2 (&x)[EPT / 2]) const {
        Vec<T, V> raw[NV];
        fetch<RING>(p, raw);
        unpack(raw, x);
    }
    template <typename T>
    __device__ __forceinline__ void store(T *p, const float2 (&x)[EPT / 2]) const {
        float f[EPT];
#pragma unroll
        for (int e = 0; e < EPT / 2; ++e) {
            f[2 * e] = x[e].x;
            f[2 * e + 1] = x[e].y;
        }
        p += base;
        each([&](int k) { Vec<T, V>::store(p + off(k), f + k * V); });
    }
    /* the sum of f(pair) over the values that exist */
    template <typename Fn>
    __device__ __forceinline__ float sum(const float2 (&x)[EPT / 2], Fn f) const {
        float2 s = kmb_f2s(0.f);
        if (full) {
#pragma unroll
            for (int e = 0; e < EPT / 2; ++e) s = kmb_add2(s, f(x[e]));
        } else {
#pragma unroll
            for (int e = 0; e < EPT / 2; ++e) {
                const float2 v = f(x[e]);
                s.x += in(2 * e / V) ? v.x : 0.f;
                s.y += in((2 * e + 1) / V) ? v.y : 0.f;
            }
        }
        return s.x + s.y;
    }
};

/* ------------------------------------------------------------------ */
/* forward                                                              */
/* ------------------------------------------------------------------ */

/* set when a wait for a row gave up (kmb_layernorm_check_error) */
__device__ int g_ln_error;

/* Threads that share rows: `rows` consecutive ones of the walk at a time.
 * With one warp a row (or several rows a warp) each warp walks on its own. */
template <int L>
struct Walk {
    int wpr, group, groups, t; /* t: the thread's place among a row's */
    __device__ __forceinline__ explicit Walk(int w) : wpr(w) {
        constexpr int per = 32 / L;
        group = w == 1 ? (int)threadIdx.x / L : 0;
        groups = w == 1 ? (int)blockDim.x / 32 * per : 1;
        t = w == 1 ? (int)threadIdx.x % L : (int)threadIdx.x;
    }
    __device__ __forceinline__ unsigned first() const { return blockIdx.x * (unsigned)groups + (unsigned)group; }
    __device__ __forceinline__ unsigned step() const { return gridDim.x * (unsigned)groups; }
};

/*
 * A ring of rows in shared memory, filled by bulk copies: the rows behind
 * the one in work are under way, whatever the registers hold.  A stage has
 * one row, and is filled again one row
 * late, behind the sums of the next row, when every thread is done with it.
 * (Only rows of more than kNarrow columns, at least 16 bytes apart.)
 *
 * A bulk copy moves whole 16-byte pieces.  A row that does not begin or end
 * on one is copied with the rest of its first and last piece, bytes of the
 * rows beside it, and read from where it begins inside.  A row whose pieces
 * would leave the tensor (the first or the last, when it is not aligned) is
 * loaded by its threads.
 */
enum { kNone, kWhole, kPieces }; /* no ring, rows of whole aligned pieces, any rows */
__host__ __device__ constexpr int ring_head(int rings) { return (rings * kStages * 8 + 127) / 128 * 128; }
__host__ __device__ constexpr int ring_slot(long bytes, int mode) {
    return mode == kPieces ? (int)((bytes + 15) / 16 * 16 + 16) : (int)bytes;
}

template <int MODE>
struct Ring {
    char *buf;     /* stage 0 */
    uint64_t *bar; /* one a stage */
    int bytes, stages;
    int stage, parity;
    bool leader;

    __device__ __forceinline__ void start(char *smem, int row_bytes, int n, int wpr) {
        const int own = wpr == 1 ? (int)threadIdx.x / 32 : 0, rings = wpr == 1 ? (int)blockDim.x / 32 : 1;
        bytes = row_bytes;
        stages = n;
        bar = reinterpret_cast<uint64_t *>(smem) + own * kStages;
        buf = smem + ring_head(rings) + own * n * row_bytes;
        leader = wpr == 1 ? threadIdx.x % 32 == 0 : threadIdx.x == 0;
        stage = parity = 0;
        if (leader)
            for (int k = 0; k < n; ++k) kmb_mbar_init(bar + k, 1);
        kmb_mbar_init_fence();
        if (wpr == 1) __syncwarp();
        else __syncthreads();
    }
    __device__ __forceinline__ char *at(int k) const { return buf + k * bytes; }
    /* A wait that gives up leaves the row unfinished (the error word says so)
     * and the walk goes on, so that all threads meet at its barriers.  The
     * leader starts no copy behind it, whose barrier would be one arrival
     * ahead, and lets the stages - 1 that are under way land, or a second go
     * by: none may write into shared memory that is no longer this CTA's.
     * (A function of its own, not inlined, cost the walk up to 4 %.) */
    __device__ __forceinline__ void wait() {
        if (kmb_mbar_wait(bar + stage, parity, &g_ln_error) || !leader) return;
        leader = false;
        const long long t0 = clock64();
        for (int n = 1, k = stage, odd = parity; n < stages; ++n) {
            while (!kmb_mbar_done(bar + k, odd) && clock64() - t0 < (1ll << 31)) {
            }
            if (++k == stages) {
                k = 0;
                odd ^= 1;
            }
        }
    }
    __device__ __forceinline__ int before() const { return stage ? stage - 1 : stages - 1; }
    __device__ __forceinline__ void next() {
        if (++stage == stages) {
            stage = 0;
            parity ^= 1;
        }
    }
};

/* One of the row's tensors in a ring: where its rows are, which of them have
 * pieces outside the tensor, and the row that the ring is filled with next. */
template <typename T, int MODE>
struct Source {
    const T *next;
    long step; /* elements between the walk's rows */
    int bytes, where;
    bool head, tail; /* the first / the last row of the tensor cannot be copied */
    __device__ __forceinline__ Source(const void *p, long ld, const KmbLayerNorm &a, unsigned row, unsigned s, int at) {
        next = (const T *)p + (long)row * ld;
        step = (long)s * ld;
        bytes = (int)(a.D * sizeof(T));
        where = at;
        head = p && lead(p);
        tail = p && ((lead((const T *)p + (a.rows - 1) * ld) + bytes) & 15u);
    }
    static __device__ __forceinline__ uint32_t lead(const void *p) {
        return MODE == kPieces ? (uint32_t)(uintptr_t)p & 15u : 0u;
    }
    __device__ __forceinline__ uint32_t span() const {
        return MODE == kPieces ? (lead(next) + (uint32_t)bytes + 15u) & ~15u : (uint32_t)bytes;
    }
    __device__ __forceinline__ void copy(const Ring<MODE> &r, int k) const {
        kmb_bulk_load(r.at(k) + where, (const char *)next - lead(next), span(), r.bar + k);
    }
};

/* KEEP: weight and bias stay in registers.  MODE: whether rows come through
 * a ring of `stages`; narrow rows without one are loaded a turn ahead. */
template <typename TX, typename TY, int V, int EPT, int L, bool KEEP, int MODE>
__global__ void __launch_bounds__(KEEP ? 512 : 1024) k_ln_fwd(const __grid_constant__ KmbLayerNorm a, int wpr,
                                                             int stages) {
    extern __shared__ __align__(128) char smem[];
    __shared__ float2 slot[2][32];
    typedef Cols<V, EPT, L> C;
    constexpr bool RING = MODE != kNone, AHEAD = !RING && L < 32;
    const Walk<L> walk(wpr);
    const C c(walk.t, (int)a.D);
    Reducer<L> red(slot, wpr);
    float2 w[KEEP ? EPT / 2 : 1], b[KEEP ? EPT / 2 : 1];
    if constexpr (KEEP) {
        c.vector(a.weight, 1.f, w);
        c.vector(a.bias, 0.f, b);
    }
    const unsigned step = walk.step(), rows = (unsigned)a.rows;
    const float inv = 1.f / (float)a.D;
    Ring<MODE> ring = {};
    Source<TX, MODE> src(a.x, a.ld_x, a, walk.first(), step, 0);
    unsigned ahead = walk.first(); /* the row that the ring is filled with next */
    const auto odd = [&](unsigned row) { return (src.head && row == 0) || (src.tail && row == rows - 1); };
    const auto fill = [&](int k) {
        if (ring.leader) {
            if (ahead >= rows || odd(ahead)) {
                kmb_mbar_arrive(ring.bar + k);
            } else {
                kmb_mbar_expect(ring.bar + k, src.span());
                src.copy(ring, k);
            }
        }
        ahead += step;
        src.next += src.step;
    };
    if (RING) {
        ring.start(smem, ring_slot(src.bytes, MODE), stages, wpr);
        for (int k = 0; k < stages - 1; ++k) fill(k);
    }
    const TX *px = (const TX *)a.x + (long)walk.first() * a.ld_x;
    TY *py = (TY *)a.y + (long)walk.first() * a.ld_y;
    const long sx = (long)step * a.ld_x, sy = (long)step * a.ld_y;
    Vec<TX, V> raw[C::NV] = {};
    if (AHEAD && walk.first() < rows) c.template fetch<false>(px, raw);
    /* with several rows a warp all of its lanes walk as long as one of them */
    const unsigned base = L < 32 ? walk.group % (32 / L) : 0;
    for (unsigned r = walk.first(); r - base < rows; r += step, px += sx, py += sy) {
        const bool live = L == 32 || r < rows;
        float2 x[EPT / 2];
        if (AHEAD) {
            C::unpack(raw, x);
            if (r + step < rows) c.template fetch<false>(px + sx, raw);
        } else {
            if (RING) ring.wait();
            if (RING && !odd(r))
                c.template load<true>((const TX *)(ring.at(ring.stage) + src.lead(px)), x);
            else
                c.template load<false>(px, x);
        }
        float mean, rstd;
        bool filled = !RING;
        row_stats(
            red,
            [&](auto f) {
                const float v = red.one(c.sum(x, f));
                if (!filled) { /* every thread is done with the row before */
                    if (wpr == 1) __syncwarp();
                    fill(ring.before());
                    filled = true;
                }
                return v;
            },
            inv, a.eps, mean, rstd);
        if (RING) ring.next();
        if (!live) continue;
        const float2 m = kmb_f2s(-mean), s = kmb_f2s(rstd);
        if constexpr (KEEP) {
#pragma unroll
            for (int e = 0; e < EPT / 2; ++e) x[e] = kmb_fma2(kmb_mul2(kmb_add2(x[e], m), s), w[e], b[e]);
        } else {
#pragma unroll
            for (int e = 0; e < EPT / 2; ++e) {
                const int i = c.base + c.off(2 * e / V) + 2 * e % V;
                const bool ok = c.in(2 * e / V);
                const float2 wv = ok && a.weight ? *reinterpret_cast<const float2 *>(a.weight + i) : kmb_f2s(1.f);
                const float2 bv = ok && a.bias ? *reinterpret_cast<const float2 *>(a.bias + i) : kmb_f2s(0.f);
                x[e] = kmb_fma2(kmb_mul2(kmb_add2(x[e], m), s), wv, bv);
            }
        }
        c.store(py, x);
        if (walk.t == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

/* rows wider than a CTA's registers: read again for each pass, from L2 */
template <typename TX, typename TY>
__global__ void __launch_bounds__(kLoop) k_ln_fwd_loop(const __grid_constant__ KmbLayerNorm a) {
    __shared__ float2 slot[2][32];
    Reducer<32> red(slot, kLoop / 32);
    const float inv = 1.f / (float)a.D;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const TX *x = (const TX *)a.x + r * a.ld_x;
        TY *y = (TY *)a.y + r * a.ld_y;
        float mean, rstd;
        row_stats(
            red,
            [&](auto f) {
                float s = 0.f;
                for (long j = threadIdx.x; j < a.D; j += kLoop) s += f(kmb_f2s(ld(x + j))).x;
                return red.one(s);
            },
            inv, a.eps, mean, rstd);
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

template <typename TX, typename TY, int V, int EPT, int L, int MODE>
__global__ void __launch_bounds__(512) k_ln_bwd(const __grid_constant__ KmbLayerNorm a, int wpr, int sums,
                                                int stages) {
    extern __shared__ __align__(128) char smem[];
    __shared__ float2 slot[2][32];
    typedef Cols<V, EPT, L> C;
    constexpr bool RING = MODE != kNone, AHEAD = !RING && L < 32;
    const Walk<L> walk(wpr);
    const C c(walk.t, (int)a.D);
    Reducer<L> red(slot, wpr);
    const float inv = 1.f / (float)a.D;
    float2 w[EPT / 2], pw[EPT / 2], pb[EPT / 2];
    c.vector(a.weight, 1.f, w);
#pragma unroll
    for (int e = 0; e < EPT / 2; ++e) pw[e] = pb[e] = kmb_f2s(0.f);
    const unsigned step = walk.step(), rows = (unsigned)a.rows;
    Ring<MODE> ring = {};
    const int xs = ring_slot(a.D * sizeof(TX), MODE), ys = ring_slot(a.D * sizeof(TY), MODE);
    Source<TX, MODE> x_src(a.x, a.ld_x, a, walk.first(), step, 0);
    Source<TY, MODE> d_src(a.dy, a.ld_dy, a, walk.first(), step, xs);
    Source<TX, MODE> r_src(a.dres, a.ld_dres, a, walk.first(), step, xs + ys);
    const bool head = x_src.head || d_src.head || r_src.head, tail = x_src.tail || d_src.tail || r_src.tail;
    unsigned ahead = walk.first(); /* the row that the ring is filled with next */
    const auto odd = [&](unsigned row) { return (head && row == 0) || (tail && row == rows - 1); };
    const auto fill = [&](int k) {
        if (ring.leader) {
            if (ahead >= rows || odd(ahead)) {
                kmb_mbar_arrive(ring.bar + k);
            } else {
                kmb_mbar_expect(ring.bar + k, x_src.span() + d_src.span() + (a.dres ? r_src.span() : 0u));
                x_src.copy(ring, k);
                d_src.copy(ring, k);
                if (a.dres) r_src.copy(ring, k);
            }
        }
        ahead += step;
        x_src.next += x_src.step;
        d_src.next += d_src.step;
        r_src.next += r_src.step;
    };
    if (RING) {
        ring.start(smem, xs + ys + (a.dres ? xs : 0), stages, wpr);
        for (int k = 0; k < stages - 1; ++k) fill(k);
    }
    const TX *px = (const TX *)a.x + (long)walk.first() * a.ld_x;
    const TY *pd = (const TY *)a.dy + (long)walk.first() * a.ld_dy;
    const TX *pr = (const TX *)a.dres + (long)walk.first() * a.ld_dres;
    TX *po = (TX *)a.dx + (long)walk.first() * a.ld_dx;
    Vec<TX, V> rx[C::NV] = {};
    Vec<TY, V> rd[C::NV] = {};
    if (AHEAD && walk.first() < rows) {
        c.template fetch<false>(px, rx);
        c.template fetch<false>(pd, rd);
    }
    const unsigned base = L < 32 ? walk.group % (32 / L) : 0;
    for (unsigned r = walk.first(); r - base < rows; r += step, px += x_src.step, pd += d_src.step,
                  pr += r_src.step, po += (long)step * a.ld_dx) {
        const bool live = L == 32 || r < rows;
        const bool here = RING && !odd(r); /* the row is in the ring */
        float2 h[EPT / 2], d[EPT / 2];
        float m = 0.f, s = 0.f;
        if (live && a.mean) {
            m = a.mean[r];
            s = a.rstd[r];
        }
        if (RING) ring.wait();
        if (AHEAD) {
            C::unpack(rx, h);
            C::unpack(rd, d);
            if (r + step < rows) {
                c.template fetch<false>(px + x_src.step, rx);
                c.template fetch<false>(pd + d_src.step, rd);
            } else { /* a lane without a row adds nothing to the columns' sums */
#pragma unroll
                for (int k = 0; k < C::NV; ++k) {
                    rx[k] = Vec<TX, V>{};
                    rd[k] = Vec<TY, V>{};
                }
            }
        } else if (here) {
            c.template load<true>((const TX *)(ring.at(ring.stage) + x_src.lead(px)), h);
            c.template load<true>((const TY *)(ring.at(ring.stage) + xs + d_src.lead(pd)), d);
        } else {
            c.template load<false>(px, h);
            c.template load<false>(pd, d);
        }
        if (!a.mean) {
            row_stats(red, [&](auto f) { return red.one(c.sum(h, f)); }, inv, a.eps, m, s);
            if (!live) m = s = 0.f; /* of zeros and eps = 0, rstd is infinite, and 0 times it no 0 */
        }
        float2 t1 = kmb_f2s(0.f), t2 = t1;
        const float2 m2 = kmb_f2s(-m), sd = kmb_f2s(s);
#pragma unroll
        for (int e = 0; e < EPT / 2; ++e) { /* d is 0 where a value does not exist */
            h[e] = kmb_mul2(kmb_add2(h[e], m2), sd);
            pw[e] = kmb_fma2(d[e], h[e], pw[e]);
            pb[e] = kmb_add2(pb[e], d[e]);
            d[e] = kmb_mul2(d[e], w[e]);
            t1 = kmb_add2(t1, d[e]);
            t2 = kmb_fma2(d[e], h[e], t2);
        }
        const float2 t = red.two(t1.x + t1.y, t2.x + t2.y);
        if (RING) { /* every thread is done with the row before */
            if (wpr == 1) __syncwarp();
            fill(ring.before());
        }
        const float2 s1 = kmb_f2s(-t.x * inv), s2 = kmb_f2s(-t.y * inv);
#pragma unroll
        for (int e = 0; e < EPT / 2; ++e) d[e] = kmb_mul2(kmb_fma2(h[e], s2, kmb_add2(d[e], s1)), sd);
        if (a.dres && live) {
            if (here)
                c.template load<true>((const TX *)(ring.at(ring.stage) + xs + ys + r_src.lead(pr)), h);
            else
                c.template load<false>(pr, h);
#pragma unroll
            for (int e = 0; e < EPT / 2; ++e) d[e] = kmb_add2(d[e], h[e]);
        }
        if (RING) ring.next();
        if (live) c.store(po, d);
    }
    if (!sums) return;
    float *part = (float *)a.workspace + (long)blockIdx.x * 2 * a.D;
    if (wpr > 1) {
        c.columns(part, pw);
        c.columns(part + a.D, pb);
        return;
    }
    /* one row a group: added through shared memory, the ring's stages when there is one */
    float *fold = reinterpret_cast<float *>(smem + (RING ? ring_head(blockDim.x / 32) : 0));
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        c.columns(fold + walk.group * (L * EPT), which ? pb : pw);
        __syncthreads();
        for (int j = threadIdx.x; j < a.D; j += blockDim.x) {
            float v = 0.f;
            for (int g = 0; g < walk.groups; ++g) v += fold[g * (L * EPT) + j];
            part[which * a.D + j] = v;
        }
    }
}

/* Wider rows: a kernel for the columns' sums (first, since dx may be x or
 * dy), before it one for the statistics when the caller has none, and one
 * for dx, which reads the row a second time, from L2.  Columns are unsigned:
 * a step behind a row of almost 2^31 passes the signed ones. */
template <typename TX>
__global__ void __launch_bounds__(kLoop) k_ln_stats_loop(const __grid_constant__ KmbLayerNorm a, float *mean,
                                                         float *rstd) {
    __shared__ float2 slot[2][32];
    Reducer<32> red(slot, kLoop / 32);
    const unsigned D = (unsigned)a.D;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const TX *x = (const TX *)a.x + r * a.ld_x;
        float m, s;
        row_stats(
            red,
            [&](auto f) {
                float t = 0.f;
                for (unsigned j = threadIdx.x; j < D; j += kLoop) t += f(kmb_f2s(ld(x + j))).x;
                return red.one(t);
            },
            1.f / (float)a.D, a.eps, m, s);
        if (threadIdx.x == 0) {
            mean[r] = m;
            rstd[r] = s;
        }
    }
}

template <typename TX, typename TY, int V>
__global__ void __launch_bounds__(kLoop) k_ln_dx_loop(const __grid_constant__ KmbLayerNorm a) {
    __shared__ float2 slot[2][32];
    Reducer<32> red(slot, kLoop / 32);
    const float inv = 1.f / (float)a.D;
    const unsigned D = (unsigned)a.D;
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
                red,
                [&](auto f) {
                    float s = 0.f;
                    for (unsigned j = threadIdx.x; j < D; j += kLoop) s += f(kmb_f2s(ld(x + j))).x;
                    return red.one(s);
                },
                inv, a.eps, mean, rstd);
        }
        float s1 = 0.f, s2 = 0.f;
        /* f(column, x, g) over the thread's values, four vectors under way */
        const auto each = [&](auto f) {
#pragma unroll 4
            for (unsigned j = threadIdx.x * V; j < D; j += kLoop * V) {
                Vec<TX, V> vx;
                Vec<TY, V> vd;
                vx.take(x + j);
                vd.take(dy + j);
                float h[V], d[V];
                vx.get(h);
                vd.get(d);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    h[e] = (h[e] - mean) * rstd;
                    if (a.weight) d[e] *= a.weight[j + e];
                }
                f(j, h, d);
            }
        };
        each([&](unsigned, const float *h, const float *g) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s1 += g[e];
                s2 = fmaf(g[e], h[e], s2);
            }
        });
        const float2 t = red.two(s1, s2);
        s1 = t.x * inv;
        s2 = t.y * inv;
        each([&](unsigned j, const float *h, const float *g) {
            float o[V], q[V];
            if (res) {
                Vec<TX, V> v;
                v.load(res + j);
                v.get(q);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                o[e] = rstd * (g[e] - s1 - h[e] * s2);
                if (res) o[e] += q[e];
            }
            Vec<TX, V>::store(dx + j, o);
        });
    }
}

/* CTA (column strip, part): the strip's sums over every gridDim.y-th row */
constexpr int kColThreads = 128;

template <typename TX, typename TY, int V>
__global__ void __launch_bounds__(kColThreads) k_ln_cols(const __grid_constant__ KmbLayerNorm a) {
    const long j = ((long)blockIdx.x * kColThreads + threadIdx.x) * V;
    if (j >= a.D) return;
    float w[V] = {}, b[V] = {};
#pragma unroll 4
    for (long r = blockIdx.y; r < a.rows; r += gridDim.y) {
        Vec<TX, V> vx;
        Vec<TY, V> vd;
        vx.load((const TX *)a.x + r * a.ld_x + j);
        vd.load((const TY *)a.dy + r * a.ld_dy + j);
        const float mean = a.mean[r], rstd = a.rstd[r];
        float x[V], d[V];
        vx.get(x);
        vd.get(d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[e] = fmaf(d[e], (x[e] - mean) * rstd, w[e]);
            b[e] += d[e];
        }
    }
    float *part = (float *)a.workspace + (long)blockIdx.y * 2 * a.D + j;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        part[e] = w[e];
        part[a.D + e] = b[e];
    }
}

/* dweight, dbias from the rows of partial sums: 32 columns a CTA, joined in
 * a fixed order */
__global__ void __launch_bounds__(1024) k_ln_sums(const float *part, long parts, long D, float *dw, float *db,
                                                  int acc) {
    __shared__ float s[32][33];
    kmb_wait_before();
    const int tx = threadIdx.x, ty = threadIdx.y, rows = blockDim.y;
    const long j = (long)blockIdx.x * 32 + tx;
    float v = 0.f;
    if (j < 2 * D) {
        float u[4] = {0.f, 0.f, 0.f, 0.f};
        long p = ty;
        for (; p + 3 * rows < parts; p += 4 * rows)
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] += part[(p + k * rows) * 2 * D + j];
        for (; p < parts; p += rows) u[0] += part[p * 2 * D + j];
        v = (u[0] + u[1]) + (u[2] + u[3]);
    }
    s[ty][tx] = v;
    __syncthreads();
    if (ty || j >= 2 * D) return;
    for (int k = 1; k < rows; ++k) v += s[k][tx];
    float *to = j < D ? dw : db;
    if (!to) return;
    to += j < D ? j : j - D;
    *to = acc ? *to + v : v;
}

/* ------------------------------------------------------------------ */
/* launches                                                             */
/* ------------------------------------------------------------------ */

/* Values of a thread.  More of them mean fewer sums across threads (each
 * costs a warp 5 shuffles and a barrier), fewer mean more rows in flight.  Up
 * to 128 columns four rows share a warp. */
int fwd_ept(long D) { return D <= 128 ? 16 : D <= 256 ? 8 : D <= 512 ? 16 : 32; }
int bwd_ept(long D) { return D <= 128 ? 16 : D <= 256 ? 8 : 16; }
constexpr long kNarrow = 128, kFwdKeep = 512 * 32, kFwdWide = 1024 * 32, kBwdMax = 512 * 16;

int warps_of(long D, int ept) { return D <= kNarrow ? 1 : (int)((D + 32 * ept - 1) / (32 * ept)); }
int threads_of(int wpr) { return 32 * (wpr == 1 ? kWarps : wpr); }

/* CTAs of a resident kernel of 512 threads an SM (128 registers each), no
 * more than there are rows (or groups of rows) */
long ctas(long rows, long D, int wpr) {
    const int per = wpr > 1 ? 1 : D <= kNarrow ? 4 * kWarps : kWarps;
    const long need = (rows + per - 1) / per;
    const int fit = 512 / threads_of(wpr);
    const long most = (long)kSMs * (fit > 0 ? fit : 1);
    return need < most ? (need > 0 ? need : 1) : most;
}

/* Stages of a ring whose rows take `bytes` each, 0 for no ring: enough that
 * an SM has 64 KB under way (its share of the memory's bandwidth times the
 * latency), two rows ahead where they fit. */
int ring_stages(long D, int wpr, long bytes) {
    const int rings = wpr == 1 ? kWarps : 1, fit = 512 / threads_of(wpr) > 0 ? 512 / threads_of(wpr) : 1;
    const long all = bytes * rings * fit; /* of an SM */
    if (D <= kNarrow) return 0;
    int n = (int)(2 + (64 * 1024 - 1) / all);
    if (n < 3) n = 3;
    if (n > kStages) n = kStages;
    while (n > 1 && n * all + fit * ring_head(rings) > 208 * 1024) --n;
    return n > 1 ? n : 0;
}
size_t ring_size(int wpr, long bytes, int stages) {
    const int rings = wpr == 1 ? kWarps : 1;
    return ring_head(rings) + (size_t)rings * stages * bytes;
}
/* whether every row begins and ends on a 16-byte piece */
bool whole(const void *p, long ld, long D, size_t es) {
    return !p || ((size_t)p % 16 == 0 && ld * es % 16 == 0 && D * es % 16 == 0);
}

bool aligned(const void *p, long ld, size_t es, int v) {
    return !p || ((size_t)p % (es * v) == 0 && ld % v == 0);
}

int done() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, "layernorm: launch");
}

template <typename K>
int more_shared(K kernel, size_t bytes) {
    if (bytes <= 40 * 1024) return KMB_OK; /* 48 KB with the static part */
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, "layernorm: shared memory");
}

template <typename TX, typename TY, int V, int EPT, int L, bool KEEP>
int run_fwd(const KmbLayerNorm *a, cudaStream_t s) {
    const int wpr = warps_of(a->D, EPT), t = threads_of(wpr);
    const unsigned n = (unsigned)ctas(a->rows, a->D, wpr);
    const bool exact = V > 1 && whole(a->x, a->ld_x, a->D, sizeof(TX));
    const long row = ring_slot(a->D * sizeof(TX), exact ? kWhole : kPieces);
    /* Long rows, one a warp (fp32, up to 1024 columns), keep 64 KB of an SM
     * under way by themselves.  From global memory and through the ring, 100M
     * values: fp32 -> fp32 1024 columns 132 and 139 us, 1000 130 and 141, 896
     * 128 and 142, 768 131 and 145, 640 145 and 151, 520 162 and 142; fp32 ->
     * bf16 1024 94 and 102, 1000 100 and 109, 896 104 and 111, 768 111 and
     * 106, 640 123 and 103, 520 142 and 126.  Both gain from 896 columns on. */
    const int stages = V > 1 && wpr == 1 && row >= 3584 ? 0 : ring_stages(a->D, wpr, row);
    const long per = wpr > 1 ? 1 : kWarps * (32 / L);
    if (L == 32 && stages && a->rows > n * per) { /* more than a row a group */
        const size_t bytes = ring_size(wpr, row, stages);
        constexpr int E = L == 32 && V > 1 ? kWhole : kNone, P = L == 32 ? kPieces : kNone;
        auto k = exact ? k_ln_fwd<TX, TY, V, EPT, L, KEEP, E> : k_ln_fwd<TX, TY, V, EPT, L, KEEP, P>;
        const int rc = more_shared(k, bytes);
        if (rc) return rc;
        k<<<n, t, bytes, s>>>(*a, wpr, stages);
    } else {
        k_ln_fwd<TX, TY, V, EPT, L, KEEP, kNone><<<n, t, 0, s>>>(*a, wpr, 0);
    }
    return done();
}

template <typename TX, typename TY, int V>
int fwd_v(const KmbLayerNorm *a, cudaStream_t s) {
    if (a->D <= kNarrow) return run_fwd<TX, TY, V, 16, 8, true>(a, s);
    if (fwd_ept(a->D) == 8) return run_fwd<TX, TY, V, 8, 32, true>(a, s);
    if (fwd_ept(a->D) == 16) return run_fwd<TX, TY, V, 16, 32, true>(a, s);
    if (a->D <= kFwdKeep) return run_fwd<TX, TY, V, 32, 32, true>(a, s);
    if (V > 1 && a->D <= kFwdWide) return run_fwd<TX, TY, V, 32, 32, V == 1>(a, s);
    k_ln_fwd_loop<TX, TY><<<(unsigned)(a->rows < 4 * kSMs ? a->rows : 4 * kSMs), kLoop, 0, s>>>(*a);
    return done();
}

template <typename TX, typename TY>
int fwd(const KmbLayerNorm *a, cudaStream_t s) {
    constexpr int V = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
    /* the widest rows read weight and bias by pairs */
    const bool vec = a->D % V == 0 && aligned(a->x, a->ld_x, sizeof(TX), V) &&
                     aligned(a->y, a->ld_y, sizeof(TY), V) &&
                     (a->D <= kFwdKeep || (aligned(a->weight, 0, 4, 2) && aligned(a->bias, 0, 4, 2)));
    return vec ? fwd_v<TX, TY, V>(a, s) : fwd_v<TX, TY, 1>(a, s);
}

template <typename TX, typename TY, int V, int EPT, int L>
int run_bwd(const KmbLayerNorm *a, int sums, cudaStream_t s) {
    const int wpr = warps_of(a->D, EPT), t = threads_of(wpr);
    const unsigned n = (unsigned)ctas(a->rows, a->D, wpr);
    const size_t fold = sums && wpr == 1 ? (size_t)kWarps * 32 * EPT * 4 : 0;
    const bool exact = V > 1 && whole(a->x, a->ld_x, a->D, sizeof(TX)) &&
                       whole(a->dy, a->ld_dy, a->D, sizeof(TY)) && whole(a->dres, a->ld_dres, a->D, sizeof(TX));
    const int mode = exact ? kWhole : kPieces;
    const long row = ring_slot(a->D * sizeof(TX), mode) * (a->dres ? 2 : 1) + ring_slot(a->D * sizeof(TY), mode);
    const int stages = ring_stages(a->D, wpr, row);
    const long per = wpr > 1 ? 1 : kWarps * (32 / L);
    if (L == 32 && stages && a->rows > n * per) {
        size_t bytes = ring_size(wpr, row, stages);
        if (fold && bytes < ring_head(kWarps) + fold) bytes = ring_head(kWarps) + fold;
        constexpr int E = L == 32 && V > 1 ? kWhole : kNone, P = L == 32 ? kPieces : kNone;
        auto k = exact ? k_ln_bwd<TX, TY, V, EPT, L, E> : k_ln_bwd<TX, TY, V, EPT, L, P>;
        const int rc = more_shared(k, bytes);
        if (rc) return rc;
        k<<<n, t, bytes, s>>>(*a, wpr, sums, stages);
    } else {
        k_ln_bwd<TX, TY, V, EPT, L, kNone><<<n, t, fold, s>>>(*a, wpr, sums, 0);
    }
    return done();
}

template <typename TX, typename TY, int V>
int bwd_v(const KmbLayerNorm *a, int sums, cudaStream_t s) {
    if (a->D <= kNarrow) return run_bwd<TX, TY, V, 16, 8>(a, sums, s);
    if (bwd_ept(a->D) == 8) return run_bwd<TX, TY, V, 8, 32>(a, sums, s);
    return run_bwd<TX, TY, V, 16, 32>(a, sums, s);
}

/* Parts of the columns' kernel: some eight CTAs an SM over its strips. */
long col_parts(long rows, long D) {
    const long strips = (D / 8 + kColThreads - 1) / kColThreads; /* vectors of 8 */
    long n = 8L * kSMs / strips;
    if (n > rows / 4) n = rows / 4;
    return n > 1 ? n : 1;
}

long sum_parts(long rows, long D) {
    return D <= kBwdMax ? ctas(rows, D, warps_of(D, bwd_ept(D))) : col_parts(rows, D);
}

template <typename TX, typename TY, int V>
int bwd_wide(const KmbLayerNorm *a, int sums, cudaStream_t s) {
    KmbLayerNorm d = *a;
    const long parts = col_parts(a->rows, a->D);
    const unsigned n = (unsigned)(a->rows < 3 * kSMs ? a->rows : 3 * kSMs);
    if (sums) {
        if (!d.mean) {
            d.mean = (float *)a->workspace + parts * 2 * a->D;
            d.rstd = d.mean + a->rows;
            k_ln_stats_loop<TX><<<n, kLoop, 0, s>>>(*a, d.mean, d.rstd);
        }
        const dim3 grid((unsigned)((a->D / V + kColThreads - 1) / kColThreads), (unsigned)parts);
        k_ln_cols<TX, TY, V><<<grid, kColThreads, 0, s>>>(d);
    }
    k_ln_dx_loop<TX, TY, V><<<n, kLoop, 0, s>>>(d);
    return done();
}

template <typename TX, typename TY>
int bwd(const KmbLayerNorm *a, cudaStream_t s) {
    constexpr int V = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
    const int sums = a->dweight || a->dbias;
    const long parts = sum_parts(a->rows, a->D);
    const bool vec = a->D % V == 0 && aligned(a->x, a->ld_x, sizeof(TX), V) &&
                     aligned(a->dy, a->ld_dy, sizeof(TY), V) && aligned(a->dx, a->ld_dx, sizeof(TX), V) &&
                     aligned(a->dres, a->ld_dres, sizeof(TX), V);
    int rc = KMB_OK;
    if (a->rows && a->D <= kBwdMax)
        rc = vec ? bwd_v<TX, TY, V>(a, sums, s) : bwd_v<TX, TY, 1>(a, sums, s);
    else if (a->rows)
        rc = vec ? bwd_wide<TX, TY, V>(a, sums, s) : bwd_wide<TX, TY, 1>(a, sums, s);
    if (rc || !sums) return rc;
    /* Rows of threads of the sums' kernel: many where its CTAs are few.  Of a
     * call with 8 and 32, fp32: 2048 x 1024 16.4 and 14.4 us, 4096 x 1024 20.5
     * and 18.5, 4096 x 2048 24.8 and 24.6; 4096 x 2560 28.7 and 30.8, 4096 x
     * 4096 39.0 and 41.2, 2048 x 8192 41.0 and 46.0, 64 x 8192 8.3 and 14.4. */
    const cudaError_t e = kmb_launch_after(
        true, k_ln_sums, (unsigned)((2 * a->D + 31) / 32), dim3(32, a->D <= 2048 ? 32 : 8), 0, s,
        (const float *)a->workspace, a->rows ? parts : 0L, a->D, a->dweight, a->dbias, a->accumulate);
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, "layernorm: launch");
}

} // namespace

/* partial sums, and behind them the statistics of wide rows */
extern "C" size_t kmb_layernorm_scratch_bytes(long rows, long D) {
    return 8 * (size_t)sum_parts(rows, D) * (size_t)D + (D > kBwdMax ? 8 * (size_t)rows : 0);
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

/* Sets the word as an expired wait does (tests of what comes after one). */
extern "C" int kmb_layernorm_expire(void) {
    const int one = 1;
    const cudaError_t e = cudaMemcpyToSymbol(g_ln_error, &one, sizeof one);
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, "layernorm: error word");
}

/* KMB_ETIMEOUT (and the word cleared) when a wait for a row gave up since
 * the last check. */
extern "C" int kmb_layernorm_check_error(void) {
    int flag = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&flag, g_ln_error, sizeof flag);
    if (e != cudaSuccess) return kmb_cuda_fail(e, "layernorm: error word");
    if (flag) {
        const int zero = 0;
        (void)cudaMemcpyToSymbol(g_ln_error, &zero, sizeof zero);
        return kmb_fail(KMB_ETIMEOUT, "layernorm: a wait for a row expired");
    }
    return KMB_OK;
}
