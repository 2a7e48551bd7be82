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
 * Both directions are one pass over the data.  A CTA takes a tile of rows x
 * 64 channels: a warp owns a run of consecutive rows, a lane two channels.
 * A run is first reduced to its affine map h -> A h + H, the maps of a
 * tile's warps are joined through shared memory, and the maps of the tiles
 * of one channel group through global memory: a tile publishes its map,
 * waits until each of the tiles before it shows either its map or its final
 * state, applies the maps from the nearest final state on, publishes its
 * own final state and only then runs its rows from the state that enters
 * them.  The final state of a tile is always the map of that tile applied
 * to the final state of the one before it, whichever of the two was read,
 * so results do not depend on timing.
 */
#include <cuda_bf16.h>

#include "kmb_common.cuh"
#include "../kmb_internal.h"

namespace {

constexpr int kChunk = KMB_GLR_CHUNK;
constexpr int kC = 64;      /* channels of a tile: two a lane */
constexpr int kWindow = 16; /* tiles before its own that a tile looks at */
constexpr unsigned kUnset = 0xffffffffu; /* workspace word not written yet */

/* set when a wait for another tile's state gave up (kmb_glr_check_error) */
__device__ int g_glr_error;

/* ------------------------------------------------------------------ */
/* two channels of one row                                              */
/* ------------------------------------------------------------------ */

__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return kmb_f2(a.x - b.x, a.y - b.y); }
__device__ __forceinline__ float2 neg2(float2 a) { return kmb_f2(-a.x, -a.y); }

/* VEC: channels 2 lane, 2 lane + 1 in one access; else lane and lane + 32,
 * for odd widths, strides and addresses (every access still covers a
 * contiguous piece of the row). */
template <typename T>
struct Raw;
template <>
struct Raw<float> {
    typedef float2 type;
    static __device__ __forceinline__ float2 f(float2 v) { return v; }
    template <bool VEC>
    static __device__ __forceinline__ float2 load(const float *p, bool ok0, bool ok1) {
        if (VEC) return ok0 ? __ldcs(reinterpret_cast<const float2 *>(p)) : kmb_f2s(0.f);
        return kmb_f2(ok0 ? __ldcs(p) : 0.f, ok1 ? __ldcs(p + 32) : 0.f);
    }
    template <bool VEC>
    static __device__ __forceinline__ void store(float *p, float2 v, bool ok0, bool ok1) {
        if (VEC) {
            if (ok0) __stcs(reinterpret_cast<float2 *>(p), v);
            return;
        }
        if (ok0) __stcs(p, v.x);
        if (ok1) __stcs(p + 32, v.y);
    }
};
template <>
struct Raw<__nv_bfloat16> {
    typedef unsigned type; /* the first channel in the low half */
    static __device__ __forceinline__ float2 f(unsigned v) {
        return kmb_f2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    template <bool VEC>
    static __device__ __forceinline__ unsigned load(const __nv_bfloat16 *p, bool ok0, bool ok1) {
        if (VEC) return ok0 ? __ldcs(reinterpret_cast<const unsigned *>(p)) : 0u;
        const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
        const unsigned a = ok0 ? __ldcs(q) : 0u, b = ok1 ? __ldcs(q + 32) : 0u;
        return a | b << 16;
    }
    template <bool VEC>
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, float2 v, bool ok0, bool ok1) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
        const unsigned u = *reinterpret_cast<const unsigned *>(&h);
        if (VEC) {
            if (ok0) __stcs(reinterpret_cast<unsigned *>(p), u);
            return;
        }
        unsigned short *q = reinterpret_cast<unsigned short *>(p);
        if (ok0) __stcs(q, (unsigned short)u);
        if (ok1) __stcs(q + 32, (unsigned short)(u >> 16));
    }
};

__device__ __forceinline__ float softplus(float v) { return v > 20.f ? v + expf(-v) : log1pf(expf(v)); }
/* sigmoid / softplus: 1 where both vanish */
__device__ __forceinline__ float decay_ratio(float v) {
    return v < -15.f ? 1.f : 1.f / (1.f + expf(-v)) / softplus(v);
}

__device__ __forceinline__ float rsqrt_mufu(float v) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(v));
    return y;
}
__device__ __forceinline__ float rcp_mufu(float v) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(v));
    return y;
}
__device__ __forceinline__ float sqrt_mufu(float v) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(v));
    return y;
}

/*
 * Polynomials of the exponent u on [0, kWeak], fitted for minimax relative
 * error with the constant term held (iteratively reweighted least squares
 * on Chebyshev nodes); in fp32 Horner form each is within 7e-8:
 *   (1 - e^-u) / u                    2.9e-9 in real arithmetic
 *   sqrt((1 - e^-2u) / (2 u))         4.8e-9
 *   kappa = u / (e^2u - 1)            3.4e-9
 * A channel whose rate is at most kWeak needs no exponential of u, no
 * square root and no cancelling 1 - a^2, and its recurrence runs on w = 1 -
 * a as h + (b - w h): a memory of 1 / w steps multiplies the error of the
 * decay, and a itself, next to 1, cannot hold w to more than 2^-25 / w.
 */
constexpr float kWeak = 0.25f;

__device__ __forceinline__ float2 poly4(float2 u, float c0, float c1, float c2, float c3, float c4) {
    float2 p = kmb_fma2(kmb_f2s(c4), u, kmb_f2s(c3));
    p = kmb_fma2(p, u, kmb_f2s(c2));
    p = kmb_fma2(p, u, kmb_f2s(c1));
    return kmb_fma2(p, u, kmb_f2s(c0));
}
__device__ __forceinline__ float2 poly_w(float2 u) {
    return poly4(u, 1.f, -0.49999964237213135f, 0.1666528880596161f, -0.04150013253092766f,
                 0.007530174218118191f);
}
__device__ __forceinline__ float2 poly_root(float2 u) {
    return poly4(u, 1.f, -0.49999940395355225f, 0.20831027626991272f, -0.06222091242671013f,
                 0.01236682292073965f);
}
__device__ __forceinline__ float2 poly_kappa(float2 u) {
    return poly4(u, 0.5f, -0.5000002980232239f, 0.1666753739118576f, -8.377274934900925e-05f,
                 -0.010830916464328766f);
}

/* Per channel: rate, and sqrt(2 rate) for root = sqrt(2 u) sqrt((1 - e^-2u) / 2u). */
struct Rates {
    float2 rate, sroot;
};

/* Of one row: c is 1 - a (WEAK) or a, q = sqrt(r) = (1 + e^-gate_r)^-1/2, i,
 * and si = root i. */
struct Terms {
    float2 c, q, i, si;
};

template <bool WEAK>
__device__ __forceinline__ Terms terms(float2 gr, float2 gi, const Rates &k) {
    Terms t;
    const float2 nl = kmb_f2s(-KMB_LOG2E), one = kmb_f2s(1.f);
    const float2 er = kmb_add2(kmb_ex2_2(kmb_mul2(gr, nl)), one);
    const float2 ei = kmb_add2(kmb_ex2_2(kmb_mul2(gi, nl)), one);
    t.q = kmb_f2(rsqrt_mufu(er.x), rsqrt_mufu(er.y));
    t.i = kmb_f2(rcp_mufu(ei.x), rcp_mufu(ei.y));
    const float2 u = kmb_mul2(k.rate, kmb_mul2(t.q, t.q));
    const float2 w = kmb_mul2(u, poly_w(u));
    float2 root = kmb_mul2(kmb_mul2(k.sroot, t.q), poly_root(u));
    if (WEAK) {
        t.c = w;
    } else {
        const float2 e = kmb_ex2_2(kmb_mul2(u, nl));
        t.c = kmb_f2(u.x <= kWeak ? 1.f - w.x : e.x, u.y <= kWeak ? 1.f - w.y : e.y);
        root = kmb_f2(u.x <= kWeak ? root.x : sqrt_mufu(fmaf(-e.x, e.x, 1.f)),
                      u.y <= kWeak ? root.y : sqrt_mufu(fmaf(-e.y, e.y, 1.f)));
    }
    t.si = kmb_mul2(root, t.i);
    return t;
}

/* a h + b */
template <bool WEAK>
__device__ __forceinline__ float2 advance(float2 c, float2 h, float2 b) {
    return WEAK ? kmb_add2(h, kmb_fma2(neg2(c), h, b)) : kmb_fma2(c, h, b);
}
/* a A */
template <bool WEAK>
__device__ __forceinline__ float2 shrink(float2 c, float2 A) {
    return WEAK ? kmb_fma2(neg2(c), A, A) : kmb_mul2(c, A);
}

/* ------------------------------------------------------------------ */
/* affine maps; A = -1 marks a constant one (a sequence began inside)    */
/* ------------------------------------------------------------------ */

__device__ __forceinline__ float apply(float A, float H, float h) { return A < 0.f ? H : fmaf(A, h, H); }

/* the map of `first` then `then` */
__device__ __forceinline__ float2 join(float2 first, float2 then) {
    if (then.x < 0.f) return then;
    return kmb_f2(first.x < 0.f ? -1.f : first.x * then.x, fmaf(then.x, first.y, then.y));
}

__device__ __forceinline__ float not_unset(float v) {
    return __float_as_uint(v) == kUnset ? __uint_as_float(0x7fffffffu) : v;
}

__device__ __forceinline__ unsigned peek(const float *p) {
    unsigned v;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void show(float *p, float v) {
    asm volatile("st.relaxed.gpu.global.f32 [%0], %1;" ::"l"(p), "f"(not_unset(v)) : "memory");
}

/* What tiles show one another: [position in the chain][chain][channel].
 * Every word is written once, and was kUnset (the workspace is filled at
 * the start of the call): a word that is not kUnset is the value itself, so
 * no fence orders flags against data. */
struct Shown {
    float *A, *H, *end; /* map, final state */
    long step;          /* words between positions of a chain */
};

/* The map of a position, or as a constant one its final state: waits for
 * whichever comes first (last: for the final state).  Bounded by about 2^31
 * cycles; then the error word is set and later waits return at once. */
__device__ __forceinline__ float2 look(const Shown &s, long pos, int ch, bool last) {
    const long o = pos * s.step + ch;
    const long long t0 = clock64();
    for (int n = 0;; ++n) {
        const unsigned e = peek(s.end + o);
        if (e != kUnset) return kmb_f2(-1.f, __uint_as_float(e));
        if (!last) {
            const unsigned a = peek(s.A + o), h = peek(s.H + o);
            if (a != kUnset && h != kUnset) return kmb_f2(__uint_as_float(a), __uint_as_float(h));
        }
        if ((n & 63) == 63) {
            if (*reinterpret_cast<volatile int *>(&g_glr_error)) return kmb_f2(-1.f, 0.f);
            if (clock64() - t0 > (1ll << 31)) {
                atomicExch(&g_glr_error, 1);
                return kmb_f2(-1.f, 0.f);
            }
        }
    }
}

/* ------------------------------------------------------------------ */
/* kernel arguments and a tile's place                                  */
/* ------------------------------------------------------------------ */

struct Dev {
    KmbGLR a;
    long tiles, groups, chains; /* tiles of a chain, channel groups, batch * groups */
    long chunks;                /* checkpoints of a chain */
    int states_only;            /* forward: checkpoints alone are wanted */
    const float *ckpt_in;
    float *ckpt_out;
    float *part;                /* [tiles * batch][groups * 64] sums of u dL/du */
    unsigned *ticket;
    Shown shown;
};

struct Place {
    long pos, chain, b, ch0; /* place in the chain, chain, sequence (0 when packed), first channel */
};

/* Tiles are taken in the order of their positions: a tile waits only for
 * tiles that another CTA has taken before. */
__device__ __forceinline__ Place place(const Dev &p, unsigned *slot) {
    if (p.tiles > 1) {
        if (threadIdx.x == 0) *slot = atomicAdd(p.ticket, 1u) + 1u; /* the fill makes it -1 */
        __syncthreads();
    }
    const long id = p.tiles > 1 ? (long)*slot : (long)blockIdx.x;
    Place t;
    t.pos = id / p.chains;
    t.chain = id - t.pos * p.chains;
    t.b = t.chain / p.groups;
    t.ch0 = (t.chain - t.b * p.groups) * kC;
    return t;
}

/* Packed rows: which sequence a row of the tile belongs to and whether it
 * is its first or last. */
template <int ROWS>
struct RowMap {
    int seq[ROWS];
    unsigned char edge[ROWS]; /* 1: first row, 2: last row */
};

/* First sequence whose end lies behind `row`: the number of ends <= row,
 * found by a warp, 32 probes at a time. */
__device__ __forceinline__ long first_sequence(const long *off, long n, long row, int lane) {
    long lo = 0, hi = n; /* the answer is in [lo, hi] */
    while (lo < hi) {
        const long step = (hi - lo + 31) / 32;
        const long k = lo + lane * step; /* probe: does sequence k end at or before row? */
        const bool past = k < hi && off[k + 1] <= row;
        const int m = __popc(__ballot_sync(~0u, past));
        if (m == 0) return lo;
        const long nlo = lo + (m - 1) * step + 1, nhi = lo + m * step;
        lo = nlo;
        hi = nhi < hi ? nhi : hi;
    }
    return lo;
}

template <int ROWS>
__device__ void map_rows(RowMap<ROWS> &m, const KmbGLR &a, long row0) {
    for (int r = threadIdx.x; r < ROWS; r += blockDim.x) {
        m.seq[r] = -1;
        m.edge[r] = 0;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        const long end = row0 + ROWS < a.L ? row0 + ROWS : a.L;
        for (long s = first_sequence(a.offsets, a.batch, row0, lane); s < a.batch; s += 32) {
            long lo = end, hi = end;
            if (s + lane < a.batch) {
                lo = a.offsets[s + lane];
                hi = a.offsets[s + lane + 1];
            }
            const long from = lo > row0 ? lo : row0, to = hi < end ? hi : end;
            for (long r = from; r < to; ++r) {
                m.seq[r - row0] = (int)(s + lane);
                m.edge[r - row0] = (unsigned char)((r == (lo < 0 ? 0 : lo) ? 1 : 0) | (r == (hi > a.L ? a.L : hi) - 1 ? 2 : 0));
            }
            if (__any_sync(~0u, s + lane < a.batch && lo >= end)) break;
        }
    }
    __syncthreads();
}

/* What an empty sequence's end is: `from` (zeros when NULL) to `to`. */
__device__ void empty_sequences(const KmbGLR &a, const float *from, float *to, long ch0) {
    if (!to) return;
    const int lane = threadIdx.x % 32, warps = blockDim.x / 32;
    for (long s = (threadIdx.x / 32) * 32L; s < a.batch; s += warps * 32L) {
        bool none = false;
        if (s + lane < a.batch) {
            long lo = a.offsets[s + lane], hi = a.offsets[s + lane + 1];
            lo = lo < 0 ? 0 : lo;
            hi = hi > a.L ? a.L : hi;
            none = lo >= hi;
        }
        unsigned m = __ballot_sync(~0u, none);
        while (m) {
            const long k = s + __ffs(m) - 1;
            m &= m - 1;
            for (long d = ch0 + lane; d < a.D && d < ch0 + kC; d += 32)
                to[k * a.D + d] = from ? from[k * a.D + d] : 0.f;
        }
    }
}

template <typename T>
__device__ __forceinline__ T *row_ptr(const KmbRows &r, long b, long t, long d) {
    return (T *)r.data + b * r.batch_stride + t * r.row_stride + d;
}

/* The lane's channels: the first, whether each exists. */
template <bool VEC>
struct Lane {
    long d;
    int off; /* within the group */
    bool ok0, ok1;
    static constexpr int kNext = VEC ? 1 : 32; /* to the second channel */
    __device__ __forceinline__ Lane(long ch0, long D) {
        const int lane = threadIdx.x % 32;
        off = VEC ? 2 * lane : lane;
        d = ch0 + off;
        ok0 = d < D;
        ok1 = d + kNext < D;
    }
    /* a [.., D] fp32 vector of the channels */
    __device__ __forceinline__ float2 get(const float *p) const {
        return kmb_f2(p && ok0 ? p[d] : 0.f, p && ok1 ? p[d + kNext] : 0.f);
    }
    __device__ __forceinline__ void put(float *p, float2 v) const {
        if (p && ok0) p[d] = v.x;
        if (p && ok1) p[d + kNext] = v.y;
    }
};

__device__ __forceinline__ Rates rates(float2 decay, float scale) {
    Rates k;
    k.rate = kmb_f2(scale * softplus(decay.x), scale * softplus(decay.y));
    k.sroot = kmb_f2(sqrtf(2.f * k.rate.x), sqrtf(2.f * k.rate.y));
    return k;
}

/* Joins the tile with the ones before it in its chain and returns the state
 * that enters it.  sagg: the warps' maps; `run` the number of warps, in the
 * order that the recurrence runs; first: the state that enters the chain. */
template <bool VEC>
__device__ __forceinline__ float2 enter_tile(const Dev &p, const Place &at, const Lane<VEC> &ln,
                                             const float2 (*sagg)[kC], float2 (*smap)[kC], int warps,
                                             bool reverse, const float *first) {
    const int warp = threadIdx.x / 32;
    const float2 init = ln.get(first);
    if (p.tiles == 1) return init;
    Shown s = p.shown;
    s.A += at.chain * kC;
    s.H += at.chain * kC;
    s.end += at.chain * kC;
    float2 m0 = kmb_f2(1.f, 0.f), m1 = m0;
    const long o = at.pos * s.step + ln.off;
    if (warp == 0) {
        for (int k = 0; k < warps; ++k) {
            const int w = reverse ? warps - 1 - k : k;
            m0 = join(m0, sagg[w][ln.off]);
            m1 = join(m1, sagg[w][ln.off + Lane<VEC>::kNext]);
        }
        if (at.pos > 0 && at.pos + 1 < p.tiles) {
            show(s.A + o, m0.x);
            show(s.H + o, m0.y);
            show(s.A + o + Lane<VEC>::kNext, m1.x);
            show(s.H + o + Lane<VEC>::kNext, m1.y);
        }
    }
    float2 h = init;
    if (at.pos > 0) {
        const int n = at.pos < kWindow ? (int)at.pos : kWindow;
        for (int k = warp; k < n; k += warps) {
            const bool last = k == kWindow - 1;
            smap[k][ln.off] = look(s, at.pos - 1 - k, ln.off, last);
            smap[k][ln.off + Lane<VEC>::kNext] = look(s, at.pos - 1 - k, ln.off + Lane<VEC>::kNext, last);
        }
        __syncthreads();
        /* from the nearest final state (or the chain's beginning) on */
        int k0 = 0, k1 = 0;
        while (k0 < n && !(smap[k0][ln.off].x < 0.f)) ++k0;
        while (k1 < n && !(smap[k1][ln.off + Lane<VEC>::kNext].x < 0.f)) ++k1;
        for (int k = k0 < n ? k0 : n - 1; k >= 0; --k) h.x = apply(smap[k][ln.off].x, smap[k][ln.off].y, h.x);
        for (int k = k1 < n ? k1 : n - 1; k >= 0; --k)
            h.y = apply(smap[k][ln.off + Lane<VEC>::kNext].x, smap[k][ln.off + Lane<VEC>::kNext].y, h.y);
    }
    if (warp == 0 && at.pos + 1 < p.tiles) {
        show(s.end + o, apply(m0.x, m0.y, h.x));
        show(s.end + o + Lane<VEC>::kNext, apply(m1.x, m1.y, h.y));
    }
    return h;
}

/* ------------------------------------------------------------------ */
/* forward                                                              */
/* ------------------------------------------------------------------ */

constexpr int kFR = 8;           /* rows of a warp */
constexpr int kFW = 16;          /* warps of a full CTA */
constexpr int kFT = kFR * kFW;   /* rows of a tile */

template <typename T, bool VEC, bool PACKED>
struct FwdShared {
    float2 agg[kFW][kC];
    float2 map[kWindow][kC];
    unsigned slot;
    RowMap<PACKED ? kFT : 1> rows;
};

template <typename T, bool VEC, bool PACKED, bool WEAK>
__device__ __forceinline__ void fwd_tile(const Dev &p, const Place &at, const Lane<VEC> &ln,
                                         const Rates &rt, FwdShared<T, VEC, PACKED> &sh,
                                         const typename Raw<T>::type (&x)[kFR],
                                         const typename Raw<T>::type (&gr)[kFR],
                                         const typename Raw<T>::type (&gi)[kFR], long row0, int live) {
    const int warp = threadIdx.x / 32, warps = blockDim.x / 32;
    float2 c[kFR], b[kFR];
    float2 A = kmb_f2s(1.f), H = kmb_f2s(0.f);
#pragma unroll
    for (int j = 0; j < kFR; ++j) {
        const Terms t = terms<WEAK>(Raw<T>::f(gr[j]), Raw<T>::f(gi[j]), rt);
        c[j] = t.c;
        b[j] = kmb_mul2(t.si, Raw<T>::f(x[j]));
    }
    bool fresh = false; /* a sequence begins in this run */
#pragma unroll
    for (int j = 0; j < kFR; ++j) {
        const int lr = warp * kFR + j;
        if (PACKED ? sh.rows.seq[lr] >= 0 : j < live) {
            if (PACKED && (sh.rows.edge[lr] & 1)) {
                H = ln.get(p.a.h0 ? p.a.h0 + sh.rows.seq[lr] * p.a.D : nullptr);
                fresh = true;
            }
            H = advance<WEAK>(c[j], H, b[j]);
            A = shrink<WEAK>(c[j], A);
        }
    }
    if (fresh) A = kmb_f2s(-1.f);
    sh.agg[warp][ln.off] = kmb_f2(A.x, H.x);
    sh.agg[warp][ln.off + Lane<VEC>::kNext] = kmb_f2(A.y, H.y);
    __syncthreads();
    const float *first = !PACKED && p.a.h0 ? p.a.h0 + at.b * p.a.D : nullptr;
    float2 h = enter_tile<VEC>(p, at, ln, sh.agg, sh.map, warps, false, first);
    for (int w = 0; w < warp; ++w) {
        const float2 m0 = sh.agg[w][ln.off], m1 = sh.agg[w][ln.off + Lane<VEC>::kNext];
        h = kmb_f2(apply(m0.x, m0.y, h.x), apply(m1.x, m1.y, h.y));
    }
    if (p.ckpt_out && row0 % kChunk == 0 && row0 < p.a.L)
        ln.put(p.ckpt_out + (at.b * p.chunks + row0 / kChunk) * p.a.D, h);
#pragma unroll
    for (int j = 0; j < kFR; ++j) {
        const int lr = warp * kFR + j;
        if (PACKED ? sh.rows.seq[lr] >= 0 : j < live) {
            if (PACKED && (sh.rows.edge[lr] & 1))
                h = ln.get(p.a.h0 ? p.a.h0 + sh.rows.seq[lr] * p.a.D : nullptr);
            h = advance<WEAK>(c[j], h, b[j]);
            if (!p.states_only)
                Raw<T>::template store<VEC>(row_ptr<T>(p.a.y, at.b, row0 + j, ln.d), h, ln.ok0, ln.ok1);
            if (PACKED && (sh.rows.edge[lr] & 2) && p.a.h_last) ln.put(p.a.h_last + sh.rows.seq[lr] * p.a.D, h);
        }
    }
    if (!PACKED && p.a.h_last && live > 0 && row0 + live == p.a.L) ln.put(p.a.h_last + at.b * p.a.D, h);
}

template <typename T, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kFW * 32, 2) k_glr_fwd(const Dev p) {
    __shared__ FwdShared<T, VEC, PACKED> sh;
    typedef typename Raw<T>::type raw;
    const int warp = threadIdx.x / 32;
    const Place at = place(p, &sh.slot);
    const Lane<VEC> ln(at.ch0, p.a.D);
    const long tile0 = at.pos * kFT, row0 = tile0 + warp * kFR;
    const long left = p.a.L - row0;
    const int live = left < 0 ? 0 : left < kFR ? (int)left : kFR;
    if (PACKED) map_rows(sh.rows, p.a, tile0);
    raw x[kFR], gr[kFR], gi[kFR];
#pragma unroll
    for (int j = 0; j < kFR; ++j) {
        const bool in = PACKED ? sh.rows.seq[warp * kFR + j] >= 0 : j < live;
        const bool k0 = in && ln.ok0, k1 = in && ln.ok1;
        gr[j] = Raw<T>::template load<VEC>(row_ptr<const T>(p.a.gate_r, at.b, row0 + j, ln.d), k0, k1);
        gi[j] = Raw<T>::template load<VEC>(row_ptr<const T>(p.a.gate_i, at.b, row0 + j, ln.d), k0, k1);
        x[j] = Raw<T>::template load<VEC>(row_ptr<const T>(p.a.x, at.b, row0 + j, ln.d), k0, k1);
    }
    const Rates rt = rates(ln.get(p.a.decay), p.a.scale);
    /* channels that do not exist have decay 0: their rate must not decide */
    const bool strong = (ln.ok0 && !(rt.rate.x <= kWeak)) || (ln.ok1 && !(rt.rate.y <= kWeak));
    if (__syncthreads_or(strong))
        fwd_tile<T, VEC, PACKED, false>(p, at, ln, rt, sh, x, gr, gi, row0, live);
    else
        fwd_tile<T, VEC, PACKED, true>(p, at, ln, rt, sh, x, gr, gi, row0, live);
    if (PACKED && at.pos == 0) empty_sequences(p.a, p.a.h0, p.a.h_last, at.ch0);
}

/* ------------------------------------------------------------------ */
/* backward                                                             */
/* ------------------------------------------------------------------ */

constexpr int kBR = 8, kBW = 8, kBT = kBR * kBW;
static_assert(kBT == kChunk, "a backward tile begins at a checkpoint");

template <typename T, bool VEC, bool PACKED>
struct BwdShared {
    float2 fagg[kBW][kC]; /* maps of the states */
    float2 agg[kBW][kC];  /* maps of the adjoint */
    float2 map[kWindow][kC];
    unsigned slot;
    RowMap<PACKED ? kBT : 1> rows;
};

/* The adjoint that reaches row t - 1 from row t is C_t = a_t (dy_t + C_{t+1}). */
template <typename T, bool VEC, bool PACKED, bool WEAK>
__device__ __forceinline__ void bwd_tile(const Dev &p, const Place &at, const Lane<VEC> &ln,
                                         const Rates &rt, BwdShared<T, VEC, PACKED> &sh,
                                         const typename Raw<T>::type (&x)[kBR],
                                         const typename Raw<T>::type (&gr)[kBR],
                                         const typename Raw<T>::type (&gi)[kBR],
                                         const typename Raw<T>::type (&dy)[kBR], long tile, long row0,
                                         int live) {
    const int warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const float2 zero = kmb_f2s(0.f), one = kmb_f2s(1.f);
    float2 c[kBR], q[kBR], in[kBR], si[kBR];
#pragma unroll
    for (int j = 0; j < kBR; ++j) {
        const Terms t = terms<WEAK>(Raw<T>::f(gr[j]), Raw<T>::f(gi[j]), rt);
        c[j] = t.c;
        q[j] = t.q;
        in[j] = t.i;
        si[j] = t.si;
    }
    float2 A = one, H = zero, K = zero;
    bool fresh = false, ends = false;
#pragma unroll
    for (int j = 0; j < kBR; ++j) {
        const int lr = warp * kBR + j;
        if (PACKED ? sh.rows.seq[lr] >= 0 : j < live) {
            if (PACKED && (sh.rows.edge[lr] & 1)) {
                H = ln.get(p.a.h0 ? p.a.h0 + sh.rows.seq[lr] * p.a.D : nullptr);
                fresh = true;
            }
            H = advance<WEAK>(c[j], H, kmb_mul2(si[j], Raw<T>::f(x[j])));
            A = shrink<WEAK>(c[j], A);
        }
    }
    sh.fagg[warp][ln.off] = kmb_f2(fresh ? -1.f : A.x, H.x);
    sh.fagg[warp][ln.off + Lane<VEC>::kNext] = kmb_f2(fresh ? -1.f : A.y, H.y);
#pragma unroll
    for (int j = kBR - 1; j >= 0; --j) {
        const int lr = warp * kBR + j;
        if (PACKED ? sh.rows.seq[lr] >= 0 : j < live) {
            if (PACKED && (sh.rows.edge[lr] & 2)) {
                K = ln.get(p.a.dh_last ? p.a.dh_last + sh.rows.seq[lr] * p.a.D : nullptr);
                ends = true;
            }
            K = shrink<WEAK>(c[j], kmb_add2(K, Raw<T>::f(dy[j])));
        }
    }
    sh.agg[warp][ln.off] = kmb_f2(ends ? -1.f : A.x, K.x);
    sh.agg[warp][ln.off + Lane<VEC>::kNext] = kmb_f2(ends ? -1.f : A.y, K.y);
    __syncthreads();

    /* the states before each row */
    float2 h = tile < p.chunks ? ln.get(p.ckpt_in + (at.b * p.chunks + tile) * p.a.D) : zero;
    for (int w = 0; w < warp; ++w) {
        const float2 m0 = sh.fagg[w][ln.off], m1 = sh.fagg[w][ln.off + Lane<VEC>::kNext];
        h = kmb_f2(apply(m0.x, m0.y, h.x), apply(m1.x, m1.y, h.y));
    }
    float2 hp[kBR];
#pragma unroll
    for (int j = 0; j < kBR; ++j) {
        const int lr = warp * kBR + j;
        if (PACKED && sh.rows.seq[lr] >= 0 && (sh.rows.edge[lr] & 1))
            h = ln.get(p.a.h0 ? p.a.h0 + sh.rows.seq[lr] * p.a.D : nullptr);
        hp[j] = h;
        h = advance<WEAK>(c[j], h, kmb_mul2(si[j], Raw<T>::f(x[j])));
    }

    const float *last = !PACKED && p.a.dh_last ? p.a.dh_last + at.b * p.a.D : nullptr;
    float2 C = enter_tile<VEC>(p, at, ln, sh.agg, sh.map, warps, true, last);
    for (int w = warps - 1; w > warp; --w) {
        const float2 m0 = sh.agg[w][ln.off], m1 = sh.agg[w][ln.off + Lane<VEC>::kNext];
        C = kmb_f2(apply(m0.x, m0.y, C.x), apply(m1.x, m1.y, C.y));
    }
    float2 sum = zero;
#pragma unroll
    for (int j = kBR - 1; j >= 0; --j) {
        const int lr = warp * kBR + j;
        if (PACKED ? sh.rows.seq[lr] >= 0 : j < live) {
            if (PACKED && (sh.rows.edge[lr] & 2))
                C = ln.get(p.a.dh_last ? p.a.dh_last + sh.rows.seq[lr] * p.a.D : nullptr);
            const float2 G = kmb_add2(C, Raw<T>::f(dy[j]));
            const float2 r = kmb_mul2(q[j], q[j]), u = kmb_mul2(rt.rate, r);
            const float2 b = kmb_mul2(si[j], Raw<T>::f(x[j]));
            float2 kappa = poly_kappa(u), ua;
            if (WEAK) {
                ua = kmb_fma2(neg2(c[j]), u, u);
            } else {
                /* e^-u is 0 long before u is 100 */
                ua = kmb_f2(u.x > 100.f ? 0.f : u.x * c[j].x, u.y > 100.f ? 0.f : u.y * c[j].y);
                kappa = kmb_f2(u.x <= kWeak ? kappa.x : ua.x * c[j].x * rcp_mufu(fmaf(-c[j].x, c[j].x, 1.f)),
                               u.y <= kWeak ? kappa.y : ua.y * c[j].y * rcp_mufu(fmaf(-c[j].y, c[j].y, 1.f)));
            }
            const float2 udu = kmb_mul2(G, kmb_fma2(neg2(ua), hp[j], kmb_mul2(kappa, b)));
            sum = kmb_add2(sum, udu);
            Raw<T>::template store<VEC>(row_ptr<T>(p.a.dx, at.b, row0 + j, ln.d), kmb_mul2(G, si[j]), ln.ok0,
                                        ln.ok1);
            Raw<T>::template store<VEC>(row_ptr<T>(p.a.dgate_r, at.b, row0 + j, ln.d),
                                        kmb_mul2(udu, sub2(one, r)), ln.ok0, ln.ok1);
            Raw<T>::template store<VEC>(row_ptr<T>(p.a.dgate_i, at.b, row0 + j, ln.d),
                                        kmb_mul2(kmb_mul2(G, b), sub2(one, in[j])), ln.ok0, ln.ok1);
            C = shrink<WEAK>(c[j], G);
            if (PACKED && (sh.rows.edge[lr] & 1) && p.a.dh0) ln.put(p.a.dh0 + sh.rows.seq[lr] * p.a.D, C);
        }
    }
    if (!PACKED && tile == 0 && warp == 0 && p.a.dh0) ln.put(p.a.dh0 + at.b * p.a.D, C);
    if (p.part) {
        __syncthreads(); /* every warp is done with the maps */
        sh.fagg[warp][ln.off].x = sum.x;
        sh.fagg[warp][ln.off + Lane<VEC>::kNext].x = sum.y;
        __syncthreads();
        for (int ch = threadIdx.x; ch < kC; ch += blockDim.x) {
            float v = 0.f;
            for (int w = 0; w < warps; ++w) v += sh.fagg[w][ch].x;
            p.part[at.pos * p.chains * kC + at.chain * kC + ch] = v;
        }
    }
}

template <typename T, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kBW * 32, 2) k_glr_bwd(const Dev p) {
    __shared__ BwdShared<T, VEC, PACKED> sh;
    typedef typename Raw<T>::type raw;
    const int warp = threadIdx.x / 32;
    const Place at = place(p, &sh.slot);
    const Lane<VEC> ln(at.ch0, p.a.D);
    const long tile = p.tiles - 1 - at.pos, tile0 = tile * kBT, row0 = tile0 + warp * kBR;
    const long left = p.a.L - row0;
    const int live = left < 0 ? 0 : left < kBR ? (int)left : kBR;
    if (PACKED) map_rows(sh.rows, p.a, tile0);
    raw x[kBR], gr[kBR], gi[kBR], dy[kBR];
#pragma unroll
    for (int j = 0; j < kBR; ++j) {
        const bool in = PACKED ? sh.rows.seq[warp * kBR + j] >= 0 : j < live;
        const bool k0 = in && ln.ok0, k1 = in && ln.ok1;
        gr[j] = Raw<T>::template load<VEC>(row_ptr<const T>(p.a.gate_r, at.b, row0 + j, ln.d), k0, k1);
        gi[j] = Raw<T>::template load<VEC>(row_ptr<const T>(p.a.gate_i, at.b, row0 + j, ln.d), k0, k1);
        x[j] = Raw<T>::template load<VEC>(row_ptr<const T>(p.a.x, at.b, row0 + j, ln.d), k0, k1);
        dy[j] = Raw<T>::template load<VEC>(row_ptr<const T>(p.a.dy, at.b, row0 + j, ln.d), k0, k1);
    }
    const Rates rt = rates(ln.get(p.a.decay), p.a.scale);
    const bool strong = (ln.ok0 && !(rt.rate.x <= kWeak)) || (ln.ok1 && !(rt.rate.y <= kWeak));
    if (__syncthreads_or(strong))
        bwd_tile<T, VEC, PACKED, false>(p, at, ln, rt, sh, x, gr, gi, dy, tile, row0, live);
    else
        bwd_tile<T, VEC, PACKED, true>(p, at, ln, rt, sh, x, gr, gi, dy, tile, row0, live);
    if (PACKED && tile == 0) empty_sequences(p.a, p.a.dh_last, p.a.dh0, at.ch0);
}

/* ddecay: the sums of all tiles and sequences, 32 columns a CTA, 32 rows of
 * threads, joined in a fixed order. */
__global__ void __launch_bounds__(1024) k_glr_ddecay(const float *part, long rows, long ld, long D,
                                                     const float *decay, float *ddecay, int acc) {
    __shared__ float s[32][33];
    const int tx = threadIdx.x, ty = threadIdx.y;
    const long d = (long)blockIdx.x * 32 + tx;
    float v = 0.f;
    if (d < D)
        for (long r = ty; r < rows; r += 32) v += part[r * ld + d];
    s[ty][tx] = v;
    __syncthreads();
    float t = s[tx][ty]; /* column ty, rows over the lanes */
#pragma unroll
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(~0u, t, o);
    const long e = (long)blockIdx.x * 32 + ty;
    if (tx == 0 && e < D) {
        t *= decay_ratio(decay[e]);
        ddecay[e] = acc ? ddecay[e] + t : t;
    }
}

/* L = 0: every sequence is empty */
__global__ void k_glr_copy(const float *from, float *to, long n) {
    for (long k = (long)blockIdx.x * blockDim.x + threadIdx.x; k < n; k += (long)gridDim.x * blockDim.x)
        to[k] = from ? from[k] : 0.f;
}

/* ------------------------------------------------------------------ */
/* one step                                                             */
/* ------------------------------------------------------------------ */

constexpr int kStepThreads = 128;

/* a row whose slot an earlier row names is left out */
template <typename T>
__global__ void __launch_bounds__(kStepThreads) k_glr_step(KmbGLRStep a, long tiles) {
    const long k = blockIdx.x / tiles;
    const long slot = a.slots ? a.slots[k] : k;
    if (slot < 0 || slot >= a.n_states) return;
    int taken = 0;
    if (a.slots)
        for (long j = threadIdx.x; j < k; j += kStepThreads) taken |= a.slots[j] == slot;
    if (__syncthreads_or(taken)) return;
    const long d = (blockIdx.x - k * tiles) * kStepThreads + threadIdx.x;
    if (d >= a.D) return;
    const float rate = a.scale * softplus(a.decay[d]);
    Rates rt;
    rt.rate = kmb_f2s(rate);
    rt.sroot = kmb_f2s(sqrtf(2.f * rate));
    const T *px = (const T *)a.x.data + k * a.x.row_stride + d;
    const T *pr = (const T *)a.gate_r.data + k * a.gate_r.row_stride + d;
    const T *pi = (const T *)a.gate_i.data + k * a.gate_i.row_stride + d;
    const float2 gr = kmb_f2s((float)*pr), gi = kmb_f2s((float)*pi), x = kmb_f2s((float)*px);
    float *s = a.state + slot * a.ld_state + d;
    float h = *s;
    if (rate <= kWeak) {
        const Terms t = terms<true>(gr, gi, rt);
        h = advance<true>(t.c, kmb_f2s(h), kmb_mul2(t.si, x)).x;
    } else {
        const Terms t = terms<false>(gr, gi, rt);
        h = advance<false>(t.c, kmb_f2s(h), kmb_mul2(t.si, x)).x;
    }
    *s = h;
    ((T *)a.y.data)[k * a.y.row_stride + d] = (T)h;
}

/* ------------------------------------------------------------------ */
/* launches                                                             */
/* ------------------------------------------------------------------ */

int done(const char *what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, what);
}

/* Whether the tensors allow two channels an access: even width, strides and
 * addresses. */
bool paired(const KmbGLR *a, const KmbRows *const *rows, int n) {
    const size_t es = a->type == KMB_BF16 ? 2 : 4;
    if (a->D % 2) return false;
    for (int i = 0; i < n; ++i) {
        const KmbRows *r = rows[i];
        if (!r->data) continue;
        if (((size_t)r->data / es) % 2 || r->row_stride % 2) return false;
        if (!a->offsets && a->batch > 1 && r->batch_stride % 2) return false;
    }
    return true;
}

struct Plan {
    long tiles, groups, batch, chains;
    size_t words; /* of each of the three shown arrays */
};

Plan plan(const KmbGLR *a, int rows) {
    Plan q;
    q.tiles = (a->L + rows - 1) / rows;
    if (a->offsets && q.tiles == 0) q.tiles = 1; /* for the empty sequences */
    q.groups = (a->D + kC - 1) / kC;
    q.batch = a->offsets ? 1 : a->batch;
    q.chains = q.groups * q.batch;
    q.words = q.tiles > 1 ? (size_t)q.tiles * q.chains * kC : 0;
    return q;
}

constexpr size_t kHead = 64; /* bytes before the shown arrays: the ticket */

size_t shown_bytes(const Plan &q) { return q.words ? kHead + 12 * q.words : 0; }

/* Fills the workspace's shown arrays and sets the pointers. */
int begin(Dev &d, const Plan &q, void *ws, cudaStream_t s) {
    if (q.tiles >= (1L << 31) / q.chains) return kmb_fail(KMB_EUNSUPPORTED, "glr: too many tiles");
    d.tiles = q.tiles;
    d.groups = q.groups;
    d.chains = q.chains;
    if (!q.words) return KMB_OK;
    const cudaError_t e = cudaMemsetAsync(ws, 0xff, shown_bytes(q), s);
    if (e != cudaSuccess) return kmb_cuda_fail(e, "glr: workspace fill");
    d.ticket = (unsigned *)ws;
    d.shown.A = (float *)((char *)ws + kHead);
    d.shown.H = d.shown.A + q.words;
    d.shown.end = d.shown.H + q.words;
    d.shown.step = q.chains * kC;
    return KMB_OK;
}

template <typename T>
int launch_fwd(const Dev &d, const Plan &q, bool vec, cudaStream_t s) {
    const long n = q.tiles * q.chains;
    const long runs = (d.a.L + kFR - 1) / kFR;
    const unsigned threads = 32u * (unsigned)(runs < 1 ? 1 : runs < kFW ? runs : kFW);
    if (d.a.offsets) {
        if (vec) k_glr_fwd<T, true, true><<<(unsigned)n, threads, 0, s>>>(d);
        else k_glr_fwd<T, false, true><<<(unsigned)n, threads, 0, s>>>(d);
    } else {
        if (vec) k_glr_fwd<T, true, false><<<(unsigned)n, threads, 0, s>>>(d);
        else k_glr_fwd<T, false, false><<<(unsigned)n, threads, 0, s>>>(d);
    }
    return done("glr: forward launch");
}

template <typename T>
int launch_bwd(const Dev &d, const Plan &q, bool vec, cudaStream_t s) {
    const long n = q.tiles * q.chains;
    const long runs = (d.a.L + kBR - 1) / kBR;
    const unsigned threads = 32u * (unsigned)(runs < 1 ? 1 : runs < kBW ? runs : kBW);
    if (d.a.offsets) {
        if (vec) k_glr_bwd<T, true, true><<<(unsigned)n, threads, 0, s>>>(d);
        else k_glr_bwd<T, false, true><<<(unsigned)n, threads, 0, s>>>(d);
    } else {
        if (vec) k_glr_bwd<T, true, false><<<(unsigned)n, threads, 0, s>>>(d);
        else k_glr_bwd<T, false, false><<<(unsigned)n, threads, 0, s>>>(d);
    }
    return done("glr: backward launch");
}

int run_fwd(const KmbGLR *a, float *ckpt, bool write_y, void *ws, cudaStream_t s) {
    const Plan q = plan(a, kFT);
    Dev d = {};
    d.a = *a;
    if (!write_y) {
        d.states_only = 1;
        d.a.y.data = nullptr;
        d.a.h_last = nullptr;
    }
    if (a->offsets)
        d.a.x.batch_stride = d.a.gate_r.batch_stride = d.a.gate_i.batch_stride = d.a.y.batch_stride = 0;
    d.ckpt_out = ckpt;
    d.chunks = (a->L + kChunk - 1) / kChunk;
    const int rc = begin(d, q, ws, s);
    if (rc) return rc;
    const KmbRows *rows[] = {&d.a.x, &d.a.gate_r, &d.a.gate_i, &d.a.y};
    const bool vec = paired(&d.a, rows, 4);
    return a->type == KMB_BF16 ? launch_fwd<__nv_bfloat16>(d, q, vec, s) : launch_fwd<float>(d, q, vec, s);
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

} // namespace

/* Backward workspace: shown arrays (the state run and the adjoint use them
 * one after the other) | sums of the tiles | checkpoints. */
extern "C" size_t kmb_glr_scratch_bytes(const KmbGLR *a, int bwd) {
    if (a->batch == 0 || (a->L == 0 && !a->offsets)) return 0;
    const size_t f = shown_bytes(plan(a, kFT));
    if (!bwd) return f;
    const Plan q = plan(a, kBT);
    const size_t b = shown_bytes(q);
    size_t n = align16(a->ckpt || f < b ? b : f);
    if (a->ddecay) n += align16(4 * (size_t)q.tiles * q.chains * kC);
    if (!a->ckpt) n += align16(4 * (size_t)kmb_glr_ckpt_elems(a));
    return n;
}

extern "C" int kmb_launch_glr_fwd(const KmbGLR *a, cudaStream_t s) {
    if (a->batch == 0) return KMB_OK;
    if (a->L == 0 && !a->offsets) {
        if (a->h_last) k_glr_copy<<<148, 256, 0, s>>>(a->h0, a->h_last, a->batch * a->D);
        return done("glr: forward launch");
    }
    return run_fwd(a, a->ckpt, true, a->workspace, s);
}

extern "C" int kmb_launch_glr_bwd(const KmbGLR *a, cudaStream_t s) {
    if (a->batch == 0 || (a->L == 0 && !a->offsets)) {
        if (a->batch && a->dh0) k_glr_copy<<<148, 256, 0, s>>>(a->dh_last, a->dh0, a->batch * a->D);
        if (a->ddecay)
            k_glr_ddecay<<<(unsigned)((a->D + 31) / 32), dim3(32, 32), 0, s>>>(nullptr, 0, 0, a->D, a->decay,
                                                                            a->ddecay, a->accumulate);
        return done("glr: backward launch");
    }
    const Plan q = plan(a, kBT);
    const size_t f = shown_bytes(plan(a, kFT)), b = shown_bytes(q);
    char *ws = (char *)a->workspace;
    size_t o = align16(a->ckpt || f < b ? b : f);
    Dev d = {};
    d.a = *a;
    if (a->offsets)
        d.a.x.batch_stride = d.a.gate_r.batch_stride = d.a.gate_i.batch_stride = d.a.dy.batch_stride =
            d.a.dx.batch_stride = d.a.dgate_r.batch_stride = d.a.dgate_i.batch_stride = 0;
    if (a->ddecay) {
        d.part = (float *)(ws + o);
        o += align16(4 * (size_t)q.tiles * q.chains * kC);
    }
    d.ckpt_in = a->ckpt;
    d.chunks = (a->L + kChunk - 1) / kChunk;
    int rc;
    if (!a->ckpt) {
        d.ckpt_in = (float *)(ws + o);
        if (a->L && (rc = run_fwd(a, (float *)(ws + o), false, ws, s))) return rc;
    }
    if ((rc = begin(d, q, ws, s))) return rc;
    const KmbRows *rows[] = {&d.a.x, &d.a.gate_r, &d.a.gate_i, &d.a.dy, &d.a.dx, &d.a.dgate_r, &d.a.dgate_i};
    const bool vec = paired(&d.a, rows, 7);
    rc = a->type == KMB_BF16 ? launch_bwd<__nv_bfloat16>(d, q, vec, s) : launch_bwd<float>(d, q, vec, s);
    if (rc || !a->ddecay) return rc;
    k_glr_ddecay<<<(unsigned)((a->D + 31) / 32), dim3(32, 32), 0, s>>>(
        d.part, q.tiles * q.batch, q.groups * kC, a->D, a->decay, a->ddecay, a->accumulate);
    return done("glr: backward launch");
}

extern "C" int kmb_launch_glr_step(const KmbGLRStep *a, cudaStream_t s) {
    const long tiles = (a->D + kStepThreads - 1) / kStepThreads;
    if (a->rows >= (1L << 31) / tiles) return kmb_fail(KMB_EUNSUPPORTED, "glr: too many rows");
    const unsigned n = (unsigned)(a->rows * tiles);
    if (a->type == KMB_BF16)
        k_glr_step<__nv_bfloat16><<<n, kStepThreads, 0, s>>>(*a, tiles);
    else
        k_glr_step<float><<<n, kStepThreads, 0, s>>>(*a, tiles);
    return done("glr: step launch");
}

/* KMB_ETIMEOUT (and the word cleared) when a wait between tiles gave up
 * since the last check. */
extern "C" int kmb_glr_check_error(void) {
    int flag = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&flag, g_glr_error, sizeof flag);
    if (e != cudaSuccess) return kmb_cuda_fail(e, "glr: error word");
    if (flag) {
        const int zero = 0;
        (void)cudaMemcpyToSymbol(g_glr_error, &zero, sizeof zero);
        return kmb_fail(KMB_ETIMEOUT, "glr: a wait for another tile's state expired");
    }
    return KMB_OK;
}
