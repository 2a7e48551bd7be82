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
 * 128 channels: a warp owns a run of consecutive rows, a lane four channels.
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
constexpr int kV = 4;       /* channels of a lane */
constexpr int kC = 32 * kV; /* channels of a tile */
constexpr int kWindow = 12; /* tiles before its own that a tile looks at */
constexpr unsigned kUnset = 0xffffffffu; /* workspace word not written yet */

/* set when a wait for another tile's state gave up (kmb_glr_check_error) */
__device__ int g_glr_error;

/* ------------------------------------------------------------------ */
/* four channels of one row, as two FFMA2 pairs                          */
/* ------------------------------------------------------------------ */

struct F4 {
    float2 l, h;
};
__device__ __forceinline__ F4 f4s(float v) { return {kmb_f2s(v), kmb_f2s(v)}; }
__device__ __forceinline__ F4 f4(float4 v) { return {kmb_f2(v.x, v.y), kmb_f2(v.z, v.w)}; }
__device__ __forceinline__ float4 v4(F4 a) { return make_float4(a.l.x, a.l.y, a.h.x, a.h.y); }
__device__ __forceinline__ F4 operator+(F4 a, F4 b) { return {kmb_add2(a.l, b.l), kmb_add2(a.h, b.h)}; }
__device__ __forceinline__ F4 operator*(F4 a, F4 b) { return {kmb_mul2(a.l, b.l), kmb_mul2(a.h, b.h)}; }
__device__ __forceinline__ F4 fma4(F4 a, F4 b, F4 c) {
    return {kmb_fma2(a.l, b.l, c.l), kmb_fma2(a.h, b.h, c.h)};
}
template <typename Fn>
__device__ __forceinline__ F4 each(Fn f) { /* f(channel) */
    return {kmb_f2(f(0), f(1)), kmb_f2(f(2), f(3))};
}
__device__ __forceinline__ float get(const F4 &a, int k) {
    return k == 0 ? a.l.x : k == 1 ? a.l.y : k == 2 ? a.h.x : a.h.y;
}

/* VEC: channels 4 lane .. 4 lane + 3 in one access; else lane + 32 k, for
 * odd widths, strides and addresses (every access still covers a contiguous
 * piece of the row).  m: bit k set where channel k exists. */
template <typename T>
struct Raw;
template <>
struct Raw<float> {
    typedef float4 type;
    static __device__ __forceinline__ F4 f(float4 v) { return f4(v); }
    template <bool VEC>
    static __device__ __forceinline__ float4 load(const float *p, unsigned m) {
        if (VEC) return m ? __ldcs(reinterpret_cast<const float4 *>(p)) : make_float4(0.f, 0.f, 0.f, 0.f);
        return make_float4(m & 1 ? __ldcs(p) : 0.f, m & 2 ? __ldcs(p + 32) : 0.f,
                           m & 4 ? __ldcs(p + 64) : 0.f, m & 8 ? __ldcs(p + 96) : 0.f);
    }
    template <bool VEC>
    static __device__ __forceinline__ void store(float *p, F4 v, unsigned m) {
        if (VEC) {
            if (m) __stcs(reinterpret_cast<float4 *>(p), v4(v));
            return;
        }
        if (m & 1) __stcs(p, v.l.x);
        if (m & 2) __stcs(p + 32, v.l.y);
        if (m & 4) __stcs(p + 64, v.h.x);
        if (m & 8) __stcs(p + 96, v.h.y);
    }
};
template <>
struct Raw<__nv_bfloat16> {
    typedef uint2 type; /* the even channels in the low halves */
    static __device__ __forceinline__ F4 f(uint2 v) {
        return {kmb_f2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u)),
                kmb_f2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u))};
    }
    static __device__ __forceinline__ unsigned pack(float2 v) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
        return *reinterpret_cast<const unsigned *>(&h);
    }
    template <bool VEC>
    static __device__ __forceinline__ uint2 load(const __nv_bfloat16 *p, unsigned m) {
        if (VEC) return m ? __ldcs(reinterpret_cast<const uint2 *>(p)) : make_uint2(0u, 0u);
        const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
        const unsigned a = m & 1 ? __ldcs(q) : 0u, b = m & 2 ? __ldcs(q + 32) : 0u;
        const unsigned c = m & 4 ? __ldcs(q + 64) : 0u, d = m & 8 ? __ldcs(q + 96) : 0u;
        return make_uint2(a | b << 16, c | d << 16);
    }
    template <bool VEC>
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, F4 v, unsigned m) {
        const uint2 u = make_uint2(pack(v.l), pack(v.h));
        if (VEC) {
            if (m) __stcs(reinterpret_cast<uint2 *>(p), u);
            return;
        }
        unsigned short *q = reinterpret_cast<unsigned short *>(p);
        if (m & 1) __stcs(q, (unsigned short)u.x);
        if (m & 2) __stcs(q + 32, (unsigned short)(u.x >> 16));
        if (m & 4) __stcs(q + 64, (unsigned short)u.y);
        if (m & 8) __stcs(q + 96, (unsigned short)(u.y >> 16));
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
 *   (e^-u - 1) / u                    2.9e-9 in real arithmetic
 *   sqrt((1 - e^-2u) / (2 u))         4.8e-9
 *   kappa = u / (e^2u - 1)            3.4e-9
 * A channel whose rate is at most kWeak needs no exponential of u, no
 * square root and no cancelling 1 - a^2, and its recurrence runs on a - 1
 * as h + (b + (a - 1) h): a memory of 1 / (1 - a) steps multiplies the error
 * of the decay, and a itself, next to 1, cannot hold it to more than
 * 2^-25 / (1 - a).
 */
constexpr float kWeak = 0.25f;

__device__ __forceinline__ F4 poly4(F4 u, float c0, float c1, float c2, float c3, float c4) {
    F4 p = fma4(f4s(c4), u, f4s(c3));
    p = fma4(p, u, f4s(c2));
    p = fma4(p, u, f4s(c1));
    return fma4(p, u, f4s(c0));
}
__device__ __forceinline__ F4 poly_expm1(F4 u) {
    return poly4(u, -1.f, 0.49999964237213135f, -0.1666528880596161f, 0.04150013253092766f,
                 -0.007530174218118191f);
}
__device__ __forceinline__ F4 poly_root(F4 u) {
    return poly4(u, 1.f, -0.49999940395355225f, 0.20831027626991272f, -0.06222091242671013f,
                 0.01236682292073965f);
}
__device__ __forceinline__ F4 poly_kappa(F4 u) {
    return poly4(u, 0.5f, -0.5000002980232239f, 0.1666753739118576f, -8.377274934900925e-05f,
                 -0.010830916464328766f);
}

/* Per channel: rate, and sqrt(2 rate) for root = sqrt(2 u) sqrt((1 - e^-2u) / 2u). */
struct Rates {
    F4 rate, sroot;
};

/* Of one row: c is a - 1 (WEAK) or a, q = sqrt(r) = (1 + e^-gate_r)^-1/2, i,
 * and si = root i. */
struct Terms {
    F4 c, q, i, si;
};

template <bool WEAK>
__device__ __forceinline__ Terms terms(F4 gr, F4 gi, const Rates &k) {
    Terms t;
    const F4 nl = f4s(-KMB_LOG2E), one = f4s(1.f);
    gr = gr * nl;
    gi = gi * nl;
    const F4 er = each([&](int n) { return kmb_ex2(get(gr, n)); }) + one;
    const F4 ei = each([&](int n) { return kmb_ex2(get(gi, n)); }) + one;
    t.q = each([&](int n) { return rsqrt_mufu(get(er, n)); });
    t.i = each([&](int n) { return rcp_mufu(get(ei, n)); });
    const F4 u = k.rate * (t.q * t.q);
    const F4 m = u * poly_expm1(u);
    F4 root = k.sroot * t.q * poly_root(u);
    if (WEAK) {
        t.c = m;
    } else {
        const F4 un = u * nl;
        const F4 e = each([&](int n) { return kmb_ex2(get(un, n)); });
        t.c = each([&](int n) { return get(u, n) <= kWeak ? 1.f + get(m, n) : get(e, n); });
        root = each([&](int n) {
            return get(u, n) <= kWeak ? get(root, n) : sqrt_mufu(fmaf(-get(e, n), get(e, n), 1.f));
        });
    }
    t.si = root * t.i;
    return t;
}

/* a h + b */
template <bool WEAK>
__device__ __forceinline__ F4 advance(F4 c, F4 h, F4 b) {
    return WEAK ? h + fma4(c, h, b) : fma4(c, h, b);
}
/* a A */
template <bool WEAK>
__device__ __forceinline__ F4 shrink(F4 c, F4 A) {
    return WEAK ? fma4(c, A, A) : c * A;
}

/* ------------------------------------------------------------------ */
/* affine maps h -> A h + H; A = -1 marks a constant one                 */
/* ------------------------------------------------------------------ */

struct Map {
    F4 A, H;
};

/* MARKED: constant maps occur (a sequence began inside, a final state) */
template <bool MARKED>
__device__ __forceinline__ F4 apply(const Map &m, F4 h) {
    const F4 r = fma4(m.A, h, m.H);
    if (!MARKED) return r;
    return each([&](int n) { return get(m.A, n) < 0.f ? get(m.H, n) : get(r, n); });
}

/* the map of `first` then `then` */
template <bool MARKED>
__device__ __forceinline__ Map join(const Map &first, const Map &then) {
    Map r;
    r.H = apply<MARKED>(then, first.H);
    r.A = first.A * then.A;
    if (MARKED)
        r.A = each([&](int n) { return get(first.A, n) < 0.f || get(then.A, n) < 0.f ? -1.f : get(r.A, n); });
    return r;
}

/* What tiles show one another: [place in the chain][chain][lane] of four
 * channels.  Every word is written once, and was kUnset (the workspace is
 * filled at the start of the call): a word that is not kUnset is the value
 * itself, so no fence orders flags against data. */
struct Shown {
    float4 *A, *H, *end; /* map, final state */
    long step;           /* entries between places of a chain */
};

__device__ __forceinline__ bool peek(const float4 *p, F4 &v) {
    unsigned a, b, c, d;
    asm volatile("ld.relaxed.gpu.global.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
                 : "l"(p)
                 : "memory");
    v = {kmb_f2(__uint_as_float(a), __uint_as_float(b)), kmb_f2(__uint_as_float(c), __uint_as_float(d))};
    return a != kUnset && b != kUnset && c != kUnset && d != kUnset;
}
__device__ __forceinline__ float not_unset(float v) {
    return __float_as_uint(v) == kUnset ? __uint_as_float(0x7fffffffu) : v;
}
__device__ __forceinline__ void show(float4 *p, F4 v) {
    asm volatile("st.relaxed.gpu.global.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(not_unset(v.l.x)),
                 "f"(not_unset(v.l.y)), "f"(not_unset(v.h.x)), "f"(not_unset(v.h.y))
                 : "memory");
}

/* The map of a place, or as a constant one its final state: waits for
 * whichever comes first (last: for the final state).  Bounded by about 2^31
 * cycles; then the error word is set and later waits return at once. */
__device__ __forceinline__ Map look(const Shown &s, long o, bool last) {
    const long long t0 = clock64();
    Map m;
    for (int n = 0;; ++n) {
        if (peek(s.end + o, m.H)) {
            m.A = f4s(-1.f);
            return m;
        }
        if (!last && peek(s.A + o, m.A) && peek(s.H + o, m.H)) return m;
        if ((n & 63) == 63) {
            const bool late = clock64() - t0 > (1ll << 31);
            if (late) atomicExch(&g_glr_error, 1);
            if (late || *reinterpret_cast<volatile int *>(&g_glr_error)) {
                m.A = f4s(-1.f);
                m.H = f4s(0.f);
                return m;
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
    float *part;                /* [tiles * batch][groups * kC] sums of u dL/du */
    unsigned *ticket;
    Shown shown;
};

struct Place {
    long pos, chain, b, ch0; /* place in the chain, chain, sequence (0 when packed), first channel */
};

/* Tiles are taken in the order of their places: a tile waits only for tiles
 * that another CTA has taken before. */
__device__ __forceinline__ Place place(const Dev &p, unsigned *slot) {
    if (p.tiles > 1) {
        if (threadIdx.x == 0) *slot = atomicAdd(p.ticket, 1u) + 1u; /* the fill makes it -1 */
        __syncthreads();
    }
    const unsigned id = p.tiles > 1 ? *slot : blockIdx.x;
    Place t;
    const unsigned pos = id / (unsigned)p.chains, chain = id - pos * (unsigned)p.chains;
    const unsigned b = chain / (unsigned)p.groups;
    t.pos = pos;
    t.chain = chain;
    t.b = b;
    t.ch0 = (long)(chain - b * (unsigned)p.groups) * kC;
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
                m.edge[r - row0] = (unsigned char)((r == (lo < 0 ? 0 : lo) ? 1 : 0) |
                                                   (r == (hi > a.L ? a.L : hi) - 1 ? 2 : 0));
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

/* The lane's channels: the first, and which exist. */
template <bool VEC>
struct Lane {
    long d;
    unsigned m;
    int lane;
    static constexpr int kNext = VEC ? 1 : 32; /* to the next channel */
    __device__ __forceinline__ Lane(long ch0, long D) {
        lane = threadIdx.x % 32;
        d = ch0 + (VEC ? kV * lane : lane);
        m = 0;
#pragma unroll
        for (int k = 0; k < kV; ++k) m |= d + k * kNext < D ? 1u << k : 0u;
    }
    /* a [.., D] fp32 vector at the channels, 0 where NULL */
    __device__ __forceinline__ F4 at(const float *p) const {
        return each([&](int k) { return p && (m >> k & 1) ? p[d + k * kNext] : 0.f; });
    }
    __device__ __forceinline__ void put(float *p, F4 v) const {
#pragma unroll
        for (int k = 0; k < kV; ++k)
            if (p && (m >> k & 1)) p[d + k * kNext] = get(v, k);
    }
};

/* A tensor's rows of the run: pointer to the lane's channels of row j. */
template <typename T, bool VEC>
struct Run {
    T *p;
    long step;
    __device__ __forceinline__ Run(const KmbRows &r, long b, long row, const Lane<VEC> &ln) {
        p = (T *)r.data + b * r.batch_stride + row * r.row_stride + ln.d;
        step = r.row_stride;
    }
    __device__ __forceinline__ T *operator[](int j) const { return p + j * step; }
};

/* The channels' rates, one thread a channel, and whether one of them is
 * above kWeak.  Ends with a barrier. */
template <bool VEC>
__device__ __forceinline__ bool make_rates(const KmbGLR &a, long ch0, float *rate, float *sroot) {
    bool strong = false;
    for (int c = threadIdx.x; c < kC; c += blockDim.x) {
        const int k = VEC ? c : (c % 32) * kV + c / 32; /* its place in the lanes' order */
        float r = 0.f;
        if (ch0 + c < a.D) {
            r = a.scale * softplus(a.decay[ch0 + c]);
            strong |= !(r <= kWeak);
        }
        rate[k] = r;
        sroot[k] = sqrtf(2.f * r);
    }
    return __syncthreads_or(strong);
}

/* Maps of the warps of a tile. */
template <int W>
struct Maps {
    float4 A[W][32], H[W][32];
    __device__ __forceinline__ void put(int w, int lane, F4 a, F4 h) {
        A[w][lane] = v4(a);
        H[w][lane] = v4(h);
    }
    __device__ __forceinline__ Map at(int w, int lane) const { return {f4(A[w][lane]), f4(H[w][lane])}; }
};

/* Joins the tile with the ones before it in its chain and returns the state
 * that enters it.  agg: the warps' maps, joined from the last when reverse;
 * first: the state that enters the chain. */
template <bool VEC, bool MARKED, bool REVERSE, int W>
__device__ __forceinline__ F4 enter_tile(const Dev &p, const Place &at, const Lane<VEC> &ln,
                                         const Maps<W> &agg, Maps<kWindow> &seen, const float *first) {
    const int warp = threadIdx.x / 32, warps = blockDim.x / 32;
    F4 h = ln.at(first);
    if (p.tiles == 1) return h;
    Shown s = p.shown;
    const long o = at.pos * s.step + at.chain * 32 + ln.lane;
    Map m = {f4s(1.f), f4s(0.f)};
    if (warp == 0 && at.pos + 1 < p.tiles) {
        for (int k = 0; k < warps; ++k) m = join<MARKED>(m, agg.at(REVERSE ? warps - 1 - k : k, ln.lane));
        if (at.pos > 0) {
            show(s.A + o, m.A);
            show(s.H + o, m.H);
        }
    }
    if (at.pos > 0) {
        const int n = at.pos < kWindow ? (int)at.pos : kWindow;
        for (int k = warp; k < n; k += warps) {
            const Map v = look(s, o - (k + 1) * s.step, k == kWindow - 1);
            seen.put(k, ln.lane, v.A, v.H);
        }
        __syncthreads();
        /* from the nearest final states on */
        int k = 0;
        for (; k < n - 1; ++k) {
            const float4 A = seen.A[k][ln.lane];
            if (A.x < 0.f && A.y < 0.f && A.z < 0.f && A.w < 0.f) break;
        }
        for (; k >= 0; --k) h = apply<true>(seen.at(k, ln.lane), h);
    }
    if (warp == 0 && at.pos + 1 < p.tiles) show(s.end + o, apply<MARKED>(m, h));
    return h;
}

/* ------------------------------------------------------------------ */
/* forward                                                              */
/* ------------------------------------------------------------------ */

constexpr int kFR = 8;         /* rows of a warp */
constexpr int kFW = 8;         /* warps of a full CTA */
constexpr int kFT = kFR * kFW; /* rows of a tile */
static_assert(kFT % kChunk == 0 || kChunk % kFT == 0, "checkpoints lie at the beginning of a run");

template <bool PACKED>
struct FwdShared {
    Maps<kFW> agg;
    Maps<kWindow> seen;
    float4 rate[32], sroot[32];
    unsigned slot;
    RowMap<PACKED ? kFT : 1> rows;
};

template <typename T, bool VEC, bool PACKED, bool WEAK>
__device__ __forceinline__ void fwd_tile(const Dev &p, const Place &at, const Lane<VEC> &ln,
                                         FwdShared<PACKED> &sh, const typename Raw<T>::type (&x)[kFR],
                                         const typename Raw<T>::type (&gr)[kFR],
                                         const typename Raw<T>::type (&gi)[kFR], long row0, int live) {
    const int warp = threadIdx.x / 32;
    F4 c[kFR], b[kFR];
    {
        const Rates rt = {f4(sh.rate[ln.lane]), f4(sh.sroot[ln.lane])};
#pragma unroll
        for (int j = 0; j < kFR; ++j) {
            const Terms t = terms<WEAK>(Raw<T>::f(gr[j]), Raw<T>::f(gi[j]), rt);
            c[j] = t.c;
            b[j] = t.si * Raw<T>::f(x[j]);
        }
    }
    const auto in = [&](int j) { return PACKED ? sh.rows.seq[warp * kFR + j] >= 0 : j < live; };
    const auto begins = [&](int j) { return PACKED && (sh.rows.edge[warp * kFR + j] & 1); };
    const auto h0 = [&](int j) { return ln.at(p.a.h0 ? p.a.h0 + sh.rows.seq[warp * kFR + j] * p.a.D : nullptr); };
    F4 A = f4s(1.f), H = f4s(0.f);
    bool fresh = false; /* a sequence begins in this run */
#pragma unroll
    for (int j = 0; j < kFR; ++j) {
        if (in(j)) {
            if (begins(j)) {
                H = h0(j);
                fresh = true;
            }
            H = advance<WEAK>(c[j], H, b[j]);
            A = shrink<WEAK>(c[j], A);
        }
    }
    sh.agg.put(warp, ln.lane, fresh ? f4s(-1.f) : A, H);
    __syncthreads();
    const float *first = !PACKED && p.a.h0 ? p.a.h0 + at.b * p.a.D : nullptr;
    F4 h = enter_tile<VEC, PACKED, false>(p, at, ln, sh.agg, sh.seen, first);
    for (int w = 0; w < warp; ++w) h = apply<PACKED>(sh.agg.at(w, ln.lane), h);
    if (p.ckpt_out && row0 % kChunk == 0 && row0 < p.a.L)
        ln.put(p.ckpt_out + (at.b * p.chunks + row0 / kChunk) * p.a.D, h);
    const Run<T, VEC> y(p.a.y, at.b, row0, ln);
#pragma unroll
    for (int j = 0; j < kFR; ++j) {
        if (in(j)) {
            if (begins(j)) h = h0(j);
            h = advance<WEAK>(c[j], h, b[j]);
            if (!p.states_only) Raw<T>::template store<VEC>(y[j], h, ln.m);
            if (PACKED && (sh.rows.edge[warp * kFR + j] & 2) && p.a.h_last)
                ln.put(p.a.h_last + sh.rows.seq[warp * kFR + j] * p.a.D, h);
        }
    }
    if (!PACKED && p.a.h_last && live > 0 && row0 + live == p.a.L) ln.put(p.a.h_last + at.b * p.a.D, h);
}

template <typename T, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kFW * 32, 2) k_glr_fwd(const __grid_constant__ Dev p) {
    __shared__ FwdShared<PACKED> sh;
    typedef typename Raw<T>::type raw;
    const int warp = threadIdx.x / 32;
    const Place at = place(p, &sh.slot);
    const Lane<VEC> ln(at.ch0, p.a.D);
    const long tile0 = at.pos * kFT, row0 = tile0 + warp * kFR;
    const long left = p.a.L - row0;
    const int live = left < 0 ? 0 : left < kFR ? (int)left : kFR;
    if (PACKED) map_rows(sh.rows, p.a, tile0);
    raw x[kFR], gr[kFR], gi[kFR];
    {
        const Run<const T, VEC> pr(p.a.gate_r, at.b, row0, ln), pi(p.a.gate_i, at.b, row0, ln),
            px(p.a.x, at.b, row0, ln);
#pragma unroll
        for (int j = 0; j < kFR; ++j) {
            const unsigned m = (PACKED ? sh.rows.seq[warp * kFR + j] >= 0 : j < live) ? ln.m : 0u;
            gr[j] = Raw<T>::template load<VEC>(pr[j], m);
            gi[j] = Raw<T>::template load<VEC>(pi[j], m);
            x[j] = Raw<T>::template load<VEC>(px[j], m);
        }
    }
    if (make_rates<VEC>(p.a, at.ch0, (float *)sh.rate, (float *)sh.sroot))
        fwd_tile<T, VEC, PACKED, false>(p, at, ln, sh, x, gr, gi, row0, live);
    else
        fwd_tile<T, VEC, PACKED, true>(p, at, ln, sh, x, gr, gi, row0, live);
    if (PACKED && at.pos == 0) empty_sequences(p.a, p.a.h0, p.a.h_last, at.ch0);
}

/* ------------------------------------------------------------------ */
/* backward                                                             */
/* ------------------------------------------------------------------ */

constexpr int kBR = 4, kBW = 16, kBT = kBR * kBW;
static_assert(kBT == kChunk, "a backward tile begins at a checkpoint");

template <bool PACKED>
struct BwdShared {
    Maps<kBW> states, agg; /* the warps' maps of the states and of the adjoint */
    Maps<kWindow> seen;
    float4 rate[32], sroot[32];
    unsigned slot;
    RowMap<PACKED ? kBT : 1> rows;
};

/* The adjoint that reaches row t - 1 from row t is C_t = a_t (dy_t + C_{t+1}). */
template <typename T, bool VEC, bool PACKED, bool WEAK>
__device__ __forceinline__ void bwd_tile(const Dev &p, const Place &at, const Lane<VEC> &ln,
                                         BwdShared<PACKED> &sh, const typename Raw<T>::type (&x)[kBR],
                                         const typename Raw<T>::type (&gr)[kBR],
                                         const typename Raw<T>::type (&gi)[kBR],
                                         const typename Raw<T>::type (&dy)[kBR], long tile, long row0,
                                         int live) {
    const int warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const F4 zero = f4s(0.f), one = f4s(1.f), minus = f4s(-1.f);
    Terms t[kBR];
    {
        const Rates rt = {f4(sh.rate[ln.lane]), f4(sh.sroot[ln.lane])};
#pragma unroll
        for (int j = 0; j < kBR; ++j) t[j] = terms<WEAK>(Raw<T>::f(gr[j]), Raw<T>::f(gi[j]), rt);
    }
    const auto in = [&](int j) { return PACKED ? sh.rows.seq[warp * kBR + j] >= 0 : j < live; };
    const auto begins = [&](int j) { return PACKED && (sh.rows.edge[warp * kBR + j] & 1); };
    const auto ends = [&](int j) { return PACKED && (sh.rows.edge[warp * kBR + j] & 2); };
    const auto of = [&](const float *v, int j) { return ln.at(v ? v + sh.rows.seq[warp * kBR + j] * p.a.D : nullptr); };
    F4 A = one, H = zero, K = zero;
    bool fresh = false, closed = false;
#pragma unroll
    for (int j = 0; j < kBR; ++j) {
        if (in(j)) {
            if (begins(j)) {
                H = of(p.a.h0, j);
                fresh = true;
            }
            H = advance<WEAK>(t[j].c, H, t[j].si * Raw<T>::f(x[j]));
            A = shrink<WEAK>(t[j].c, A);
        }
    }
    sh.states.put(warp, ln.lane, fresh ? minus : A, H);
#pragma unroll
    for (int j = kBR - 1; j >= 0; --j) {
        if (in(j)) {
            if (ends(j)) {
                K = of(p.a.dh_last, j);
                closed = true;
            }
            K = shrink<WEAK>(t[j].c, K + Raw<T>::f(dy[j]));
        }
    }
    sh.agg.put(warp, ln.lane, closed ? minus : A, K);
    __syncthreads();

    const float *last = !PACKED && p.a.dh_last ? p.a.dh_last + at.b * p.a.D : nullptr;
    F4 C = enter_tile<VEC, PACKED, true>(p, at, ln, sh.agg, sh.seen, last);
    for (int w = warps - 1; w > warp; --w) C = apply<PACKED>(sh.agg.at(w, ln.lane), C);

    /* the states before each row */
    F4 hp[kBR];
    {
        F4 h = tile < p.chunks ? ln.at(p.ckpt_in + (at.b * p.chunks + tile) * p.a.D) : zero;
        for (int w = 0; w < warp; ++w) h = apply<PACKED>(sh.states.at(w, ln.lane), h);
#pragma unroll
        for (int j = 0; j < kBR; ++j) {
            if (begins(j)) h = of(p.a.h0, j);
            hp[j] = h;
            h = advance<WEAK>(t[j].c, h, t[j].si * Raw<T>::f(x[j]));
        }
    }
    F4 sum = zero;
    const F4 rate = f4(sh.rate[ln.lane]);
    const Run<T, VEC> dx(p.a.dx, at.b, row0, ln), dgr(p.a.dgate_r, at.b, row0, ln), dgi(p.a.dgate_i, at.b, row0, ln);
#pragma unroll
    for (int j = kBR - 1; j >= 0; --j) {
        if (in(j)) {
            if (ends(j)) C = of(p.a.dh_last, j);
            const F4 c = t[j].c, G = C + Raw<T>::f(dy[j]);
            const F4 r = t[j].q * t[j].q, u = rate * r, b = t[j].si * Raw<T>::f(x[j]);
            F4 kappa = poly_kappa(u), ua; /* ua: -u a */
            if (WEAK) {
                ua = fma4(c, u, u) * minus;
            } else {
                /* e^-u is 0 long before u is 100 */
                ua = each([&](int n) { return get(u, n) > 100.f ? 0.f : -get(u, n) * get(c, n); });
                kappa = each([&](int n) {
                    const float a = get(c, n);
                    return get(u, n) <= kWeak ? get(kappa, n) : -get(ua, n) * a * rcp_mufu(fmaf(-a, a, 1.f));
                });
            }
            const F4 udu = G * fma4(ua, hp[j], kappa * b);
            sum = sum + udu;
            Raw<T>::template store<VEC>(dx[j], G * t[j].si, ln.m);
            Raw<T>::template store<VEC>(dgr[j], udu * fma4(r, minus, one), ln.m);
            Raw<T>::template store<VEC>(dgi[j], G * b * fma4(t[j].i, minus, one), ln.m);
            C = shrink<WEAK>(c, G);
            if (begins(j) && p.a.dh0) ln.put(p.a.dh0 + sh.rows.seq[warp * kBR + j] * p.a.D, C);
        }
    }
    if (!PACKED && tile == 0 && warp == 0 && p.a.dh0) ln.put(p.a.dh0 + at.b * p.a.D, C);
    if (p.part) {
        __syncthreads(); /* every warp is done with the states' maps */
        sh.states.H[warp][ln.lane] = v4(sum);
        __syncthreads();
        for (int k = threadIdx.x; k < kC; k += blockDim.x) {
            float v = 0.f;
            for (int w = 0; w < warps; ++w) v += ((const float *)sh.states.H[w])[k];
            const int ch = VEC ? k : (k % kV) * 32 + k / kV;
            p.part[(at.pos * p.chains + at.chain) * kC + ch] = v;
        }
    }
}

template <typename T, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kBW * 32, 1) k_glr_bwd(const __grid_constant__ Dev p) {
    __shared__ BwdShared<PACKED> sh;
    typedef typename Raw<T>::type raw;
    const int warp = threadIdx.x / 32;
    const Place at = place(p, &sh.slot);
    const Lane<VEC> ln(at.ch0, p.a.D);
    const long tile = p.tiles - 1 - at.pos, tile0 = tile * kBT, row0 = tile0 + warp * kBR;
    const long left = p.a.L - row0;
    const int live = left < 0 ? 0 : left < kBR ? (int)left : kBR;
    if (PACKED) map_rows(sh.rows, p.a, tile0);
    raw x[kBR], gr[kBR], gi[kBR], dy[kBR];
    {
        const Run<const T, VEC> pr(p.a.gate_r, at.b, row0, ln), pi(p.a.gate_i, at.b, row0, ln),
            px(p.a.x, at.b, row0, ln), pd(p.a.dy, at.b, row0, ln);
#pragma unroll
        for (int j = 0; j < kBR; ++j) {
            const unsigned m = (PACKED ? sh.rows.seq[warp * kBR + j] >= 0 : j < live) ? ln.m : 0u;
            gr[j] = Raw<T>::template load<VEC>(pr[j], m);
            gi[j] = Raw<T>::template load<VEC>(pi[j], m);
            x[j] = Raw<T>::template load<VEC>(px[j], m);
            dy[j] = Raw<T>::template load<VEC>(pd[j], m);
        }
    }
    if (make_rates<VEC>(p.a, at.ch0, (float *)sh.rate, (float *)sh.sroot))
        bwd_tile<T, VEC, PACKED, false>(p, at, ln, sh, x, gr, gi, dy, tile, row0, live);
    else
        bwd_tile<T, VEC, PACKED, true>(p, at, ln, sh, x, gr, gi, dy, tile, row0, live);
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
    const Rates rt = {f4s(rate), f4s(sqrtf(2.f * rate))};
    const T *px = (const T *)a.x.data + k * a.x.row_stride + d;
    const T *pr = (const T *)a.gate_r.data + k * a.gate_r.row_stride + d;
    const T *pi = (const T *)a.gate_i.data + k * a.gate_i.row_stride + d;
    const F4 gr = f4s((float)*pr), gi = f4s((float)*pi), x = f4s((float)*px);
    float *s = a.state + slot * a.ld_state + d;
    float h = *s;
    if (rate <= kWeak) {
        const Terms t = terms<true>(gr, gi, rt);
        h = advance<true>(t.c, f4s(h), t.si * x).l.x;
    } else {
        const Terms t = terms<false>(gr, gi, rt);
        h = advance<false>(t.c, f4s(h), t.si * x).l.x;
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

/* Whether the tensors allow four channels an access: width, strides and
 * addresses are multiples of four elements. */
bool vectors(const KmbGLR *a, const KmbRows *const *rows, int n) {
    const size_t es = a->type == KMB_BF16 ? 2 : 4;
    if (a->D % kV) return false;
    for (int i = 0; i < n; ++i) {
        const KmbRows *r = rows[i];
        if (!r->data) continue;
        if (((size_t)r->data / es) % kV || r->row_stride % kV) return false;
        if (!a->offsets && a->batch > 1 && r->batch_stride % kV) return false;
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
    d.shown.A = (float4 *)((char *)ws + kHead);
    d.shown.H = d.shown.A + q.words / kV;
    d.shown.end = d.shown.H + q.words / kV;
    d.shown.step = q.chains * 32;
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
    const bool vec = vectors(&d.a, rows, 4);
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
    const bool vec = vectors(&d.a, rows, 7);
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
