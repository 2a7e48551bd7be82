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
 * Both directions are one pass over the data (a single-pass scan with
 * decoupled look-back).  A CTA takes a tile of rows x
 * channels: a warp owns a run of consecutive rows, a lane two channels.
 * A run is first reduced to its affine map h -> A h + H, the maps of a
 * tile's warps are joined through shared memory, and the maps of the tiles
 * of one channel group through global memory: a tile publishes its map,
 * waits until each of the tiles before it shows either its map or its final
 * state, applies the maps from the nearest final state on, publishes its
 * own final state and only then runs its rows from the state that enters
 * them.  The final state of a tile is always the map of that tile applied
 * to the final state of the one before it, whichever of the two was read,
 * so results do not depend on timing.
 *
 * Measured (B200, 6.56 TB/s copy): forward 8 x 4096 x 1536 fp32 135 us (6.0
 * TB/s), bf16 103 us (3.9 TB/s); 1 x 65536 x 2048 bf16 352 us (3.0 TB/s);
 * backward 8 x 4096 x 1536 bf16 163 us (4.3 TB/s); rows that are not 16-byte
 * aligned, 24001 x 771 fp32, 109 and 234 us (2.7 and 2.2 TB/s).
 */
#include <cuda.h>
#include <cuda_bf16.h>

#include "kmb_common.cuh"
#include "kmb_tma.cuh"
#include "../kmb_internal.h"

namespace {

/* tiles before its own that a tile looks at: the kernels for any alignment,
 * the resident ones */
constexpr int kWindow = 12, kRingWindow = 16;
constexpr unsigned kUnset = 0xffffffffu; /* workspace word not written yet */

/* set when a wait gave up (kmb_glr_check_error) */
__device__ int g_glr_error;

/* ------------------------------------------------------------------ */
/* V channels of one row, as FFMA2 pairs                                */
/* ------------------------------------------------------------------ */

template <int V>
struct Pack;
template <>
struct Pack<2> {
    typedef float2 type;
};

template <int V>
struct F {
    float2 p[V / 2];
    __device__ __forceinline__ float operator[](int k) const { return k % 2 ? p[k / 2].y : p[k / 2].x; }
};
template <int V>
__device__ __forceinline__ F<V> all(float v) {
    F<V> r;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = kmb_f2s(v);
    return r;
}
__device__ __forceinline__ F<2> from(float2 v) { return {{v}}; }
__device__ __forceinline__ float2 to(F<2> a) { return a.p[0]; }
template <int V>
__device__ __forceinline__ F<V> operator+(F<V> a, F<V> b) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) a.p[i] = kmb_add2(a.p[i], b.p[i]);
    return a;
}
template <int V>
__device__ __forceinline__ F<V> operator*(F<V> a, F<V> b) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) a.p[i] = kmb_mul2(a.p[i], b.p[i]);
    return a;
}
template <int V>
__device__ __forceinline__ F<V> fma(F<V> a, F<V> b, F<V> c) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) c.p[i] = kmb_fma2(a.p[i], b.p[i], c.p[i]);
    return c;
}
template <int V, typename Fn>
__device__ __forceinline__ F<V> each(Fn f) { /* f(channel) */
    F<V> r;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = kmb_f2(f(2 * i), f(2 * i + 1));
    return r;
}

__device__ __forceinline__ unsigned pack(float2 v) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const unsigned *>(&h);
}
__device__ __forceinline__ float2 unpack(unsigned v) {
    return kmb_f2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

/* V channels as stored: of bf16, two in a word, the first in the low half. */
template <typename T, int V>
struct Raw;
template <int V>
struct Raw<float, V> {
    typedef typename Pack<V>::type type;
    static __device__ __forceinline__ F<V> f(type v) { return from(v); }
    static __device__ __forceinline__ type r(F<V> v) { return to(v); }
};
template <>
struct Raw<__nv_bfloat16, 2> {
    typedef unsigned type;
    static __device__ __forceinline__ F<2> f(unsigned v) { return {{unpack(v)}}; }
    static __device__ __forceinline__ unsigned r(F<2> v) { return pack(v.p[0]); }
};

/* A lane's two channels in global memory.  VEC: 2 lane and 2 lane + 1 in one
 * access; else lane and lane + 32, for odd widths, strides and addresses
 * (every access still covers a contiguous piece of the row).  m: bit k set
 * where channel k exists. */
constexpr int kV = 2;
constexpr int kC = 32 * kV;

template <bool VEC>
__device__ __forceinline__ float2 load(const float *p, unsigned m) {
    if (VEC) return m ? __ldcs(reinterpret_cast<const float2 *>(p)) : make_float2(0.f, 0.f);
    return make_float2(m & 1 ? __ldcs(p) : 0.f, m & 2 ? __ldcs(p + 32) : 0.f);
}
template <bool VEC>
__device__ __forceinline__ unsigned load(const __nv_bfloat16 *p, unsigned m) {
    if (VEC) return m ? __ldcs(reinterpret_cast<const unsigned *>(p)) : 0u;
    const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
    const unsigned a = m & 1 ? __ldcs(q) : 0u, b = m & 2 ? __ldcs(q + 32) : 0u;
    return a | b << 16;
}
template <bool VEC>
__device__ __forceinline__ void store(float *p, F<2> v, unsigned m) {
    if constexpr (VEC) {
        if (m) __stcs(reinterpret_cast<float2 *>(p), to(v));
    } else {
        if (m & 1) __stcs(p, v[0]);
        if (m & 2) __stcs(p + 32, v[1]);
    }
}
template <bool VEC>
__device__ __forceinline__ void store(__nv_bfloat16 *p, F<2> v, unsigned m) {
    const unsigned u = Raw<__nv_bfloat16, 2>::r(v);
    if constexpr (VEC) {
        if (m) __stcs(reinterpret_cast<unsigned *>(p), u);
    } else {
        unsigned short *q = reinterpret_cast<unsigned short *>(p);
        if (m & 1) __stcs(q, (unsigned short)u);
        if (m & 2) __stcs(q + 32, (unsigned short)(u >> 16));
    }
}

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
 *   (e^-u - 1) / u                    3.0e-9 in real arithmetic, as stored
 *   sqrt((1 - e^-2u) / (2 u))         5.1e-9
 *   kappa = u / (e^2u - 1)            6.6e-9
 * A tile's channels whose rates are all at most kWeak need no exponential of
 * u, no square root and no cancelling 1 - a^2, and their recurrence runs on
 * a - 1 as h + (b + (a - 1) h): a memory of 1 / (1 - a) steps multiplies the error
 * of the decay, and a itself, next to 1, cannot hold it to more than
 * 2^-25 / (1 - a).
 */
constexpr float kWeak = 0.25f;

template <int V>
__device__ __forceinline__ F<V> poly4(F<V> u, float c0, float c1, float c2, float c3, float c4) {
    F<V> p = fma(all<V>(c4), u, all<V>(c3));
    p = fma(p, u, all<V>(c2));
    p = fma(p, u, all<V>(c1));
    return fma(p, u, all<V>(c0));
}
template <int V>
__device__ __forceinline__ F<V> poly_expm1(F<V> u) {
    return poly4(u, -1.f, 0.49999964237213135f, -0.1666528880596161f, 0.04150013253092766f,
                 -0.007530174218118191f);
}
template <int V>
__device__ __forceinline__ F<V> poly_root(F<V> u) {
    return poly4(u, 1.f, -0.49999940395355225f, 0.20831027626991272f, -0.06222091242671013f,
                 0.01236682292073965f);
}
template <int V>
__device__ __forceinline__ F<V> poly_kappa(F<V> u) {
    return poly4(u, 0.5f, -0.5000002980232239f, 0.1666753739118576f, -8.377274934900925e-05f,
                 -0.010830916464328766f);
}

/* Per channel: rate, and sqrt(2 rate) for root = sqrt(2 u) sqrt((1 - e^-2u) / 2u). */
template <int V>
struct Rates {
    F<V> rate, sroot;
};

/* Of one row: c is a - 1 (WEAK) or a, q = sqrt(r) = (1 + e^-gate_r)^-1/2, i,
 * and si = root i. */
template <int V>
struct Terms {
    F<V> c, q, i, si;
};

template <bool WEAK, int V>
__device__ __forceinline__ Terms<V> terms(F<V> gr, F<V> gi, const Rates<V> &k) {
    Terms<V> t;
    const F<V> nl = all<V>(-KMB_LOG2E), one = all<V>(1.f);
    gr = gr * nl;
    gi = gi * nl;
    const F<V> er = each<V>([&](int n) { return kmb_ex2(gr[n]); }) + one;
    const F<V> ei = each<V>([&](int n) { return kmb_ex2(gi[n]); }) + one;
    t.q = each<V>([&](int n) { return rsqrt_mufu(er[n]); });
    t.i = each<V>([&](int n) { return rcp_mufu(ei[n]); });
    const F<V> u = k.rate * (t.q * t.q);
    const F<V> m = u * poly_expm1(u);
    F<V> root = k.sroot * t.q * poly_root(u);
    if (WEAK) {
        t.c = m;
    } else {
        const F<V> un = u * nl;
        const F<V> e = each<V>([&](int n) { return kmb_ex2(un[n]); });
        t.c = each<V>([&](int n) { return u[n] <= kWeak ? 1.f + m[n] : e[n]; });
        root = each<V>([&](int n) { return u[n] <= kWeak ? root[n] : sqrt_mufu(fmaf(-e[n], e[n], 1.f)); });
    }
    t.si = root * t.i;
    return t;
}

/* a h + b */
template <bool WEAK, int V>
__device__ __forceinline__ F<V> advance(F<V> c, F<V> h, F<V> b) {
    return WEAK ? h + fma(c, h, b) : fma(c, h, b);
}
/* a A */
template <bool WEAK, int V>
__device__ __forceinline__ F<V> shrink(F<V> c, F<V> A) {
    return WEAK ? fma(c, A, A) : c * A;
}

/* What multiplies G, what the row's state is worth, in its gradients; hp is
 * the state before it.  dx = G si; udu = G f; dgate_r = udu q; dgate_i = G i:
 * q becomes 1 - r, i becomes b (1 - i). */
template <bool WEAK, int V>
__device__ __forceinline__ void factors(Terms<V> &t, F<V> rate, F<V> x, F<V> hp, F<V> &f) {
    const F<V> one = all<V>(1.f), minus = all<V>(-1.f);
    const F<V> r = t.q * t.q, u = rate * r, b = t.si * x;
    F<V> kappa = poly_kappa(u), ua; /* ua: -u a */
    if (WEAK) {
        ua = fma(t.c, u, u) * minus;
    } else {
        /* e^-u is 0 long before u is 100 */
        ua = each<V>([&](int n) { return u[n] > 100.f ? 0.f : -u[n] * t.c[n]; });
        kappa = each<V>([&](int n) {
            return u[n] <= kWeak ? kappa[n] : -ua[n] * t.c[n] * rcp_mufu(fmaf(-t.c[n], t.c[n], 1.f));
        });
    }
    f = fma(ua, hp, kappa * b);
    t.q = fma(r, minus, one);
    t.i = b * fma(t.i, minus, one);
}

/* ------------------------------------------------------------------ */
/* affine maps h -> A h + H; A = -1 marks a constant one                 */
/* ------------------------------------------------------------------ */

template <int V>
struct Map {
    F<V> A, H;
};

/* MARKED: constant maps occur (a sequence began inside, a final state) */
template <bool MARKED, int V>
__device__ __forceinline__ F<V> apply(const Map<V> &m, F<V> h) {
    const F<V> r = fma(m.A, h, m.H);
    if (!MARKED) return r;
    return each<V>([&](int n) { return m.A[n] < 0.f ? m.H[n] : r[n]; });
}

/* the map of `first` then `then` */
template <bool MARKED, int V>
__device__ __forceinline__ Map<V> join(const Map<V> &first, const Map<V> &then) {
    Map<V> r;
    r.H = apply<MARKED>(then, first.H);
    r.A = first.A * then.A;
    if (MARKED) r.A = each<V>([&](int n) { return first.A[n] < 0.f || then.A[n] < 0.f ? -1.f : r.A[n]; });
    return r;
}

/* What tiles show one another: [place in the chain][chain][lane] of V
 * channels.  Every word is written once, and was kUnset (the workspace is
 * filled at the start of the call): a word that is not kUnset is the value
 * itself, so no fence orders flags against data. */
struct Shown {
    float *A, *H, *end; /* map, final state */
    long step;          /* lanes between places of a chain */
};

__device__ __forceinline__ bool peek(const float *p, F<2> &v) {
    unsigned a, b;
    asm volatile("ld.relaxed.gpu.global.v2.u32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "l"(p) : "memory");
    v = {{kmb_f2(__uint_as_float(a), __uint_as_float(b))}};
    return a != kUnset && b != kUnset;
}
__device__ __forceinline__ float not_unset(float v) {
    return __float_as_uint(v) == kUnset ? __uint_as_float(0x7fffffffu) : v;
}
__device__ __forceinline__ void show(float *p, F<2> v) {
    asm volatile("st.relaxed.gpu.global.v2.f32 [%0], {%1, %2};" ::"l"(p), "f"(not_unset(v[0])),
                 "f"(not_unset(v[1]))
                 : "memory");
}

template <int V>
__device__ __forceinline__ void show(const Shown &s, long o, const Map<V> &m) {
    show(s.A + o * V, m.A);
    show(s.H + o * V, m.H);
}

/* whether the lane's maps are all constant ones */
template <int V>
__device__ __forceinline__ bool constant(F<V> A) {
    bool c = true;
#pragma unroll
    for (int e = 0; e < V; ++e) c &= A[e] < 0.f;
    return c;
}

/* The map of a place, or as a constant one its final state: whichever is
 * there (last: the final state alone will do).  The three loads take one trip
 * to the L2 cache together. */
template <int V>
__device__ __forceinline__ bool glance(const Shown &s, long o, bool last, Map<V> &m) {
    F<V> end;
    const bool done = peek(s.end + o * V, end);
    const bool map = peek(s.A + o * V, m.A) & peek(s.H + o * V, m.H);
    if (done) {
        m.A = all<V>(-1.f);
        m.H = end;
    }
    return done || (map && !last);
}

/* The same, waiting for it.  Bounded by about 2^31 cycles; then the error
 * word is set and later waits return at once.  (The clock is read only when
 * the first glances fail: it costs more than they do.) */
template <int V>
__device__ __forceinline__ Map<V> look(const Shown &s, long o, bool last) {
    Map<V> m;
    long long t0 = 0;
    for (int n = 1; !glance(s, o, last, m); ++n) {
        if (n % 64) continue;
        const long long t = clock64();
        if (n == 64) t0 = t;
        const bool late = t - t0 > (1ll << 31);
        if (late) atomicExch(&g_glr_error, 1);
        if (late || *reinterpret_cast<volatile int *>(&g_glr_error)) {
            m.A = all<V>(-1.f);
            m.H = all<V>(0.f);
            return m;
        }
    }
    return m;
}

/* ------------------------------------------------------------------ */
/* kernel arguments and a tile's place                                  */
/* ------------------------------------------------------------------ */

/* rows between checkpoints */
template <typename T>
constexpr int chunk_of = KMB_GLR_CHUNK(sizeof(T) == 2 ? KMB_BF16 : KMB_F32);

struct Dev {
    KmbGLR a;
    unsigned tiles, groups, chains; /* tiles of a chain, channel groups, batch * groups */
    long chunks;                    /* checkpoints of a chain */
    int states_only;                /* forward: checkpoints alone are wanted */
    const float *ckpt_in;
    float *ckpt_out;
    float *part;                    /* [tiles * chains][channels of a tile] sums of u dL/du */
    unsigned *ticket;
    Shown shown;
    const float2 *rates;            /* of all groups' channels: rate, sqrt(2 rate) (resident kernels) */
};

struct Place {
    unsigned pos, chain, b, group; /* place in the chain, chain, sequence (0 when packed), channel group */
    __device__ __forceinline__ Place(const Dev &p, unsigned id) {
        pos = id / p.chains;
        chain = id - pos * p.chains;
        b = chain / p.groups;
        group = chain - b * p.groups;
    }
};

/* Tiles are taken in the order of their places: a tile waits only for tiles
 * that another CTA has taken before.  The fill makes the ticket -1. */
__device__ __forceinline__ unsigned take_ticket(const Dev &p) { return atomicAdd(p.ticket, 1u) + 1u; }

/* Packed rows: which sequence a row of the tile belongs to and whether it
 * is its first or last. */
template <int ROWS>
struct RowMap {
    int seq[ROWS];
    unsigned char edge[ROWS]; /* 1: first row, 2: last row */
    int whole;                /* every row of the tile that the tensors have is of a sequence */
    int plain;                /* all rows are, and none begins or ends one */
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

/* by one warp; ends with its barrier */
template <int ROWS>
__device__ void map_rows(RowMap<ROWS> &m, const KmbGLR &a, long row0) {
    const int lane = threadIdx.x % 32;
    for (int r = lane; r < ROWS; r += 32) {
        m.seq[r] = -1;
        m.edge[r] = 0;
    }
    __syncwarp();
    const long end = row0 + ROWS < a.L ? row0 + ROWS : a.L;
    int count = 0, edges = 0;
    for (long s = first_sequence(a.offsets, a.batch, row0, lane); s < a.batch; s += 32) {
        long lo = end, hi = end;
        if (s + lane < a.batch) {
            lo = a.offsets[s + lane];
            hi = a.offsets[s + lane + 1];
        }
        const bool past = s + lane < a.batch && lo >= end;
        lo = lo < 0 ? 0 : lo;
        hi = hi > a.L ? a.L : hi;
        /* the sequence's rows within the tile, and its edges among them */
        const int from = (int)((lo > row0 ? lo : row0) - row0), until = (int)((hi < end ? hi : end) - row0);
        const int first = lo >= row0 ? (int)(lo - row0) : -1, last = hi <= end ? (int)(hi - 1 - row0) : -1;
        unsigned some = __ballot_sync(~0u, !past && from < until);
        while (some) {
            const int k = __ffs(some) - 1;
            some &= some - 1;
            const int b = __shfl_sync(~0u, from, k), e = __shfl_sync(~0u, until, k);
            const int f = __shfl_sync(~0u, first, k), l = __shfl_sync(~0u, last, k);
            for (int r = b + lane; r < e; r += 32) {
                m.seq[r] = (int)(s + k);
                m.edge[r] = (unsigned char)((r == f ? 1 : 0) | (r == l ? 2 : 0));
            }
            count += e - b;
            edges += (f >= 0) + (l >= 0);
        }
        if (__any_sync(~0u, past)) break;
    }
    if (lane == 0) {
        m.whole = count >= end - row0;
        m.plain = count == ROWS && edges == 0;
    }
    __syncwarp();
}

/* What an empty sequence's end is: `from` (zeros when NULL) to `to`, for
 * the channels [ch0, ch1); by `warps` warps. */
__device__ void empty_sequences(const KmbGLR &a, const float *from, float *to, long ch0, long ch1, int warp,
                                int warps) {
    if (!to) return;
    const int lane = threadIdx.x % 32;
    for (long s = warp * 32L; s < a.batch; s += warps * 32L) {
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
            for (long d = ch0 + lane; d < a.D && d < ch1; d += 32)
                to[k * a.D + d] = from ? from[k * a.D + d] : 0.f;
        }
    }
}

/* The lane's channels: the first, and which exist. */
template <bool VEC, int V>
struct Lane {
    long d;
    unsigned m;
    int lane;
    static constexpr int kNext = VEC ? 1 : 32; /* to the next channel */
    __device__ __forceinline__ Lane(long ch0, long D) {
        lane = threadIdx.x % 32;
        d = ch0 + (VEC ? V * lane : lane);
        if (VEC) { /* D is a multiple of V */
            m = d < D ? (1u << V) - 1 : 0u;
            return;
        }
        m = 0;
#pragma unroll
        for (int k = 0; k < V; ++k) m |= d + k * kNext < D ? 1u << k : 0u;
    }
    /* a [.., D] fp32 vector at the channels, 0 where NULL */
    __device__ __forceinline__ F<V> at(const float *p) const {
        return each<V>([&](int k) { return p && (m >> k & 1) ? p[d + k * kNext] : 0.f; });
    }
    __device__ __forceinline__ void put(float *p, F<V> v) const {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (p && (m >> k & 1)) p[d + k * kNext] = v[k];
    }
};

/* A tensor's rows of the run: pointer to the lane's channels of row j. */
template <typename T>
struct Run {
    T *p;
    long step;
    __device__ __forceinline__ Run(const KmbRows &r, long b, long row, long d) {
        p = (T *)r.data + b * r.batch_stride + row * r.row_stride + d;
        step = r.row_stride;
    }
    __device__ __forceinline__ T *operator[](int j) const { return p + j * step; }
};

/* Maps of the warps of a tile. */
template <int W, int V>
struct Maps {
    typename Pack<V>::type A[W][32], H[W][32];
    __device__ __forceinline__ void put(int w, int lane, F<V> a, F<V> h) {
        A[w][lane] = to(a);
        H[w][lane] = to(h);
    }
    __device__ __forceinline__ Map<V> at(int w, int lane) const { return {from(A[w][lane]), from(H[w][lane])}; }
};

/* Joins the tile with the ones before it in its chain and returns the state
 * that enters it.  agg: the warps' maps, joined from the last when REVERSE;
 * h: the state that enters the chain (place 0).  For kernels with one tile a
 * CTA: every warp looks at other tiles, then all go through what was seen. */
template <bool VEC, bool MARKED, bool REVERSE, int W, int N, int V>
__device__ __forceinline__ F<V> enter_tile(const Dev &p, const Place &at, const Lane<VEC, V> &ln,
                                           const Maps<W, V> &agg, Maps<N, V> &seen, int warps, F<V> h) {
    const int warp = threadIdx.x / 32;
    if (p.tiles == 1) return h;
    const Shown &s = p.shown;
    const long o = at.pos * s.step + at.chain * 32 + ln.lane;
    Map<V> m = {all<V>(1.f), all<V>(0.f)};
    if (warp == 0 && at.pos + 1 < p.tiles) {
        for (int k = 0; k < warps; ++k) m = join<MARKED>(m, agg.at(REVERSE ? warps - 1 - k : k, ln.lane));
        if (at.pos > 0) show(s, o, m);
    }
    if (at.pos > 0) {
        const int n = at.pos < N ? (int)at.pos : N;
        int k;
        /* warp 0, which joins the tile's maps, comes last */
        for (k = warp ? warp - 1 : warps - 1; k < n; k += warps) {
            const Map<V> v = look<V>(s, o - (k + 1) * s.step, k == N - 1);
            seen.put(k, ln.lane, v.A, v.H);
        }
        __syncthreads();
        /* from the nearest final states on; the first tile shows nothing else */
        for (k = 0; k < n - 1; ++k)
            if (constant(from(seen.A[k][ln.lane]))) break;
        for (; k >= 0; --k) h = apply<true>(seen.at(k, ln.lane), h);
    }
    if (warp == 0 && at.pos + 1 < p.tiles) show(s.end + o * V, apply<MARKED>(m, h));
    return h;
}

/*
 * The same for the resident kernels, by one warp, while the others work or
 * other CTAs do: m is the tile's map.  Most often the tile before has its
 * final state, so places are looked at one by one; 8 at a time (24 loads
 * under way) took 3300 cycles a tile, one 1900.
 */
template <bool MARKED, int N, int V>
__device__ __forceinline__ F<V> enter_chain(const Dev &p, const Place &at, const Lane<true, V> &ln, const Map<V> &m,
                                            Maps<N, V> &seen, const float *first) {
    const Shown &s = p.shown;
    const long o = at.pos * s.step + at.chain * 32 + ln.lane;
    const bool next = at.pos + 1 < p.tiles; /* a tile waits for this one */
    if (at.pos == 0) {
        const F<V> h = ln.at(first);
        if (next) show(s.end + o * V, apply<MARKED>(m, h));
        return h;
    }
    if (next) show(s, o, m);
    const int n = at.pos < N ? (int)at.pos : N;
    int k = 0;
    for (bool found = false; !found && k < n; ++k) {
        const Map<V> v = look<V>(s, o - (k + 1) * s.step, k == N - 1);
        seen.put(k, ln.lane, v.A, v.H);
        found = __all_sync(~0u, constant(v.A));
    }
    F<V> h = all<V>(0.f);
    while (--k >= 0) h = apply<true>(seen.at(k, ln.lane), h);
    if (next) show(s.end + o * V, apply<MARKED>(m, h));
    return h;
}

/* ------------------------------------------------------------------ */
/* a warp's run of rows                                                 */
/* ------------------------------------------------------------------ */

/*
 * What the forward and the backward do with a run of R rows; where the rows
 * come from and go to is the caller's: io.x(j), io.gr(j), io.gi(j), io.dy(j),
 * io.y(j, v), io.grads(j, dx, dgate_r, dgate_i).  FULL: all rows exist and none begins or ends a
 * sequence.  Packed rows else look themselves up in `rows`.
 */
template <typename Io, bool VEC, bool PACKED, bool FULL, bool WEAK, int R, int ROWS, int V>
struct RunOf {
    const Dev &p;
    const Place &at;
    const Lane<VEC, V> &ln;
    const RowMap<ROWS> &rows;
    Io &io;
    long row0;
    int live, warp; /* rows that exist (not PACKED) */

    __device__ __forceinline__ bool in(int j) const {
        return FULL || (PACKED ? rows.seq[warp * R + j] >= 0 : j < live);
    }
    __device__ __forceinline__ bool begins(int j) const {
        return PACKED && !FULL && (rows.edge[warp * R + j] & 1);
    }
    __device__ __forceinline__ bool ends(int j) const { return PACKED && !FULL && (rows.edge[warp * R + j] & 2); }
    /* the sequence's row of a [batch, D] tensor */
    __device__ __forceinline__ F<V> of(const float *v, int j) const {
        return ln.at(v ? v + rows.seq[warp * R + j] * p.a.D : nullptr);
    }
    __device__ __forceinline__ void put(float *v, int j, F<V> x) const {
        if (v) ln.put(v + rows.seq[warp * R + j] * p.a.D, x);
    }

    /* The forward before the state that enters is known: decays and input
     * terms of the rows (a sequence's first row: its state), and the run's
     * map. */
    __device__ __forceinline__ Map<V> forward_map(const Rates<V> &rt, F<V> (&c)[R], F<V> (&b)[R]) const {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const Terms<V> t = terms<WEAK>(io.gr(j), io.gi(j), rt);
            c[j] = t.c;
            b[j] = t.si * io.x(j);
        }
        Map<V> m = {all<V>(1.f), all<V>(0.f)};
        bool fresh = false; /* a sequence begins in this run */
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (in(j)) {
                if (begins(j)) {
                    m.H = of(p.a.h0, j);
                    fresh = true;
                }
                m.H = advance<WEAK>(c[j], m.H, b[j]);
                m.A = shrink<WEAK>(c[j], m.A);
                if (begins(j)) b[j] = m.H; /* h0 is not read again: h_last may be h0, and another warp's to write */
            }
        }
        if (fresh) m.A = all<V>(-1.f);
        return m;
    }
    /* h: the state that enters the run */
    __device__ __forceinline__ void forward_rows(F<V> h, const F<V> (&c)[R], const F<V> (&b)[R]) const {
        /* the run's row with a checkpoint, if any */
        constexpr int chunk = Io::kChunk;
        static_assert(chunk >= R, "at most one checkpoint a run");
        const int mark = p.ckpt_out ? Io::mark(row0, warp) : -1;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (in(j)) {
                if (j == mark) ln.put(p.ckpt_out + (at.b * p.chunks + (row0 + j) / chunk) * p.a.D, h);
                h = begins(j) ? b[j] : advance<WEAK>(c[j], h, b[j]);
                io.y(j, h);
                if (ends(j)) put(p.a.h_last, j, h);
            }
        }
        if (!PACKED && p.a.h_last && live > 0 && row0 + live == p.a.L) ln.put(p.a.h_last + at.b * p.a.D, h);
    }

    /* The backward, likewise: the terms of the rows, what the states of
     * sequences that end here are worth, and the run's maps, of the states and
     * of the adjoint.  The adjoint that reaches row t - 1 from
     * row t is C_t = a_t (dy_t + C_{t+1}). */
    __device__ __forceinline__ void backward_maps(const Rates<V> &rt, Terms<V> (&t)[R], F<V> (&last)[R],
                                                  Map<V> &state, Map<V> &adjoint) const {
#pragma unroll
        for (int j = 0; j < R; ++j) t[j] = terms<WEAK>(io.gr(j), io.gi(j), rt);
        F<V> A = all<V>(1.f), H = all<V>(0.f), K = H;
        bool fresh = false, closed = false;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (in(j)) {
                if (begins(j)) {
                    H = of(p.a.h0, j);
                    fresh = true;
                }
                H = advance<WEAK>(t[j].c, H, t[j].si * io.x(j));
                A = shrink<WEAK>(t[j].c, A);
            }
        }
#pragma unroll
        for (int j = R - 1; j >= 0; --j) {
            if (in(j)) {
                if (ends(j)) {
                    K = last[j] = of(p.a.dh_last, j); /* not read again: dh0 may be dh_last */
                    closed = true;
                }
                K = shrink<WEAK>(t[j].c, K + io.dy(j));
            }
        }
        state = {fresh ? all<V>(-1.f) : A, H};
        adjoint = {closed ? all<V>(-1.f) : A, K};
    }
    /* h: the state that enters the run.  Leaves in t what the gradients are
     * when a row's adjoint is one: c, si (dx) as they were, q (dgate_r over
     * udu), i (dgate_i), and udu in f. */
    __device__ __forceinline__ void backward_factors(F<V> h, F<V> rate, Terms<V> (&t)[R], F<V> (&f)[R]) const {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (begins(j)) h = of(p.a.h0, j);
            const F<V> x = io.x(j), hp = h;
            h = advance<WEAK>(t[j].c, h, t[j].si * x);
            factors<WEAK>(t[j], rate, x, hp, f[j]);
        }
    }
    /* C: the adjoint that reaches the run.  Returns the sum of udu. */
    __device__ __forceinline__ F<V> backward_rows(F<V> C, const Terms<V> (&t)[R], const F<V> (&last)[R],
                                                  const F<V> (&f)[R]) const {
        F<V> sum = all<V>(0.f);
#pragma unroll
        for (int j = R - 1; j >= 0; --j) {
            if (in(j)) {
                if (ends(j)) C = last[j];
                const F<V> G = C + io.dy(j), udu = G * f[j];
                sum = sum + udu;
                io.grads(j, G * t[j].si, udu * t[j].q, G * t[j].i);
                C = shrink<WEAK>(t[j].c, G);
                if (begins(j)) put(p.a.dh0, j, C);
            }
        }
        if (!PACKED && row0 == 0 && p.a.dh0) ln.put(p.a.dh0 + at.b * p.a.D, C);
        return sum;
    }
};

/* ------------------------------------------------------------------ */
/* kernels for any alignment: rows loaded by the threads that own them   */
/* ------------------------------------------------------------------ */

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

template <int W, int ROWS, bool PACKED>
struct AnyShared {
    Maps<W, kV> agg;
    Maps<kWindow, kV> seen;
    typename Pack<kV>::type rate[32], sroot[32];
    unsigned slot;
    RowMap<PACKED ? ROWS : 1> rows;
};

/* the tile's number; ends with a barrier when a chain has several tiles */
__device__ __forceinline__ unsigned tile_id(const Dev &p, unsigned *slot) {
    if (p.tiles == 1) return blockIdx.x;
    if (threadIdx.x == 0) *slot = take_ticket(p);
    __syncthreads();
    return *slot;
}

constexpr int kFR = 8, kFW = 8, kFT = kFR * kFW;

template <typename T, bool VEC>
struct AnyFwdIo {
    static constexpr int kChunk = chunk_of<T>;
    static __device__ __forceinline__ int mark(long row0, int) {
        return (int)((row0 + kChunk - 1) / kChunk * kChunk - row0);
    }
    typename Raw<T, kV>::type rx[kFR], rr[kFR], ri[kFR];
    Run<T> out;
    unsigned m;
    __device__ __forceinline__ F<kV> x(int j) const { return Raw<T, kV>::f(rx[j]); }
    __device__ __forceinline__ F<kV> gr(int j) const { return Raw<T, kV>::f(rr[j]); }
    __device__ __forceinline__ F<kV> gi(int j) const { return Raw<T, kV>::f(ri[j]); }
    __device__ __forceinline__ void y(int j, F<kV> v) const {
        if (out.p) store<VEC>(out[j], v, m);
    }
};

template <bool WEAK, typename T, bool VEC, bool PACKED>
__device__ __forceinline__ void any_forward(const Dev &p, const Place &at, const Lane<VEC, kV> &ln,
                                            AnyShared<kFW, kFT, PACKED> &sh, AnyFwdIo<T, VEC> &io,
                                            const Rates<kV> &rt, long row0, int live, int warp) {
    const RunOf<AnyFwdIo<T, VEC>, VEC, PACKED, false, WEAK, kFR, PACKED ? kFT : 1, kV> run = {
        p, at, ln, sh.rows, io, row0, live, warp};
    F<kV> c[kFR], b[kFR];
    const Map<kV> m = run.forward_map(rt, c, b);
    sh.agg.put(warp, ln.lane, m.A, m.H);
    /* before the barrier: h_last may be h0, and another warp's to write */
    const F<kV> first = ln.at(!PACKED && p.a.h0 && at.pos == 0 ? p.a.h0 + at.b * p.a.D : nullptr);
    __syncthreads();
    F<kV> h = enter_tile<VEC, PACKED, false>(p, at, ln, sh.agg, sh.seen, blockDim.x / 32, first);
    for (int w = 0; w < warp; ++w) h = apply<PACKED>(sh.agg.at(w, ln.lane), h);
    run.forward_rows(h, c, b);
}

template <typename T, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kFW * 32, 3) k_glr_fwd(const __grid_constant__ Dev p) {
    __shared__ AnyShared<kFW, kFT, PACKED> sh;
    kmb_wait_before();
    const int warp = threadIdx.x / 32;
    const Place at(p, tile_id(p, &sh.slot));
    const long ch0 = (long)at.group * kC;
    const Lane<VEC, kV> ln(ch0, p.a.D);
    const long tile0 = (long)at.pos * kFT, row0 = tile0 + warp * kFR;
    const long left = p.a.L - row0;
    const int live = left < 0 ? 0 : left < kFR ? (int)left : kFR;
    if (PACKED) {
        if (warp == 0) map_rows(sh.rows, p.a, tile0);
        __syncthreads();
    }
    AnyFwdIo<T, VEC> io = {{}, {}, {}, Run<T>(p.a.y, at.b, row0, ln.d), ln.m};
    if (p.states_only) io.out.p = nullptr;
    {
        const Run<const T> pr(p.a.gate_r, at.b, row0, ln.d), pi(p.a.gate_i, at.b, row0, ln.d),
            px(p.a.x, at.b, row0, ln.d);
#pragma unroll
        for (int j = 0; j < kFR; ++j) {
            const unsigned m = (PACKED ? sh.rows.seq[warp * kFR + j] >= 0 : j < live) ? ln.m : 0u;
            io.rr[j] = load<VEC>(pr[j], m);
            io.ri[j] = load<VEC>(pi[j], m);
            io.rx[j] = load<VEC>(px[j], m);
        }
    }
    const bool strong = make_rates<VEC>(p.a, ch0, (float *)sh.rate, (float *)sh.sroot);
    const Rates<kV> rt = {from(sh.rate[ln.lane]), from(sh.sroot[ln.lane])};
    if (strong) any_forward<false, T, VEC, PACKED>(p, at, ln, sh, io, rt, row0, live, warp);
    else any_forward<true, T, VEC, PACKED>(p, at, ln, sh, io, rt, row0, live, warp);
    if (PACKED && at.pos == 0 && !p.states_only)
        empty_sequences(p.a, p.a.h0, p.a.h_last, ch0, ch0 + kC, warp, blockDim.x / 32);
}

constexpr int kBW = 7;
template <typename T>
constexpr int kBR = sizeof(T) == 2 ? 8 : 4;
template <typename T>
constexpr int kBT = kBR<T> * kBW;
static_assert(kBT<float> % KMB_GLR_CHUNK(KMB_F32) == 0 && kBT<__nv_bfloat16> % KMB_GLR_CHUNK(KMB_BF16) == 0,
              "a backward tile begins at a checkpoint");

template <typename T, bool VEC>
struct AnyBwdIo {
    typename Raw<T, kV>::type rx[kBR<T>], rr[kBR<T>], ri[kBR<T>], rd[kBR<T>];
    Run<T> dx, dgr, dgi;
    unsigned m;
    __device__ __forceinline__ F<kV> x(int j) const { return Raw<T, kV>::f(rx[j]); }
    __device__ __forceinline__ F<kV> gr(int j) const { return Raw<T, kV>::f(rr[j]); }
    __device__ __forceinline__ F<kV> gi(int j) const { return Raw<T, kV>::f(ri[j]); }
    __device__ __forceinline__ F<kV> dy(int j) const { return Raw<T, kV>::f(rd[j]); }
    __device__ __forceinline__ void grads(int j, F<kV> x, F<kV> r, F<kV> i) const {
        store<VEC>(dx[j], x, m);
        store<VEC>(dgr[j], r, m);
        store<VEC>(dgi[j], i, m);
    }
};

template <int W, int ROWS, bool PACKED>
struct AnyBwdShared : AnyShared<W, ROWS, PACKED> {
    Maps<W, kV> states;
};

template <bool WEAK, typename T, bool VEC, bool PACKED>
__device__ __forceinline__ F<kV> any_backward(const Dev &p, const Place &at, const Lane<VEC, kV> &ln,
                                              AnyBwdShared<kBW, kBT<T>, PACKED> &sh, AnyBwdIo<T, VEC> &io,
                                              const Rates<kV> &rt, F<kV> entry, long row0, int live, int warp) {
    const int warps = blockDim.x / 32;
    const RunOf<AnyBwdIo<T, VEC>, VEC, PACKED, false, WEAK, kBR<T>, PACKED ? kBT<T> : 1, kV> run = {
        p, at, ln, sh.rows, io, row0, live, warp};
    Terms<kV> t[kBR<T>];
    F<kV> ends[kBR<T>];
    Map<kV> state, adjoint;
    run.backward_maps(rt, t, ends, state, adjoint);
    sh.states.put(warp, ln.lane, state.A, state.H);
    sh.agg.put(warp, ln.lane, adjoint.A, adjoint.H);
    /* before the barrier: dh0 may be dh_last, and another warp's to write */
    const F<kV> last = ln.at(!PACKED && p.a.dh_last && at.pos == 0 ? p.a.dh_last + at.b * p.a.D : nullptr);
    __syncthreads();
    F<kV> f[kBR<T>];
    for (int w = 0; w < warp; ++w) entry = apply<PACKED>(sh.states.at(w, ln.lane), entry);
    run.backward_factors(entry, rt.rate, t, f);
    F<kV> C = enter_tile<VEC, PACKED, true>(p, at, ln, sh.agg, sh.seen, warps, last);
    for (int w = warps - 1; w > warp; --w) C = apply<PACKED>(sh.agg.at(w, ln.lane), C);
    return run.backward_rows(C, t, ends, f);
}

/* CTAs of an SM.  Four of 4 rows (72 registers a thread, 112 to 212 bytes of
 * it spilled) take 237 us, three 262 and two (128 registers) 260 (24001 x 771
 * fp32).  8 rows spill 56 to 248 bytes with two CTAs already. */
template <typename T>
constexpr int kBCtas = sizeof(T) == 2 ? 2 : 4;

template <typename T, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kBW * 32, kBCtas<T>) k_glr_bwd(const __grid_constant__ Dev p) {
    __shared__ AnyBwdShared<kBW, kBT<T>, PACKED> sh;
    kmb_wait_before();
    const int warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const Place at(p, tile_id(p, &sh.slot));
    const long ch0 = (long)at.group * kC;
    const Lane<VEC, kV> ln(ch0, p.a.D);
    const long tile0 = (long)(p.tiles - 1 - at.pos) * kBT<T>, row0 = tile0 + warp * kBR<T>;
    const long left = p.a.L - row0;
    const int live = left < 0 ? 0 : left < kBR<T> ? (int)left : kBR<T>;
    if (PACKED) {
        if (warp == 0) map_rows(sh.rows, p.a, tile0);
        __syncthreads();
    }
    AnyBwdIo<T, VEC> io = {{}, {}, {}, {}, Run<T>(p.a.dx, at.b, row0, ln.d), Run<T>(p.a.dgate_r, at.b, row0, ln.d),
                           Run<T>(p.a.dgate_i, at.b, row0, ln.d), ln.m};
    {
        const Run<const T> pr(p.a.gate_r, at.b, row0, ln.d), pi(p.a.gate_i, at.b, row0, ln.d),
            px(p.a.x, at.b, row0, ln.d), pd(p.a.dy, at.b, row0, ln.d);
#pragma unroll
        for (int j = 0; j < kBR<T>; ++j) {
            const unsigned m = (PACKED ? sh.rows.seq[warp * kBR<T> + j] >= 0 : j < live) ? ln.m : 0u;
            io.rr[j] = load<VEC>(pr[j], m);
            io.ri[j] = load<VEC>(pi[j], m);
            io.rx[j] = load<VEC>(px[j], m);
            io.rd[j] = load<VEC>(pd[j], m);
        }
    }
    const F<kV> entry = ln.at(tile0 < p.a.L ? p.ckpt_in + (at.b * p.chunks + tile0 / chunk_of<T>) * p.a.D : nullptr);
    const bool strong = make_rates<VEC>(p.a, ch0, (float *)sh.rate, (float *)sh.sroot);
    const Rates<kV> rt = {from(sh.rate[ln.lane]), from(sh.sroot[ln.lane])};
    const F<kV> sum = strong ? any_backward<false, T, VEC, PACKED>(p, at, ln, sh, io, rt, entry, row0, live, warp)
                             : any_backward<true, T, VEC, PACKED>(p, at, ln, sh, io, rt, entry, row0, live, warp);
    if (p.part) {
        __syncthreads(); /* every warp is done with the states' maps */
        sh.states.H[warp][ln.lane] = to(sum);
        __syncthreads();
        for (int k = threadIdx.x; k < kC; k += blockDim.x) {
            float v = 0.f;
            for (int w = 0; w < warps; ++w) v += ((const float *)sh.states.H[w])[k];
            const int ch = VEC ? k : (k % kV) * 32 + k / kV;
            p.part[((long)at.pos * p.chains + at.chain) * kC + ch] = v;
        }
    }
    if (PACKED && tile0 == 0) empty_sequences(p.a, p.a.dh_last, p.a.dh0, ch0, ch0 + kC, warp, warps);
}

/* ------------------------------------------------------------------ */
/* resident kernels: tiles through a ring of tensor copies               */
/* ------------------------------------------------------------------ */

/*
 * For tensors that tensor copies can take, and enough tiles to fill the GPU.
 * Two or three CTAs an SM stay for the whole call.  Their last warp, the
 * feeder, takes tickets, brings tiles into a ring of stages by tensor copies,
 * prepares what depends on the channel (rates, the checkpoint) or the row
 * (which sequence), and stores the results, which the seven workers leave in
 * place of the inputs that they came from.  The workers own a run of rows
 * each, in shared memory at fixed offsets; the first of them also finds the
 * state that enters the tile, meanwhile the others (in the backward) work out
 * the states of their rows and all of the gradients but the factor that comes
 * along the chain.
 *
 * What bounds them: issue and latency.  A tile's terms are 23 instructions a
 * value in the forward (4 of them MUFU), and the trips to the L2 cache along
 * the chain are hidden by the other CTAs of the SM only.  Tried and left: four
 * channels a lane (128 registers, two CTAs; 130 against 105 us on 8 x 4096 x
 * 1536 bf16), a warp of its own for the chain with the next tile's terms
 * ahead (113), all warps looking at other tiles (111).
 */
constexpr int kW = 7; /* workers */
constexpr int kThreads = 32 * (kW + 1);

template <typename T, bool BWD>
struct Shape {
    static constexpr bool kHalf = sizeof(T) == 2;
    static constexpr int V = 2;                      /* channels of a lane */
    static constexpr int R = BWD && !kHalf ? 4 : 8;  /* rows of a worker */
    static constexpr int C = 32 * V, ROWS = R * kW;
    static constexpr int N = BWD ? 4 : 3;            /* tensors in */
    static constexpr int kTile = ROWS * C * (int)sizeof(T); /* bytes of one */
    static constexpr int kStage = N * kTile;
    static constexpr int kStages = 2;
    static constexpr int kCtas = BWD || !kHalf ? 2 : 3; /* an SM's: 128 or 80 registers a thread */
};
static_assert(Shape<float, true>::ROWS % KMB_GLR_CHUNK(KMB_F32) == 0 &&
                  Shape<__nv_bfloat16, true>::ROWS % KMB_GLR_CHUNK(KMB_BF16) == 0,
              "a tile begins at a checkpoint");

struct TensorMaps {
    CUtensorMap in[4], out[3]; /* x, gate_r, gate_i, dy; y or dx, dgate_r, dgate_i */
};

template <typename T, bool BWD, bool PACKED>
struct Stage { /* what the feeder prepares beside the tile, and the sums that it takes away */
    typedef Shape<T, BWD> S;
    typedef typename Pack<S::V>::type pack;
    pack rate[32], sroot[32], entry[32];
    Place at;
    int row, ch0; /* the tile's first */
    int strong, more;
    RowMap<PACKED ? S::ROWS : 1> rows;
    pack sums[BWD ? kW : 1][32];
    uint64_t full, done;
};

template <typename T, bool BWD, bool PACKED>
struct RingShared {
    typedef Shape<T, BWD> S;
    Stage<T, BWD, PACKED> stage[S::kStages];
    Maps<kW, S::V> agg, states; /* the workers' maps, of the recurrence and (backward) of the states */
    Maps<kRingWindow, S::V> seen;
    typename Pack<S::V>::type in[32]; /* what enters the tile */
};

/* barrier 1: the workers; 2: the first warp arrives, the others wait */
struct Workers {
    static __device__ __forceinline__ void sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kW) : "memory"); }
    static __device__ __forceinline__ bool any(bool p) {
        int r;
        asm volatile("{\n\t.reg .pred p, q;\n\t"
                     "setp.ne.b32 p, %1, 0;\n\t"
                     "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
                     "selp.b32 %0, 1, 0, q;\n\t}"
                     : "=r"(r)
                     : "r"((int)p), "n"(32 * kW)
                     : "memory");
        return r != 0;
    }
    static __device__ __forceinline__ void entered() { asm volatile("bar.arrive 2, %0;" ::"n"(32 * kW) : "memory"); }
    static __device__ __forceinline__ void enter() { asm volatile("bar.sync 2, %0;" ::"n"(32 * kW) : "memory"); }
};

/* a stage and the parity of its barriers' phase */
template <int N>
struct Turn {
    int k = 0, parity = 0;
    __device__ __forceinline__ void next() {
        if (++k == N) {
            k = 0;
            parity ^= 1;
        }
    }
};

__device__ __forceinline__ bool wait(uint64_t *bar, int parity) { return kmb_mbar_wait(bar, parity, &g_glr_error); }

__device__ __forceinline__ void tensor_load(void *dst, const CUtensorMap *m, int x, int y, int z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
                 "[%2];" ::"r"(kmb_smem(dst)),
                 "l"(m), "r"(kmb_smem(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void tensor_store(const CUtensorMap *m, int x, int y, int z, const void *src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(m),
                 "r"(kmb_smem(src)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}

template <typename T, bool BWD, bool PACKED>
__device__ __forceinline__ void feed(const Dev &p, const TensorMaps &tm, char *tiles, RingShared<T, BWD, PACKED> &sh) {
    typedef Shape<T, BWD> S;
    constexpr int N = S::kStages;
    const int lane = threadIdx.x % 32;
    const unsigned total = p.tiles * p.chains;
    /* the results of the tile in a stage leave it; false when a wait gave up */
    const auto leave = [&](const Turn<N> &t) {
        Stage<T, BWD, PACKED> &st = sh.stage[t.k];
        if (!wait(&st.done, t.parity)) return false;
        if (!p.states_only && (!PACKED || st.rows.whole) && lane == 0) {
            char *tile = tiles + t.k * S::kStage;
            for (int n = 0; n < (BWD ? 3 : 1); ++n)
                tensor_store(&tm.out[n], st.ch0, st.row, (int)st.at.b, tile + n * S::kTile);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        if (BWD && p.part) {
            F<S::V> v = all<S::V>(0.f);
            for (int w = 0; w < kW; ++w) v = v + from(st.sums[BWD ? w : 0][lane]);
            typedef typename Pack<S::V>::type pack;
            *reinterpret_cast<pack *>(p.part + ((long)st.at.pos * p.chains + st.at.chain) * S::C + S::V * lane) = to(v);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
        return true;
    };
    Turn<N> turn, out; /* the stage to fill, the oldest one that is in work */
    int held = 0;      /* stages filled */
    bool ok = true;
    for (;;) {
        if (held == N) {
            if (!(ok = leave(out))) break;
            out.next();
            --held;
        }
        Stage<T, BWD, PACKED> &st = sh.stage[turn.k];
        /* not before the stage is free: a tile that is held and not in work
         * keeps those behind it in the chain waiting */
        unsigned id = 0;
        if (lane == 0) id = take_ticket(p);
        id = __shfl_sync(~0u, id, 0);
        if (id >= total) {
            if (lane == 0) {
                st.more = 0;
                kmb_mbar_arrive(&st.full);
                kmb_mbar_arrive(&st.full);
            }
            break;
        }
        const Place at(p, id);
        const int row = (int)((BWD ? p.tiles - 1 - at.pos : at.pos) * (unsigned)S::ROWS), ch0 = (int)at.group * S::C;
        if (lane == 0) {
            char *tile = tiles + turn.k * S::kStage;
            kmb_mbar_expect(&st.full, S::kStage);
            for (int n = 0; n < S::N; ++n)
                tensor_load(tile + n * S::kTile, &tm.in[n], ch0, row, (int)at.b, &st.full);
            st.at = at;
            st.row = row;
            st.ch0 = ch0;
            st.more = 1;
        }
        const Lane<true, S::V> ln(ch0, p.a.D);
        float2 rs[S::V];
#pragma unroll
        for (int e = 0; e < S::V; ++e) rs[e] = p.rates[ch0 + S::V * lane + e];
        bool strong = false;
#pragma unroll
        for (int e = 0; e < S::V; ++e) strong |= !(rs[e].x <= kWeak);
        st.rate[lane] = to(each<S::V>([&](int e) { return rs[e].x; }));
        st.sroot[lane] = to(each<S::V>([&](int e) { return rs[e].y; }));
        if (BWD) st.entry[lane] = to(ln.at(row < p.a.L ? p.ckpt_in + (at.b * p.chunks + row / chunk_of<T>) * p.a.D : nullptr));
        strong = __any_sync(~0u, strong);
        if (lane == 0) st.strong = strong;
        if constexpr (PACKED) map_rows(st.rows, p.a, row);
        __syncwarp();
        if (lane == 0) kmb_mbar_arrive(&st.full);
        turn.next();
        ++held;
    }
    for (; ok && held; --held, out.next()) ok = leave(out);
    if (!ok) { /* copies that may still be under way land before the CTA ends, or a second goes by */
        const long long t0 = clock64();
        for (; held; --held, out.next())
            while (!kmb_mbar_done(&sh.stage[out.k].full, out.parity) && clock64() - t0 < (1ll << 31)) {
            }
    }
}

/* the lane's channels of the tile in shared memory, rows of the worker's run */
template <typename T, bool BWD>
struct TileIo {
    typedef Shape<T, BWD> S;
    typedef Raw<T, S::V> W;
    typedef typename W::type raw;
    static constexpr int kChunk = chunk_of<T>;
    static_assert(S::ROWS % kChunk == 0, "a tile begins at a checkpoint");
    raw *base;     /* row 0 of the run in the first tensor */
    const Dev *p;  /* rows go to global memory themselves when some are of no sequence */
    long b, row0;
    int lane_ch;   /* the lane's first channel */
    unsigned m;
    bool direct, skip;
    static __device__ __forceinline__ int mark(long, int warp) { /* a tile begins at a checkpoint */
        return (kChunk - warp * S::R % kChunk) % kChunk;
    }
    __device__ __forceinline__ raw *at(int n, int j) const {
        return base + (n * S::kTile + j * S::C * (int)sizeof(T)) / (int)sizeof(raw);
    }
    __device__ __forceinline__ F<S::V> x(int j) const { return W::f(*at(0, j)); }
    __device__ __forceinline__ F<S::V> gr(int j) const { return W::f(*at(1, j)); }
    __device__ __forceinline__ F<S::V> gi(int j) const { return W::f(*at(2, j)); }
    __device__ __forceinline__ F<S::V> dy(int j) const { return W::f(*at(3, j)); }
    __device__ __forceinline__ void out(int n, int j, F<S::V> v, const KmbRows &r) const {
        if (!direct) {
            *at(n, j) = W::r(v);
        } else if (m) {
            *reinterpret_cast<raw *>((T *)r.data + b * r.batch_stride + (row0 + j) * r.row_stride + lane_ch) = W::r(v);
        }
    }
    __device__ __forceinline__ void y(int j, F<S::V> v) const {
        if (!skip) out(0, j, v, p->a.y);
    }
    __device__ __forceinline__ void grads(int j, F<S::V> x, F<S::V> r, F<S::V> i) const {
        out(0, j, x, p->a.dx);
        out(1, j, r, p->a.dgate_r);
        out(2, j, i, p->a.dgate_i);
    }
};

template <bool B>
struct Const {};
/* f(Const<FULL>, Const<WEAK>) for the tile's kind */
template <typename Fn>
__device__ __forceinline__ void by_kind(bool full, bool strong, Fn f) {
    if (strong) {
        if (full) f(Const<true>(), Const<false>());
        else f(Const<false>(), Const<false>());
    } else {
        if (full) f(Const<true>(), Const<true>());
        else f(Const<false>(), Const<true>());
    }
}

/* A worker's place in a tile. */
template <typename T, bool BWD, bool PACKED>
struct Bench {
    typedef Shape<T, BWD> S;
    static constexpr int V = S::V, R = S::R;
    const Dev &p;
    Stage<T, BWD, PACKED> &st;
    Lane<true, V> ln;
    TileIo<T, BWD> io;
    Place at;
    int worker, live;
    bool full;

    __device__ __forceinline__ Bench(const Dev &d, char *tile, Stage<T, BWD, PACKED> &s, int w)
        : p(d), st(s), ln(s.ch0, d.a.D), at(s.at), worker(w) {
        const int row0 = st.row + worker * R, left = (int)p.a.L - row0;
        live = left < 0 ? 0 : left < R ? left : R;
        full = st.row + S::ROWS <= p.a.L;
        io.direct = false;
        if constexpr (PACKED) {
            full = st.rows.plain;
            io.direct = !st.rows.whole;
        }
        io.base = reinterpret_cast<typename TileIo<T, BWD>::raw *>(tile + (worker * R * S::C + ln.lane * V) * (int)sizeof(T));
        io.p = &p;
        io.b = at.b;
        io.row0 = row0;
        io.lane_ch = (int)ln.d;
        io.m = ln.m;
        io.skip = p.states_only;
    }
    template <bool FULL, bool WEAK>
    using Rows = RunOf<TileIo<T, BWD>, true, PACKED, FULL, WEAK, R, PACKED ? S::ROWS : 1, V>;
    template <bool FULL, bool WEAK>
    __device__ __forceinline__ Rows<FULL, WEAK> run(Const<FULL>, Const<WEAK>) {
        return {p, at, ln, st.rows, io, io.row0, live, worker};
    }
    __device__ __forceinline__ Rates<V> rates() const { return {from(st.rate[ln.lane]), from(st.sroot[ln.lane])}; }
    /* by the first worker, when all maps are there */
    __device__ __forceinline__ void enter(RingShared<T, BWD, PACKED> &sh) {
        Map<V> m = sh.agg.at(BWD ? kW - 1 : 0, ln.lane);
        for (int k = 1; k < kW; ++k) m = join<PACKED>(m, sh.agg.at(BWD ? kW - 1 - k : k, ln.lane));
        const float *first = BWD ? p.a.dh_last : p.a.h0;
        first = !PACKED && first ? first + at.b * p.a.D : nullptr;
        sh.in[ln.lane] = to(enter_chain<PACKED>(p, at, ln, m, sh.seen, first));
        Workers::entered();
    }
    __device__ __forceinline__ void finish() {
        if (PACKED && st.row == 0 && !p.states_only)
            empty_sequences(p.a, BWD ? p.a.dh_last : p.a.h0, BWD ? p.a.dh0 : p.a.h_last, st.ch0, st.ch0 + S::C, worker, kW);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); /* the results, for the tensor stores */
        __syncwarp();
        if (ln.lane == 0) kmb_mbar_arrive(&st.done);
    }
};

template <typename T, bool BWD, bool PACKED>
__device__ __forceinline__ void work(const Dev &p, char *tiles, RingShared<T, BWD, PACKED> &sh, int worker) {
    typedef Shape<T, BWD> S;
    constexpr int V = S::V, R = S::R;
    for (Turn<S::kStages> t;; t.next()) {
        Stage<T, BWD, PACKED> &st = sh.stage[t.k];
        /* all go on or none; and all are done with the maps of the tile before */
        if (Workers::any(!wait(&st.full, t.parity)) || !st.more) return;
        Bench<T, BWD, PACKED> bench(p, tiles + t.k * S::kStage, st, worker);
        const int lane = bench.ln.lane;
        by_kind(bench.full, st.strong, [&](auto full, auto weak) {
            const auto run = bench.run(full, weak);
            if constexpr (BWD) {
                Terms<V> x[R];
                F<V> f[R], ends[R];
                {
                    Map<V> state, adjoint;
                    run.backward_maps(bench.rates(), x, ends, state, adjoint);
                    sh.states.put(worker, lane, state.A, state.H);
                    sh.agg.put(worker, lane, adjoint.A, adjoint.H);
                }
                Workers::sync();
                if (worker == 0) bench.enter(sh);
                F<V> h = from(st.entry[lane]);
                for (int w = 0; w < worker; ++w) h = apply<PACKED>(sh.states.at(w, lane), h);
                run.backward_factors(h, from(st.rate[lane]), x, f);
                if (worker != 0) Workers::enter();
                F<V> C = from(sh.in[lane]);
                for (int w = kW - 1; w > worker; --w) C = apply<PACKED>(sh.agg.at(w, lane), C);
                st.sums[worker][lane] = to(run.backward_rows(C, x, ends, f));
            } else {
                F<V> c[R], b[R];
                {
                    const Map<V> m = run.forward_map(bench.rates(), c, b);
                    sh.agg.put(worker, lane, m.A, m.H);
                }
                Workers::sync();
                if (worker == 0) bench.enter(sh);
                else Workers::enter();
                F<V> h = from(sh.in[lane]);
                for (int w = 0; w < worker; ++w) h = apply<PACKED>(sh.agg.at(w, lane), h);
                run.forward_rows(h, c, b);
            }
        });
        bench.finish();
    }
}

template <typename T, bool BWD, bool PACKED>
__global__ void __launch_bounds__(kThreads, (Shape<T, BWD>::kCtas)) k_glr_ring(const __grid_constant__ Dev p,
                                                                           const __grid_constant__ TensorMaps tm) {
    typedef Shape<T, BWD> S;
    extern __shared__ __align__(128) char tiles[];
    RingShared<T, BWD, PACKED> &sh = *reinterpret_cast<RingShared<T, BWD, PACKED> *>(tiles + S::kStages * S::kStage);
    kmb_wait_before();
    const int warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        for (int k = 0; k < S::kStages; ++k) {
            kmb_mbar_init(&sh.stage[k].full, 2);
            kmb_mbar_init(&sh.stage[k].done, kW);
        }
        kmb_mbar_init_fence();
    }
    __syncthreads();
    if (warp == kW) feed(p, tm, tiles, sh);
    else work(p, tiles, sh, warp);
}

/* ddecay: the sums of all tiles and sequences, 32 columns a CTA, 32 rows of
 * threads, joined in a fixed order. */
__global__ void __launch_bounds__(1024) k_glr_ddecay(const float *part, long rows, long ld, long D,
                                                     const float *decay, float *ddecay, int acc) {
    __shared__ float s[32][33];
    kmb_wait_before();
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

/* Before a call whose chains have several tiles: fills the shown arrays and
 * the ticket, and works out the channels' rates (0 beyond the last). */
__global__ void __launch_bounds__(256) k_glr_begin(uint4 *fill, long n, float2 *rates, long channels, long D,
                                                   const float *decay, float scale) {
    kmb_let_after();
    const long at = (long)blockIdx.x * 256 + threadIdx.x, step = (long)gridDim.x * 256;
    for (long k = at; k < n; k += step) fill[k] = make_uint4(kUnset, kUnset, kUnset, kUnset);
    for (long c = at; c < channels; c += step) {
        const float r = c < D ? scale * softplus(decay[c]) : 0.f;
        rates[c] = make_float2(r, sqrtf(2.f * r));
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

/*
 * A thread has W channels of a row (4 where the tensors allow vectors).  A
 * row whose slot an earlier row names is left out: the threads of the CTA
 * look for it among the slots before, while their channels are on their way.
 * Memory bounds it, and for a handful of rows the trips to memory: slot, then
 * state.
 */
template <typename T, int W>
__global__ void __launch_bounds__(kStepThreads) k_glr_step(const __grid_constant__ KmbGLRStep a, unsigned tiles) {
    const unsigned k = blockIdx.x / tiles;
    const long slot = a.slots ? a.slots[k] : (long)k;
    if (slot < 0 || slot >= a.n_states) return;
    const long d = ((long)(blockIdx.x - k * tiles) * kStepThreads + threadIdx.x) * W;
    const bool in = d < a.D;
    float x[W], gr[W], gi[W], h[W], rate[W];
    const auto fetch = [&](const KmbRows &r, float (&v)[W]) {
        const T *p = (const T *)r.data + k * r.row_stride + d;
        if constexpr (W == 1) {
            v[0] = (float)*p;
        } else if constexpr (sizeof(T) == 4) {
            const float4 u = __ldcs(reinterpret_cast<const float4 *>(p));
            v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
        } else {
            const uint2 u = __ldcs(reinterpret_cast<const uint2 *>(p));
            const float2 l = unpack(u.x), m = unpack(u.y);
            v[0] = l.x, v[1] = l.y, v[2] = m.x, v[3] = m.y;
        }
    };
    float *s = a.state + slot * a.ld_state + d;
    if (in) {
        fetch(a.gate_r, gr);
        fetch(a.gate_i, gi);
        fetch(a.x, x);
        if constexpr (W == 4) {
            const float4 u = *reinterpret_cast<const float4 *>(s);
            h[0] = u.x, h[1] = u.y, h[2] = u.z, h[3] = u.w;
        } else {
            h[0] = *s;
        }
#pragma unroll
        for (int e = 0; e < W; ++e) rate[e] = a.scale * softplus(a.decay[d + e]);
    }
    if (a.slots) {
        int taken = 0;
        for (unsigned j = threadIdx.x; j < k; j += kStepThreads) taken |= a.slots[j] == slot;
        if (__syncthreads_or(taken)) return;
    }
    if (!in) return;
#pragma unroll
    for (int e = 0; e < W; ++e) {
        const Rates<2> rt = {all<2>(rate[e]), all<2>(sqrtf(2.f * rate[e]))};
        if (rate[e] <= kWeak) {
            const Terms<2> t = terms<true>(all<2>(gr[e]), all<2>(gi[e]), rt);
            h[e] = advance<true>(t.c, all<2>(h[e]), t.si * all<2>(x[e]))[0];
        } else {
            const Terms<2> t = terms<false>(all<2>(gr[e]), all<2>(gi[e]), rt);
            h[e] = advance<false>(t.c, all<2>(h[e]), t.si * all<2>(x[e]))[0];
        }
    }
    T *y = (T *)a.y.data + k * a.y.row_stride + d;
    if constexpr (W == 1) {
        *s = h[0];
        *y = (T)h[0];
    } else {
        *reinterpret_cast<float4 *>(s) = make_float4(h[0], h[1], h[2], h[3]);
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(y) = make_float4(h[0], h[1], h[2], h[3]);
        } else {
            *reinterpret_cast<uint2 *>(y) = make_uint2(pack(kmb_f2(h[0], h[1])), pack(kmb_f2(h[2], h[3])));
        }
    }
}

/* ------------------------------------------------------------------ */
/* launches                                                             */
/* ------------------------------------------------------------------ */

int started(cudaError_t e) { return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, "glr: launch"); }
int done(const char *what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KMB_OK : kmb_cuda_fail(e, what);
}

/* Whether the tensors allow two channels an access: width, strides and
 * addresses are multiples of two elements. */
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

/* Tiles and their order for one of the kernels. */
struct Plan {
    long tiles, groups, batch, chains;
    int rows, channels;
    bool ring;
    size_t words; /* of each of the three shown arrays */
};

Plan plan(const KmbGLR *a, int rows, int channels) {
    Plan q;
    q.rows = rows;
    q.channels = channels;
    q.ring = false;
    q.tiles = (a->L + rows - 1) / rows;
    if (a->offsets && q.tiles == 0) q.tiles = 1; /* for the empty sequences */
    q.groups = (a->D + channels - 1) / channels;
    q.batch = a->offsets ? 1 : a->batch;
    q.chains = q.groups * q.batch;
    q.words = q.tiles > 1 ? (size_t)q.tiles * q.chains * channels : 0;
    return q;
}

constexpr int kSMs = 148;

/* Whether tensor copies can take the tensor: whole 16-byte pieces, batch
 * after batch, coordinates of 32 bits. */
bool tensor_ok(const KmbGLR *a, const KmbRows &r) {
    const long es = a->type == KMB_BF16 ? 2 : 4;
    if ((size_t)r.data % 16 || r.row_stride * es % 16 || r.row_stride * es >= (1L << 40)) return false;
    if (a->offsets || a->batch <= 1) return true;
    return r.batch_stride * es % 16 == 0 && r.batch_stride >= a->L * r.row_stride && r.batch_stride * es < (1L << 40);
}

/*
 * The plan of a direction: the resident kernel where the tensors allow it
 * and there is a tile for each SM, else the kernel for any alignment, one CTA
 * a tile.  Below that the two are close, above it the resident one gains.
 * Forward + backward, by threads and resident, us (tiles of the forward):
 *   1 x 1024 x 128 (38)     fp32  9.1 + 14.4, 10.3 + 13.3   bf16  8.8 + 12.4, 10.3 + 12.4
 *   1 x 1024 x 512 (152)    fp32 10.3 + 16.5, 10.3 + 14.6   bf16 10.2 + 14.4, 10.3 + 14.0
 *   4 x 1024 x 256 (304)    fp32 10.6 + 20.4, 12.3 + 18.5   bf16 10.3 + 16.5, 12.0 + 16.2
 *   1 x 16384 x 128 (586)   fp32 39.0 + 91.4, 26.7 + 52.9   bf16 37.4 + 48.9, 25.4 + 31.9
 *   8 x 1024 x 512 (1216)   fp32 22.6 + 43.0, 22.6 + 38.5   bf16 20.5 + 41.0, 18.6 + 28.5
 */
template <typename T>
Plan plan_of(const KmbGLR *a, bool bwd) {
    const Plan any = bwd ? plan(a, kBT<T>, kC) : plan(a, kFT, kC);
    const KmbRows fwd_rows[] = {a->x, a->gate_r, a->gate_i, a->y};
    const KmbRows bwd_rows[] = {a->x, a->gate_r, a->gate_i, a->dy, a->dx, a->dgate_r, a->dgate_i};
    Plan q = bwd ? plan(a, Shape<T, true>::ROWS, Shape<T, true>::C) : plan(a, Shape<T, false>::ROWS, Shape<T, false>::C);
    if (a->D % 4 || a->L >= (1L << 31) - 1024 || q.tiles < 2 || q.tiles * q.chains < kSMs) return any;
    if (q.tiles * q.chains >= (1L << 31)) return any;
    for (int i = 0; i < (bwd ? 7 : 4); ++i) {
        const KmbRows &r = bwd ? bwd_rows[i] : fwd_rows[i];
        if (r.data && !tensor_ok(a, r)) return any;
    }
    q.ring = true;
    return q;
}
Plan plan_of(const KmbGLR *a, bool bwd) {
    return a->type == KMB_BF16 ? plan_of<__nv_bfloat16>(a, bwd) : plan_of<float>(a, bwd);
}

constexpr size_t kHead = 64; /* bytes before the shown arrays: the ticket */

size_t shown_bytes(const Plan &q) { return q.words ? kHead + 12 * q.words + 8 * (size_t)q.groups * q.channels : 0; }
/* for either kernel, whatever the pointers turn out to be */
size_t shown_most(const KmbGLR *a, bool bwd) {
    const bool half = a->type == KMB_BF16;
    const Plan any = bwd ? plan(a, half ? kBT<__nv_bfloat16> : kBT<float>, kC) : plan(a, kFT, kC);
    const Plan ring = bwd ? (half ? plan(a, Shape<__nv_bfloat16, true>::ROWS, Shape<__nv_bfloat16, true>::C)
                                  : plan(a, Shape<float, true>::ROWS, Shape<float, true>::C))
                          : (half ? plan(a, Shape<__nv_bfloat16, false>::ROWS, Shape<__nv_bfloat16, false>::C)
                                  : plan(a, Shape<float, false>::ROWS, Shape<float, false>::C));
    const size_t m = shown_bytes(any), n = shown_bytes(ring);
    return m > n ? m : n;
}
size_t part_most(const KmbGLR *a) {
    const Plan any = plan(a, a->type == KMB_BF16 ? kBT<__nv_bfloat16> : kBT<float>, kC);
    const Plan ring = a->type == KMB_BF16 ? plan(a, Shape<__nv_bfloat16, true>::ROWS, Shape<__nv_bfloat16, true>::C)
                                          : plan(a, Shape<float, true>::ROWS, Shape<float, true>::C);
    const size_t m = (size_t)any.tiles * any.chains * kC, n = (size_t)ring.tiles * ring.chains * ring.channels;
    return 4 * (m > n ? m : n);
}

/* Fills the workspace's shown arrays and sets the pointers. */
int begin(Dev &d, const Plan &q, void *ws, cudaStream_t s) {
    if (q.tiles >= (1L << 31) / q.chains) return kmb_fail(KMB_EUNSUPPORTED, "glr: too many tiles");
    d.tiles = (unsigned)q.tiles;
    d.groups = (unsigned)q.groups;
    d.chains = (unsigned)q.chains;
    const long chunk = KMB_GLR_CHUNK(d.a.type);
    d.chunks = (d.a.L + chunk - 1) / chunk;
    if (!q.words) return KMB_OK;
    const long n = (long)(kHead + 12 * q.words) / 16, channels = q.ring ? q.groups * q.channels : 0;
    float2 *rates = (float2 *)((char *)ws + kHead + 12 * q.words);
    const long blocks = ((n > channels ? n : channels) + 255) / 256;
    k_glr_begin<<<(unsigned)(blocks < 8 * kSMs ? blocks : 8 * kSMs), 256, 0, s>>>((uint4 *)ws, n, rates, channels,
                                                                                 d.a.D, d.a.decay, d.a.scale);
    const int rc = done("glr: launch");
    if (rc) return rc;
    d.rates = rates;
    d.ticket = (unsigned *)ws;
    d.shown.A = (float *)((char *)ws + kHead);
    d.shown.H = d.shown.A + q.words;
    d.shown.end = d.shown.H + q.words;
    d.shown.step = q.chains * 32;
    return KMB_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
        else
            (void)cudaGetLastError();
    }
    return fn;
}

/* [batch, L, D] with boxes of rows x channels; outside, loads give zeros and
 * stores do nothing */
int tensor_map(CUtensorMap *m, const KmbGLR &a, const KmbRows &r, const Plan &q) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return kmb_fail(KMB_ECUDA, "glr: cuTensorMapEncodeTiled unavailable");
    const cuuint64_t es = a.type == KMB_BF16 ? 2 : 4;
    const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.L, (cuuint64_t)q.batch};
    const cuuint64_t batch = q.batch > 1 ? (cuuint64_t)r.batch_stride * es : (cuuint64_t)a.L * r.row_stride * es;
    const cuuint64_t strides[2] = {(cuuint64_t)r.row_stride * es, batch};
    const cuuint32_t box[3] = {(cuuint32_t)q.channels, (cuuint32_t)q.rows, 1}, one[3] = {1, 1, 1};
    const CUresult rc = fn(m, a.type == KMB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                           3, r.data, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? KMB_OK : kmb_fail(KMB_EINVAL, "glr: tensor map rejected (CUresult %d)", (int)rc);
}

template <typename T, bool BWD, bool PACKED>
int launch_ring(const Dev &d, const Plan &q, const TensorMaps &tm, cudaStream_t s) {
    typedef Shape<T, BWD> S;
    auto k = k_glr_ring<T, BWD, PACKED>;
    const size_t bytes = S::kStages * S::kStage + sizeof(RingShared<T, BWD, PACKED>);
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return kmb_cuda_fail(e, "glr: shared memory");
    const long n = q.tiles * q.chains;
    const long most = (long)S::kCtas * kSMs;
    return started(kmb_launch_after(d.ticket != nullptr, k, (unsigned)(n < most ? n : most), kThreads, bytes, s, d, tm));
}

template <typename T>
int launch(const Dev &d, const Plan &q, bool bwd, bool vec, cudaStream_t s) {
    const bool packed = d.a.offsets != nullptr;
    if (q.ring) {
        TensorMaps tm;
        const KmbRows in[] = {d.a.x, d.a.gate_r, d.a.gate_i, d.a.dy};
        const KmbRows out[] = {bwd ? d.a.dx : d.a.y, d.a.dgate_r, d.a.dgate_i};
        for (int i = 0; i < (bwd ? 4 : 3); ++i) {
            const int rc = tensor_map(&tm.in[i], d.a, in[i], q);
            if (rc) return rc;
        }
        for (int i = 0; i < (bwd ? 3 : d.states_only ? 0 : 1); ++i) {
            const int rc = tensor_map(&tm.out[i], d.a, out[i], q);
            if (rc) return rc;
        }
        if (bwd) return packed ? launch_ring<T, true, true>(d, q, tm, s) : launch_ring<T, true, false>(d, q, tm, s);
        return packed ? launch_ring<T, false, true>(d, q, tm, s) : launch_ring<T, false, false>(d, q, tm, s);
    }
    const unsigned n = (unsigned)(q.tiles * q.chains);
    const int most = bwd ? kBW : kFW;
    const long run = bwd ? kBR<T> : kFR, runs = (d.a.L + run - 1) / run;
    const unsigned threads = 32u * (unsigned)(runs < 1 ? 1 : runs < most ? runs : most);
    if (bwd) {
        auto k = packed ? (vec ? k_glr_bwd<T, true, true> : k_glr_bwd<T, false, true>)
                        : (vec ? k_glr_bwd<T, true, false> : k_glr_bwd<T, false, false>);
        return started(kmb_launch_after(d.ticket != nullptr, k, n, threads, 0, s, d));
    } else {
        auto k = packed ? (vec ? k_glr_fwd<T, true, true> : k_glr_fwd<T, false, true>)
                        : (vec ? k_glr_fwd<T, true, false> : k_glr_fwd<T, false, false>);
        return started(kmb_launch_after(d.ticket != nullptr, k, n, threads, 0, s, d));
    }
}
int launch(const Dev &d, const Plan &q, bool bwd, bool vec, cudaStream_t s) {
    return d.a.type == KMB_BF16 ? launch<__nv_bfloat16>(d, q, bwd, vec, s) : launch<float>(d, q, bwd, vec, s);
}

/* packed rows have no batch */
void drop_batch(KmbGLR &a) {
    KmbRows *const all[] = {&a.x, &a.gate_r, &a.gate_i, &a.y, &a.dy, &a.dx, &a.dgate_r, &a.dgate_i};
    if (a.offsets)
        for (KmbRows *r : all) r->batch_stride = 0;
}

int run_fwd(const KmbGLR *a, float *ckpt, bool write_y, void *ws, cudaStream_t s) {
    Dev d = {};
    d.a = *a;
    if (!write_y) {
        d.states_only = 1;
        d.a.y.data = nullptr;
        d.a.h_last = nullptr;
    }
    drop_batch(d.a);
    const Plan q = plan_of(&d.a, false);
    d.ckpt_out = ckpt;
    const int rc = begin(d, q, ws, s);
    if (rc) return rc;
    const KmbRows *rows[] = {&d.a.x, &d.a.gate_r, &d.a.gate_i, &d.a.y};
    return launch(d, q, false, vectors(&d.a, rows, 4), s);
}

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

} // namespace

/* Backward workspace: shown arrays (the state run and the adjoint use them
 * one after the other) | sums of the tiles | checkpoints. */
extern "C" size_t kmb_glr_scratch_bytes(const KmbGLR *a, int bwd) {
    if (a->batch == 0 || (a->L == 0 && !a->offsets)) return 0;
    const size_t f = shown_most(a, false);
    if (!bwd) return f;
    const size_t b = shown_most(a, true);
    size_t n = align16(a->ckpt || f < b ? b : f);
    if (a->ddecay) n += align16(part_most(a));
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
    const size_t f = shown_most(a, false), b = shown_most(a, true);
    char *ws = (char *)a->workspace;
    size_t o = align16(a->ckpt || f < b ? b : f);
    Dev d = {};
    d.a = *a;
    drop_batch(d.a);
    const Plan q = plan_of(&d.a, true);
    if (a->ddecay) {
        d.part = (float *)(ws + o);
        o += align16(part_most(a));
    }
    d.ckpt_in = a->ckpt;
    int rc;
    if (!a->ckpt) {
        d.ckpt_in = (float *)(ws + o);
        if (a->L && (rc = run_fwd(a, (float *)(ws + o), false, ws, s))) return rc;
    }
    if ((rc = begin(d, q, ws, s))) return rc;
    const KmbRows *rows[] = {&d.a.x, &d.a.gate_r, &d.a.gate_i, &d.a.dy, &d.a.dx, &d.a.dgate_r, &d.a.dgate_i};
    rc = launch(d, q, true, vectors(&d.a, rows, 7), s);
    if (rc || !a->ddecay) return rc;
    return started(kmb_launch_after(true, k_glr_ddecay, (unsigned)((a->D + 31) / 32), dim3(32, 32), 0, s,
                                    (const float *)d.part, q.tiles * q.batch, q.groups * q.channels, a->D, a->decay,
                                    a->ddecay, a->accumulate));
}

template <typename T>
static int launch_step(const KmbGLRStep *a, cudaStream_t s) {
    const long es = sizeof(T);
    bool vec = a->D % 4 == 0 && (size_t)a->state % 16 == 0 && a->ld_state % 4 == 0;
    for (const KmbRows *r : {&a->x, &a->gate_r, &a->gate_i, &a->y})
        vec = vec && (size_t)r->data % (4 * es) == 0 && r->row_stride % 4 == 0;
    /* A few rows are a matter of latency: one channel a thread.  Scalars and
     * vectors, us: 64 x 1536 4.2 both, 128 x 1536 fp32 4.2 and 5.1, 64 x 4096
     * 6.2 and 5.2, 256 x 1536 6.2 both, 512 x 1024 8.2 and 6.2; of narrow rows
     * vectors leave most of a CTA without work: 2000 x 128 6.2 and 8.2. */
    if (a->rows * a->D < 4L * kSMs * kStepThreads) vec = false;
    const long per = kStepThreads * (vec ? 4 : 1), tiles = (a->D + per - 1) / per;
    if (a->rows >= (1L << 31) / tiles) return kmb_fail(KMB_EUNSUPPORTED, "glr: too many rows");
    const unsigned n = (unsigned)(a->rows * tiles);
    if (vec) k_glr_step<T, 4><<<n, kStepThreads, 0, s>>>(*a, (unsigned)tiles);
    else k_glr_step<T, 1><<<n, kStepThreads, 0, s>>>(*a, (unsigned)tiles);
    return done("glr: step launch");
}

extern "C" int kmb_launch_glr_step(const KmbGLRStep *a, cudaStream_t s) {
    return a->type == KMB_BF16 ? launch_step<__nv_bfloat16>(a, s) : launch_step<float>(a, s);
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
