"""GPU parity of the gated linear recurrence (kmb_glr_fwd / _bwd / _step)
with its float64 definition.  Tolerances: the first-order bounds of
oracle/recurrent_ref.py, carried through the recurrence entry by entry, plus
half a step of bf16 outputs."""
import ctypes as C

import numpy as np
import pytest
import torch

import kmamba_b200 as kb
import recurrent_ref as ref
from recurrent_util import SENTINEL, Banded, byref, typed, within

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
TYPE = {F32: kb.KMB_F32, BF16: kb.KMB_BF16}
IN = ("x", "gate_r", "gate_i", "dy")
OUT = ("y", "dx", "dgate_r", "dgate_i")


def f32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda()


def decays(rng, D, kind="mixed"):
    """mixed: memories of a few to a few thousand steps, with channels that
    forget within a step; slow: every channel near 1."""
    lo = 0.9 if kind == "slow" else 0.5
    a = rng.uniform(lo, 0.999, D)
    d = np.log(np.expm1(-np.log(a) / 8.0))
    if kind == "mixed":
        d[::5] = rng.uniform(-1.0, 3.0, d[::5].shape)
    return typed(d, F32)


class Case:
    """offsets: packed rows (L = capacity); else batch sequences of L rows."""

    def __init__(self, batch, L, D, dtype=F32, offsets=None, gap=0, shift=0, time_major=False, seed=0,
                 h0=True, kind="mixed", scale=8.0, values=None):
        rng = np.random.default_rng(seed)
        self.batch, self.L, self.D, self.dtype, self.scale = batch, L, D, dtype, scale
        self.off = None if offsets is None else np.asarray(offsets, np.int64)
        shape = (L, D) if offsets is not None else (batch, L, D)
        self.v = {k: typed(rng.standard_normal(shape), dtype) for k in IN}
        for k, f in (values or {}).items():
            self.v[k] = typed(f(self.v[k]), dtype)
        mk = lambda fill: Banded(shape, dtype, fill, gap, shift, time_major)  # noqa: E731
        for k in IN:
            setattr(self, k, mk(float("nan")).set(self.v[k]))
        for k in OUT:
            setattr(self, k, mk(SENTINEL))
        self.decay = decays(rng, D, kind)
        self.h0v = typed(rng.standard_normal((batch, D)), F32) if h0 else None
        self.dlv = typed(rng.standard_normal((batch, D)), F32) if h0 else None
        self.t = {"decay": f32(self.decay)}
        if h0:
            self.t["h0"], self.t["dh_last"] = f32(self.h0v), f32(self.dlv)
        for k, s in (("h_last", (batch, D)), ("dh0", (batch, D)), ("ddecay", (D,))):
            self.t[k] = torch.full(s, SENTINEL, device="cuda")
        if self.off is not None:
            self.t["offsets"] = torch.from_numpy(self.off).cuda()

    def args(self):
        a = kb.KmbGLR()
        for k in IN + OUT:
            setattr(a, k, getattr(self, k).rows())
        for k, t in self.t.items():
            setattr(a, k, t.data_ptr())
        a.batch, a.L, a.D, a.scale, a.type = self.batch, self.L, self.D, self.scale, TYPE[self.dtype]
        return a

    def ref(self, grads=True):
        flat = lambda a: a.reshape(-1, self.D)  # noqa: E731
        seqs = ref.sequences(self.batch, self.L, self.off)
        v, e = ref.glr(flat(self.v["x"]), flat(self.v["gate_r"]), flat(self.v["gate_i"]), self.decay,
                       self.scale, seqs, self.h0v, flat(self.v["dy"]) if grads else None, self.dlv)
        self.inside = np.zeros(flat(self.v["x"]).shape[0], bool)
        for lo, hi in seqs:
            self.inside[lo:hi] = True
        return v, e

    def check(self, v, e, names):
        for k in names:
            if k in OUT:
                got = getattr(self, k).np().reshape(-1, self.D)
                within(k, got[self.inside], v[k][self.inside], e[k][self.inside], self.dtype)
                # rows of no sequence, and everything around the tensor, as they were
                assert np.all(got[~self.inside] == SENTINEL), k
                assert getattr(self, k).untouched_outside(), k
            else:
                within(k, self.t[k].double().cpu().numpy(), v[k], e[k])


def workspace(lib, a, bwd):
    n = lib.kmb_glr_workspace_bytes(byref(a), bwd)
    w = torch.full((max(n, 16),), 85, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = w.data_ptr(), n
    return w


def run(lib, c, ckpt=True, ws=True, bwd=True):
    a = c.args()
    keep = []
    if ckpt:
        c.ckpt = torch.full((max(1, lib.kmb_glr_ckpt_elems(byref(a))),), SENTINEL, device="cuda")
        a.ckpt = c.ckpt.data_ptr()
    if ws:
        keep.append(workspace(lib, a, 0))
    kb.check(lib, lib.kmb_glr_fwd(byref(a)))
    if bwd:
        if ws:
            keep.append(workspace(lib, a, 1))
        kb.check(lib, lib.kmb_glr_bwd(byref(a)))
    torch.cuda.synchronize()
    return a


ALL = ("y", "h_last", "dx", "dgate_r", "dgate_i", "dh0", "ddecay")

# one row, runs and tiles of rows that end inside, at and behind every boundary
LENGTHS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 191, 193, 300, 511, 513]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", LENGTHS)
def test_lengths(lib, cuda, L, dtype):
    c = Case(2, L, 70, dtype, seed=L)
    run(lib, c)
    c.check(*c.ref(), ALL)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1, 2, 3, 5, 8, 31, 32, 33, 62, 63, 64, 65, 66, 127, 128, 130, 192, 257])
def test_widths(lib, cuda, D, dtype):
    for gap, shift in ((0, 0), (1, 0), (3, 1), (8, 0)):
        c = Case(3, 75, D, dtype, gap=gap, shift=shift, seed=D)
        run(lib, c)
        c.check(*c.ref(), ALL)


@pytest.mark.parametrize("kind", ["mixed", "slow"])
@pytest.mark.parametrize("batch,L,D,dtype", [(1, 4000, 64, F32), (1, 9001, 33, BF16), (3, 2049, 130, F32),
                                             (700, 70, 8, F32), (2, 1000, 700, BF16)])
def test_many_tiles(lib, cuda, batch, L, D, dtype, kind):
    c = Case(batch, L, D, dtype, seed=L, kind=kind)
    run(lib, c)
    c.check(*c.ref(), ALL)


# aligned tensors with more tiles than SMs: the resident kernels
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["mixed", "slow"])
@pytest.mark.parametrize("batch,L,D", [(2, 1500, 512), (1, 5600, 516), (3, 1121, 260), (40, 113, 256), (1, 5599, 384),
                                       (20, 57, 1032)])
def test_resident_kernels(lib, cuda, batch, L, D, kind, dtype):
    for gap in (0, 8):
        c = Case(batch, L, D, dtype, seed=L, kind=kind, gap=gap)
        run(lib, c, ckpt=gap == 0)
        c.check(*c.ref(), ALL)


def ragged(rng, n, total, gap=0):
    cuts = np.sort(rng.integers(gap, total - gap + 1, n + 1))
    return cuts.astype(np.int64)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [256, 516])
@pytest.mark.parametrize("off,tail", [
    ([0, 5600], 0), ([0, 5600], 1), ([0, 0, 56, 112, 112, 3000, 5599, 5600], 0), ([70, 71, 72, 4000, 5500], 117),
    ([0, 28, 28, 84, 140, 141, 5600], 500), ("ragged", 300), ("many", 0)])
def test_resident_kernels_packed(lib, cuda, off, tail, D, dtype):
    """Sequences that begin and end at and inside tiles; rows of no sequence
    before, behind and in whole tiles."""
    rng = np.random.default_rng(D)
    if off == "ragged":
        off = ragged(rng, 30, 5700, 60)
    elif off == "many":
        off = np.concatenate([[0], np.cumsum(np.minimum(rng.geometric(0.05, 400) - 1, 90))])
    c = Case(len(off) - 1, int(off[-1]) + tail, D, dtype, offsets=off, seed=D, kind="slow" if tail else "mixed")
    run(lib, c)
    c.check(*c.ref(), ALL)


@pytest.mark.parametrize("packed", [False, True])
def test_resident_kernels_in_place_and_same_bits(lib, cuda, packed):
    for dtype in (F32, BF16):
        off = [0, 100, 2900, 2900, 4000] if packed else None
        mk = lambda: Case(4, 4000 if packed else 1000, 512, dtype, offsets=off, seed=9)  # noqa: E731
        c = mk()
        run(lib, c)
        v, e = c.ref()
        c.check(v, e, ALL)
        first = {k: getattr(c, k).t.clone() for k in OUT} | {k: c.t[k].clone() for k in ("h_last", "dh0", "ddecay")}
        for _ in range(4):
            run(lib, c)
            for k, t in first.items():
                assert torch.equal(t, getattr(c, k).t if k in OUT else c.t[k]), k
        d = mk()
        a = d.args()
        d.ckpt = torch.empty(lib.kmb_glr_ckpt_elems(byref(a)), device="cuda")
        a.ckpt, a.dx, a.dgate_r, a.dgate_i = d.ckpt.data_ptr(), a.x, a.gate_r, a.gate_i
        kb.check(lib, lib.kmb_glr_fwd(byref(a)))
        kb.check(lib, lib.kmb_glr_bwd(byref(a)))
        for k, o in (("dx", d.x), ("dgate_r", d.gate_r), ("dgate_i", d.gate_i)):
            assert torch.equal(o.t, first[k]), k
        d = mk()
        a = d.args()
        a.y, a.h_last = a.x, a.h0
        kb.check(lib, lib.kmb_glr_fwd(byref(a)))
        assert torch.equal(d.x.t, first["y"]) and torch.equal(d.t["h0"], first["h_last"])
        d = mk()
        a = d.args()
        a.dh0 = a.dh_last
        kb.check(lib, lib.kmb_glr_bwd(byref(a)))
        assert torch.equal(d.t["dh_last"], first["dh0"])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [256, 70])
def test_short_sequences_with_states_in_place(lib, cuda, D, dtype):
    """Sequences that begin and end in one tile, in rows of different warps:
    the last state goes where the first one came from."""
    rng = np.random.default_rng(D)
    off = np.concatenate([[0], np.cumsum(rng.integers(0, 40, 300))])
    mk = lambda: Case(300, int(off[-1]), D, dtype, offsets=off, seed=7)  # noqa: E731
    c = mk()
    v, e = c.ref()
    inside = c.inside
    for _ in range(5):
        c = mk()
        c.inside = inside
        a = c.args()
        a.h_last = a.h0
        kb.check(lib, lib.kmb_glr_fwd(byref(a)))
        within("h_last", c.t["h0"].double().cpu().numpy(), v["h_last"], e["h_last"])
        c.check(v, e, ("y",))
        c = mk()
        c.inside = inside
        a = c.args()
        a.dh0 = a.dh_last
        kb.check(lib, lib.kmb_glr_bwd(byref(a)))
        within("dh0", c.t["dh_last"].double().cpu().numpy(), v["dh0"], e["dh0"])
        c.check(v, e, ("dx", "dgate_r", "dgate_i", "ddecay"))


@pytest.mark.parametrize("ckpt,ws", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("offsets", [None, [0, 100, 100, 290]])
def test_without_checkpoints_or_workspace(lib, cuda, ckpt, ws, offsets):
    c = Case(3, 290, 70, offsets=offsets)
    run(lib, c, ckpt, ws)
    c.check(*c.ref(), ALL)


def test_time_major_and_fused_projection(lib, cuda):
    c = Case(4, 150, 68, time_major=True)
    run(lib, c)
    c.check(*c.ref(), ALL)
    # x | gate_r | gate_i as parts of one matrix, and their gradients of another
    c = Case(2, 150, 48, BF16)
    both = []
    for names in (("x", "gate_r", "gate_i"), ("dx", "dgate_r", "dgate_i")):
        p = torch.full((2, 150, 3 * 48), SENTINEL, dtype=BF16, device="cuda")
        both.append(p)
        for k, n in enumerate(names):
            part = p[..., k * 48:(k + 1) * 48]
            if n in c.v:
                part.copy_(torch.from_numpy(c.v[n]).to(BF16))
            getattr(c, n).t = part
    run(lib, c)
    v, e = c.ref()
    c.check(v, e, ("y", "h_last", "dh0", "ddecay"))
    for k in ("dx", "dgate_r", "dgate_i"):
        within(k, getattr(c, k).np().reshape(-1, 48), v[k], e[k], BF16)


def test_optional_tensors(lib, cuda):
    c = Case(2, 140, 40, h0=False)
    for k in ("h_last", "dh0", "ddecay"):
        c.t.pop(k)
    run(lib, c)
    v, e = c.ref()
    c.check(v, e, OUT)
    c = Case(2, 140, 40, h0=False)
    run(lib, c)
    c.check(*c.ref(), ALL)
    # accumulate adds to ddecay alone
    before = c.t["ddecay"].clone()
    a = c.args()
    a.accumulate = 1
    kb.check(lib, lib.kmb_glr_bwd(byref(a)))
    v, e = c.ref()
    within("ddecay", c.t["ddecay"].double().cpu().numpy() - before.double().cpu().numpy(), v["ddecay"],
           e["ddecay"] * 2 + 4 * ref.U * np.abs(v["ddecay"]))
    c.check(v, e, OUT)


PACKED = [
    [0, 300], [0, 0, 300, 300], [0, 1, 2, 3, 67], [0, 64, 128, 192], [0, 63, 64, 65, 129, 129, 129, 200],
    [0, 0, 0, 0], [5, 9, 9, 70], [0, 10, 140, 141, 260], [0, 7, 300, 301, 302, 400, 640, 641],
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tail", [0, 1, 63, 130])
@pytest.mark.parametrize("off", PACKED)
def test_packed(lib, cuda, off, tail, dtype):
    L = off[-1] + tail
    c = Case(len(off) - 1, L, 70, dtype, offsets=off, seed=len(off) + tail)
    run(lib, c)
    c.check(*c.ref(), ALL)


def test_packed_many_sequences(lib, cuda):
    rng = np.random.default_rng(5)
    n = np.minimum(rng.geometric(0.08, 900) - 1, 200)
    off = np.concatenate([[0], np.cumsum(n)])
    for dtype, h0 in ((F32, True), (BF16, False)):
        c = Case(900, int(off[-1]) + 17, 66, dtype, offsets=off, h0=h0)
        run(lib, c)
        c.check(*c.ref(), ALL)


@pytest.mark.parametrize("batch,L", [(0, 5), (3, 0), (0, 0)])
@pytest.mark.parametrize("packed", [False, True])
def test_nothing_to_do(lib, cuda, batch, L, packed):
    c = Case(batch, L, 33, offsets=[0] * (batch + 1) if packed else None)
    run(lib, c)
    assert torch.equal(c.t["h_last"], c.t["h0"]) and torch.equal(c.t["dh0"], c.t["dh_last"])
    assert bool((c.t["ddecay"] == 0).all())


def test_extreme_gates_and_decays(lib, cuda):
    """Gates far out on both sides and decays that forget nothing or all."""
    def far(v):
        v = v.copy()
        v[:, ::7] = 60.0
        v[:, 1::7] = -60.0
        v[:, 2::7] = 15.0
        v[:, 3::7] = -15.0
        return v
    for dtype in (F32, BF16):
        c = Case(2, 200, 64, dtype, values={"gate_r": far, "gate_i": lambda v: far(v[:, ::-1])})
        c.decay[:8] = [-40.0, -25.0, -12.0, 10.0, 40.0, 0.0, -3.0, -80.0]
        c.t["decay"] = f32(c.decay)
        run(lib, c)
        c.check(*c.ref(), ALL)


def test_infinite_gates(lib, cuda):
    """sigmoid(+-inf) is 1 / 0: a closed recurrence gate keeps the state, a
    closed input gate lets nothing in, and no gradient is NaN."""
    def far(v):
        v = v.copy()
        v[:, ::3] = np.inf
        v[:, 1::3] = -np.inf
        return v
    c = Case(1, 100, 64, values={"gate_r": far, "gate_i": lambda v: np.where(np.arange(64) % 2, np.inf, -np.inf) + 0 * v})
    run(lib, c)
    for k in OUT:
        assert np.isfinite(getattr(c, k).np()).all(), k
    with np.errstate(all="ignore"):
        big = {k: np.clip(c.v[k], -200, 200) for k in ("gate_r", "gate_i")}
    c.v.update(big)
    c.check(*c.ref(), ALL)


def test_nan_stays_in_its_sequence(lib, cuda):
    """Rows outside the sequences hold NaN (never read), and a NaN inside one
    sequence reaches neither another sequence nor another channel."""
    off = [3, 80, 80, 200, 330]
    c = Case(4, 350, 70, offsets=off, values={k: (lambda v: np.where(((np.arange(350) < 3) | (np.arange(350) >= 330))[:, None], np.nan, v))
                                              for k in IN})
    run(lib, c)
    c.check(*c.ref(), ALL)
    clean = {k: getattr(c, k).np() for k in OUT}
    c.x.t[100, 11] = float("nan")
    run(lib, c)
    y = c.y.np()
    assert np.isnan(y[100:200, 11]).all()
    y[100:200, 11] = clean["y"][100:200, 11]
    assert np.array_equal(y, clean["y"])
    for k in ("dx", "dgate_r", "dgate_i"):
        g = getattr(c, k).np()
        g[80:200, 11] = clean[k][80:200, 11]
        assert np.array_equal(g, clean[k]), k
    c.x.set(c.v["x"])
    c.dy.t[150, 11] = float("nan")
    run(lib, c)
    assert np.isnan(c.dx.np()[80:151, 11]).all()
    for k in ("dx", "dgate_r", "dgate_i"):
        g = getattr(c, k).np()
        g[80:200, 11] = clean[k][80:200, 11]
        assert np.array_equal(g, clean[k]), k


def test_in_place(lib, cuda):
    """y over x; the gradients over x and the gates; h_last over h0 and dh0 over dh_last."""
    for off in (None, [0, 150, 150, 420], [0, 3, 17, 40, 41, 41, 120, 420]):
        c = Case(len(off) - 1 if off else 3, 420, 66, BF16, offsets=off)
        v, e = c.ref()
        a = c.args()
        a.h_last, a.y = a.h0, a.x
        kb.check(lib, lib.kmb_glr_fwd(byref(a)))
        c.t["h_last"], c.y = c.t["h0"], c.x
        c.check(v, e, ("h_last",))
        within("y", c.y.np().reshape(-1, 66), v["y"], e["y"], BF16)
        c = Case(len(off) - 1 if off else 3, 420, 66, BF16, offsets=off)
        a = c.args()
        a.dx, a.dgate_r, a.dgate_i, a.dh0 = a.x, a.gate_r, a.gate_i, a.dh_last
        kb.check(lib, lib.kmb_glr_bwd(byref(a)))
        c.t["dh0"] = c.t["dh_last"]
        c.check(v, e, ("dh0", "ddecay"))
        for k, o in (("dx", c.x), ("dgate_r", c.gate_r), ("dgate_i", c.gate_i)):
            within(k, o.np().reshape(-1, 66), v[k], e[k], BF16)


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("D,L", [(66, 420), (256, 6000)])
@pytest.mark.parametrize("packed", [False, True])
def test_outputs_over_other_inputs(lib, cuda, packed, D, L, ckpt):
    """y over a gate; each gradient over another's input, dh0 over h0."""
    off = [0, 3, 17, 40, 41, 41, 120, L] if packed else None
    batch = 7 if packed else 3
    for dx, dr, di in (("dy", "x", "gate_r"), ("gate_r", "gate_i", "dy"), ("gate_i", "dy", "x")):
        c = Case(batch, L, D, BF16, offsets=off)
        v, e = c.ref()
        a = c.args()
        if ckpt:
            states = torch.full((max(1, lib.kmb_glr_ckpt_elems(byref(a))),), SENTINEL, device="cuda")
            a.ckpt = states.data_ptr()
            kb.check(lib, lib.kmb_glr_fwd(byref(a)))
        a.dx, a.dgate_r, a.dgate_i, a.dh0 = getattr(a, dx), getattr(a, dr), getattr(a, di), a.h0
        kb.check(lib, lib.kmb_glr_bwd(byref(a)))
        within("dh0", c.t["h0"].double().cpu().numpy(), v["dh0"], e["dh0"])
        c.check(v, e, ("ddecay",))
        for k, o in (("dx", dx), ("dgate_r", dr), ("dgate_i", di)):
            within(k, getattr(c, o).np().reshape(-1, D), v[k], e[k], BF16)
    for over in ("gate_r", "gate_i"):
        c = Case(batch, L, D, BF16, offsets=off)
        a = c.args()
        a.y = getattr(a, over)
        kb.check(lib, lib.kmb_glr_fwd(byref(a)))
        within("y", getattr(c, over).np().reshape(-1, D), v["y"], e["y"], BF16)


def test_same_bits_every_run(lib, cuda):
    for off in (None, [0, 1000, 1003, 3000]):
        c = Case(3, 3000, 100, offsets=off)
        run(lib, c)
        first = {k: getattr(c, k).t.clone() for k in OUT} | {k: c.t[k].clone() for k in ("h_last", "dh0", "ddecay")}
        for _ in range(3):
            run(lib, c)
            for k, t in first.items():
                assert torch.equal(t, getattr(c, k).t if k in OUT else c.t[k]), k


def test_gradient_against_differences(lib, cuda):
    """Along one direction of all inputs: central differences of the forward,
    the loss summed in float64; t = 2^-7: truncation ~ t^2 of the third
    derivative, rounding ~ 2^-24 / t."""
    c = Case(2, 90, 24, kind="slow")
    run(lib, c)
    rng = np.random.default_rng(1)
    names = {"x": "dx", "gate_r": "dgate_r", "gate_i": "dgate_i"}
    dirs = {k: rng.standard_normal(c.v[k].shape) * 0.1 for k in names}
    dot = sum(float((getattr(c, g).np() * dirs[k]).sum()) for k, g in names.items())
    scale = sum(float(np.abs(getattr(c, g).np() * dirs[k]).sum()) for k, g in names.items())
    t, f = 2.0 ** -7, []
    for sgn in (1, -1):
        for k in names:
            getattr(c, k).set(c.v[k] + sgn * t * dirs[k])
        run(lib, c, bwd=False)
        f.append(float((c.y.np() * c.v["dy"]).sum() + (c.t["h_last"].double().cpu().numpy() * c.dlv).sum()))
    want = (f[0] - f[1]) / (2 * t)
    assert abs(dot - want) <= (t * t + 8 * 2.0 ** -24 / t) * scale, (dot, want, scale)


def test_prefill_then_steps(lib, cuda):
    """A prefill of 77 rows from h0, then one step a row, against one forward."""
    n, L, D = 5, 90, 68
    for dtype in (F32, BF16):
        c = Case(n, L, D, dtype)
        v, e = c.ref(grads=False)
        a = c.args()
        a.L = 77
        kb.check(lib, lib.kmb_glr_fwd(byref(a)))
        # states in slots of a larger table
        table = torch.full((11, D + 4), SENTINEL, device="cuda")
        slots = torch.tensor([7, 0, 10, 3, 4], device="cuda")
        table[slots, :D] = c.t["h_last"]
        for t in range(77, L):
            s = kb.KmbGLRStep()
            for k in ("x", "gate_r", "gate_i", "y"):
                b = getattr(c, k).t[:, t]
                setattr(s, k, kb.KmbRows(b.data_ptr(), b.stride(0), 0))
            s.decay, s.state, s.slots = c.t["decay"].data_ptr(), table.data_ptr(), slots.data_ptr()
            s.rows, s.n_states, s.D, s.ld_state, s.scale, s.type = n, 11, D, D + 4, 8.0, TYPE[dtype]
            kb.check(lib, lib.kmb_glr_step(byref(s)))
        within("y", c.y.np().reshape(-1, D), v["y"], e["y"], dtype)
        within("state", table[slots, :D].double().cpu().numpy(), v["h_last"], e["h_last"])
        rest = torch.ones(11, dtype=torch.bool, device="cuda")
        rest[slots] = False
        assert bool((table[rest] == SENTINEL).all()) and bool((table[:, D:] == SENTINEL).all())
        assert c.y.untouched_outside()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,D,gap,shift", [(0, 8, 0, 0), (1, 1, 0, 0), (1, 1024, 0, 0), (3, 130, 2, 1), (64, 300, 0, 0),
                                              (301, 64, 1, 0), (700, 96, 0, 0), (64, 1284, 0, 0),
                                              (64, 1284, 4, 0), (64, 1284, 1, 0)])
def test_step_slots(lib, cuda, rows, D, gap, shift, dtype):
    """Padded rows (negative, beyond the table) are left out, and of the rows
    that name one slot only the first is taken."""
    rng = np.random.default_rng(rows)
    n = rows + 3
    c = Case(rows, 1, D, dtype, gap=gap, shift=shift)
    slots = rng.permutation(n)[:rows].astype(np.int64)
    live = np.ones(rows, bool)
    for k, s in ((1, -1), (2, n), (5, -(1 << 40)), (7, 1 << 40)):
        if k < rows:
            slots[k], live[k] = s, False
    for k, j in ((40, 9), (41, 9), (63, 0), (300, 299), (690, 10)):
        if k < rows and live[j]:
            slots[k], live[k] = slots[j], False
    tab = typed(rng.standard_normal((n, D)), F32)
    state = f32(tab)
    ts = torch.from_numpy(slots).cuda()
    s = kb.KmbGLRStep()
    for k in ("x", "gate_r", "gate_i", "y"):
        b = getattr(c, k).t[:, 0] if rows else getattr(c, k).t.view(0, D)
        setattr(s, k, kb.KmbRows(b.data_ptr(), getattr(c, k).ld, 0))
    s.decay, s.state, s.slots = c.t["decay"].data_ptr(), state.data_ptr(), ts.data_ptr()
    s.rows, s.n_states, s.D, s.ld_state, s.scale, s.type = rows, n, D, D, 8.0, TYPE[dtype]
    kb.check(lib, lib.kmb_glr_step(byref(s)))
    want, bound = tab.copy(), np.zeros_like(tab)
    y = c.y.np().reshape(rows, D)
    for k in range(rows):
        if not live[k]:
            assert np.all(y[k] == SENTINEL)
            continue
        h, e = ref.glr_fwd(c.v["x"][k], c.v["gate_r"][k], c.v["gate_i"][k], c.decay, 8.0, tab[slots[k]])
        within("y", y[k], h[0], e[0], dtype)
        want[slots[k]], bound[slots[k]] = h[0], e[0]
    within("state", state.double().cpu().numpy(), want, bound)
    assert c.y.untouched_outside()


def test_step_without_slots(lib, cuda):
    c = Case(6, 1, 40)
    state = c.t["h0"].clone()
    s = kb.KmbGLRStep()
    for k in ("x", "gate_r", "gate_i", "y"):
        setattr(s, k, kb.KmbRows(getattr(c, k).t.data_ptr(), 40, 0))
    s.decay, s.state = c.t["decay"].data_ptr(), state.data_ptr()
    s.rows, s.n_states, s.D, s.ld_state, s.scale = 6, 6, 40, 40, 8.0
    kb.check(lib, lib.kmb_glr_step(byref(s)))
    v, e = c.ref(grads=False)
    within("state", state.double().cpu().numpy(), v["h_last"], e["h_last"])
    c.check(v, e, ("y",))


def test_graphs_share_a_workspace(lib, cuda):
    """Two captured forward + backward passes with one workspace, replayed one
    after the other on new inputs; refusals during capture."""
    cases = [Case(2, 700, 96, seed=1), Case(3, 700, 96, offsets=[0, 20, 650, 700], seed=2)]
    calls = []
    for c in cases:
        a = c.args()
        c.ckpt = torch.empty(lib.kmb_glr_ckpt_elems(byref(a)), device="cuda")
        a.ckpt = c.ckpt.data_ptr()
        calls.append(a)
    size = max(lib.kmb_glr_workspace_bytes(byref(a), 1) for a in calls)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    for a in calls:
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
    stream = torch.cuda.Stream()
    graphs = []
    try:
        lib.kmb_set_sync(0)
        lib.kmb_set_stream(stream.cuda_stream)
        for a in calls:
            kb.check(lib, lib.kmb_glr_fwd(byref(a)))
            kb.check(lib, lib.kmb_glr_bwd(byref(a)))
        stream.synchronize()
        for a in calls:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                kb.check(lib, lib.kmb_glr_fwd(byref(a)))
                kb.check(lib, lib.kmb_glr_bwd(byref(a)))
                b = kb.KmbGLR.from_buffer_copy(a)
                b.workspace, b.workspace_bytes = None, 0
                assert lib.kmb_glr_bwd(byref(b)) == kb.KMB_EINVAL
                assert b"capture" in lib.kmb_last_error()
                lib.kmb_set_sync(1)
                assert lib.kmb_glr_fwd(byref(a)) == kb.KMB_EINVAL
                lib.kmb_set_sync(0)
            graphs.append(g)
        for c in cases:
            for k in IN:
                c.v[k] = typed(c.v[k][::-1] * 0.5, F32)
                getattr(c, k).set(c.v[k])
        # a replay reads the offsets that are there then
        cases[1].off = np.array([0, 333, 333, 690])
        cases[1].t["offsets"].copy_(torch.from_numpy(cases[1].off))
        for k in OUT:
            getattr(cases[1], k).t.fill_(SENTINEL)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for g in graphs + graphs:
                g.replay()
        torch.cuda.synchronize()
    finally:
        lib.kmb_set_stream(None)
        lib.kmb_set_sync(1)
    for c in cases:
        c.check(*c.ref(), ALL)


def test_two_streams_at_once(lib, cuda):
    """Calls in flight on two streams, each with its own workspace."""
    cases = [Case(1, 6000, 128, seed=s) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    keep = []
    calls = []
    for c in cases:
        a = c.args()
        keep.append(workspace(lib, a, 1))
        calls.append(a)
    torch.cuda.synchronize()
    try:
        lib.kmb_set_sync(0)
        for _ in range(5):
            for s, a in zip(streams, calls):
                lib.kmb_set_stream(s.cuda_stream)
                kb.check(lib, lib.kmb_glr_fwd(byref(a)))
                kb.check(lib, lib.kmb_glr_bwd(byref(a)))
        torch.cuda.synchronize()
    finally:
        lib.kmb_set_stream(None)
        lib.kmb_set_sync(1)
    for c in cases:
        c.check(*c.ref(), ALL)


def test_rows_past_32_bits(lib, cuda):
    """Rows whose offsets pass 2^32 elements."""
    D, L = 64, 5
    ld = (1 << 30) + 4
    buf = torch.empty((L - 1) * ld + D, dtype=BF16, device="cuda")
    c = Case(1, L, D, BF16)
    c.x.t = buf.as_strided((1, L, D), (D, ld, 1))
    c.x.t.copy_(torch.from_numpy(c.v["x"]).to(BF16))
    run(lib, c)
    c.check(*c.ref(), ALL)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("batch,L,D,spare", [(3, 1200, 520, 0), (3, 1121, 520, 40), (1, 5600, 264, 8), (2, 1300, 1032, 3)])
def test_resident_kernels_on_slices(lib, cuda, batch, L, D, spare, packed, dtype):
    """More tiles than SMs on the three parts of one projection, whose width is
    no multiple of a tile's 64 channels: a tile's last columns reach into the
    part beside it, which it neither takes nor writes.  `spare` rows of another
    kind lie behind every sequence (batch strides above L rows)."""
    total = batch * L
    off = [0, 0, 300, 301, total - 7, total] if packed else None
    c = Case(5 if packed else batch, total if packed else L, D, dtype, offsets=off, seed=D + L)
    lead = (1, total) if packed else (batch, L)
    parts = {}
    for names in (("x", "gate_r", "gate_i"), ("dx", "dgate_r", "dgate_i"), ("y", "dy")):
        p = torch.full((lead[0], lead[1] + spare, len(names) * D + 16), SENTINEL, dtype=dtype, device="cuda")
        for k, n in enumerate(names):
            part = p[:, :lead[1], 8 + k * D:8 + (k + 1) * D]
            if n in c.v:
                part.copy_(torch.from_numpy(c.v[n]).to(dtype).view(part.shape))
            getattr(c, n).t = part[0] if packed else part
        parts[names] = p
    before = {k: p.clone() for k, p in parts.items()}
    for ckpt in (True, False):
        for k, p in parts.items():
            p.copy_(before[k])
        run(lib, c, ckpt=ckpt)
        v, e = c.ref()
        c.check(v, e, ("h_last", "dh0", "ddecay"))
        for k in OUT:
            within(k, getattr(c, k).np().reshape(-1, D), v[k], e[k], dtype)
        for names, p in parts.items():
            after, was = p.clone(), before[names]
            for n in names:
                if n in OUT:
                    k = names.index(n)
                    after[:, :lead[1], 8 + k * D:8 + (k + 1) * D] = SENTINEL
            assert torch.equal(after, was), names
