"""GPU parity of the layer norm (kmb_layernorm_fwd / _bwd) with its float64
definition.  Tolerances: the first-order bounds of oracle/recurrent_ref.py,
entry by entry, plus half a step of bf16 outputs."""
import numpy as np
import pytest
import torch

import kmamba_b200 as kb
import recurrent_ref as ref
from recurrent_util import SENTINEL, Banded, byref, typed, within

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
TYPE = {F32: kb.KMB_F32, BF16: kb.KMB_BF16}
EPS = 1e-5


def f32(a):
    return None if a is None else torch.from_numpy(np.asarray(a, np.float32)).cuda()


class Case:
    def __init__(self, rows, D, xt=F32, yt=F32, gap=0, shift=0, seed=0, affine=True, offset=0.3, x=None):
        rng = np.random.default_rng(seed)
        self.rows, self.D, self.xt, self.yt = rows, D, xt, yt
        self.xv = typed(rng.standard_normal((rows, D)) * rng.uniform(0.5, 3, (rows, 1)) + offset if x is None else x, xt)
        self.w = typed(1 + 0.1 * rng.standard_normal(D), F32) if affine else None
        self.b = typed(0.1 * rng.standard_normal(D), F32) if affine else None
        self.dyv = typed(rng.standard_normal((rows, D)), yt)
        self.resv = typed(rng.standard_normal((rows, D)), xt)
        mk = lambda t, fill: Banded((rows, D), t, fill, gap, shift)  # noqa: E731
        self.x = mk(xt, float("nan")).set(self.xv)
        self.dy = mk(yt, float("nan")).set(self.dyv)
        self.res = mk(xt, float("nan")).set(self.resv)
        self.y, self.dx = mk(yt, SENTINEL), mk(xt, SENTINEL)
        self.tw, self.tb = f32(self.w), f32(self.b)
        self.mean = torch.full((rows,), SENTINEL, device="cuda")
        self.rstd = torch.full((rows,), SENTINEL, device="cuda")
        self.dw = torch.full((D,), SENTINEL, device="cuda")
        self.db = torch.full((D,), SENTINEL, device="cuda")

    def args(self):
        a = kb.KmbLayerNorm()
        for n in ("x", "y", "dy", "dx"):
            setattr(a, n, getattr(self, n).t.data_ptr())
            setattr(a, "ld_" + n, getattr(self, n).ld)
        a.weight = self.tw.data_ptr() if self.tw is not None else None
        a.bias = self.tb.data_ptr() if self.tb is not None else None
        a.rows, a.D, a.eps, a.x_type, a.y_type = self.rows, self.D, EPS, TYPE[self.xt], TYPE[self.yt]
        return a


def fwd(lib, c, stats=True):
    a = c.args()
    if stats:
        a.mean, a.rstd = c.mean.data_ptr(), c.rstd.data_ptr()
    kb.check(lib, lib.kmb_layernorm_fwd(byref(a)))
    torch.cuda.synchronize()


def check_fwd(c):
    (y, m, r), (ey, em, er) = ref.ln_fwd(c.xv, c.w, c.b, EPS)
    within("y", c.y.np(), y, ey, c.yt)
    within("mean", c.mean.double().cpu().numpy(), m, em)
    within("rstd", c.rstd.double().cpu().numpy(), r, er)
    assert c.y.untouched_outside()


def bwd(lib, c, res=False, stats=True, sums=True, acc=0, ws=True):
    a = c.args()
    if res:
        a.dres, a.ld_dres = c.res.t.data_ptr(), c.res.ld
    if stats:
        (_, m, r), _ = ref.ln_fwd(c.xv, None, None, EPS)
        c.mean, c.rstd = f32(m), f32(r)
        a.mean, a.rstd = c.mean.data_ptr(), c.rstd.data_ptr()
    if sums:
        a.dweight, a.dbias, a.accumulate = c.dw.data_ptr(), c.db.data_ptr(), acc
    if ws:
        c.ws = torch.full((lib.kmb_layernorm_workspace_bytes(byref(a)),), 255, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = c.ws.data_ptr(), c.ws.numel()
    kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
    torch.cuda.synchronize()


def check_bwd(c, res=False, stats=True, sums=True, base=0.0):
    m, r = (c.mean.double().cpu().numpy(), c.rstd.double().cpu().numpy()) if stats else (None, None)
    (dx, dw, db), (ex, ew, eb) = ref.ln_bwd(c.xv, c.w, c.dyv, EPS, c.resv if res else None, m, r)
    within("dx", c.dx.np(), dx, ex, c.xt)
    assert c.dx.untouched_outside()
    if sums:
        within("dweight", c.dw.double().cpu().numpy() - base, dw, ew + 2 * ref.U * abs(base))
        within("dbias", c.db.double().cpu().numpy() - base, db, eb + 2 * ref.U * abs(base))
    else:
        assert bool((c.dw == SENTINEL).all())


# widths around every vector and warp size, and above what a CTA's registers hold
WIDTHS = [1, 2, 3, 7, 8, 31, 32, 33, 64, 96, 127, 128, 255, 256, 257, 384, 512, 513, 768, 1000, 1024, 1025, 1537,
          2048, 2050, 4096, 4097, 5000, 8192, 8200, 12288, 16384, 16400, 20000, 33000, 70001]


@pytest.mark.parametrize("xt,yt", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(lib, cuda, D, xt, yt):
    rows = 5 if D < 8000 else 2
    for gap, shift in ((0, 0), (3, 1)):
        c = Case(rows, D, xt, yt, gap, shift, seed=D)
        fwd(lib, c)
        check_fwd(c)
        bwd(lib, c, res=bool(gap))
        check_bwd(c, res=bool(gap))


@pytest.mark.parametrize("rows", [0, 1, 2, 3, 4, 5, 8, 9, 147, 149, 1000, 4097])
@pytest.mark.parametrize("D", [24, 96, 300, 1024])
def test_rows(lib, cuda, rows, D):
    c = Case(rows, D, F32, BF16, seed=rows)
    fwd(lib, c)
    check_fwd(c)
    bwd(lib, c, res=True, stats=False)
    check_bwd(c, res=True, stats=False)


@pytest.mark.parametrize("D", [40, 512, 1030, 9000, 40000])
def test_optional_arguments(lib, cuda, D):
    c = Case(37, D, affine=False)
    fwd(lib, c, stats=False)
    assert bool((c.mean == SENTINEL).all())
    (y, _, _), (ey, _, _) = ref.ln_fwd(c.xv, None, None, EPS)
    within("y", c.y.np(), y, ey)
    bwd(lib, c, sums=False, stats=False)
    check_bwd(c, sums=False, stats=False)
    # one of the two sums alone, added to what is there, through pooled scratch
    c = Case(37, D, BF16, BF16)
    c.db.fill_(3.0)
    c.dw.fill_(3.0)
    bwd(lib, c, acc=1, ws=False)
    check_bwd(c, base=3.0)
    a = c.args()
    c.dw.fill_(SENTINEL)
    a.dbias, a.workspace, a.workspace_bytes = c.db.data_ptr(), None, 0
    kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
    (_, _, db), (_, _, eb) = ref.ln_bwd(c.xv, c.w, c.dyv, EPS)
    within("dbias", c.db.double().cpu().numpy(), db, eb)
    assert bool((c.dw == SENTINEL).all())


def test_large_mean_and_constant_rows(lib, cuda):
    """A mean far above the spread (the squares are of centred values), rows
    of one value (variance 0: y = bias), and huge and tiny scales."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 1000))
    x[0] += 1000.0
    x[1] = 5.0
    x[2] *= 1e18
    x[3] *= 1e-18
    x[4] = 0.0
    c = Case(6, 1000, x=x)
    fwd(lib, c)
    check_fwd(c)
    bwd(lib, c, stats=False)
    check_bwd(c, stats=False)


@pytest.mark.parametrize("D", [96, 1024, 9000, 70001])
def test_non_finite_rows_stay_alone(lib, cuda, D):
    c = Case(9, D)
    c.x.t[3, D // 2] = float("nan")
    c.x.t[6, 0] = float("inf")
    fwd(lib, c)
    y = c.y.np()
    assert np.isnan(y[3]).all() and np.isnan(y[6]).all()
    keep = [0, 1, 2, 4, 5, 7, 8]
    (want, _, _), (ey, _, _) = ref.ln_fwd(c.xv[keep], c.w, c.b, EPS)
    within("y", y[keep], want, ey)
    bwd(lib, c, stats=False)
    (dx, _, _), (ex, _, _) = ref.ln_bwd(c.xv[keep], c.w, c.dyv[keep], EPS)
    within("dx", c.dx.np()[keep], dx, ex)


@pytest.mark.parametrize("D", [100, 1024, 5000, 40000])
def test_in_place(lib, cuda, D):
    c = Case(7, D)
    a = c.args()
    a.y = a.x
    kb.check(lib, lib.kmb_layernorm_fwd(byref(a)))
    (y, _, _), (ey, _, _) = ref.ln_fwd(c.xv, c.w, c.b, EPS)
    within("y", c.x.np(), y, ey)
    for target in ("x", "dy", "res"):
        c = Case(7, D)
        a = c.args()
        a.dres, a.ld_dres = c.res.t.data_ptr(), c.res.ld
        a.dweight, a.dbias = c.dw.data_ptr(), c.db.data_ptr()
        t = getattr(c, target)
        a.dx, a.ld_dx = t.t.data_ptr(), t.ld
        kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
        (dx, dw, db), (ex, ew, eb) = ref.ln_bwd(c.xv, c.w, c.dyv, EPS, c.resv)
        within("dx", t.np(), dx, ex)
        within("dweight", c.dw.double().cpu().numpy(), dw, ew)


@pytest.mark.parametrize("rows,D", [(5000, 64), (3000, 1024), (700, 9000)])
def test_same_bits_every_run(lib, cuda, rows, D):
    c = Case(rows, D, BF16, BF16)
    bwd(lib, c)
    first = (c.dx.t.clone(), c.dw.clone(), c.db.clone())
    for _ in range(3):
        bwd(lib, c)
        assert all(torch.equal(p, q) for p, q in zip(first, (c.dx.t, c.dw, c.db)))


@pytest.mark.parametrize("rows,D", [(1, 1), (33, 1), (3, 1000), (255, 128), (1024, 128), (1025, 128), (256, 129), (257, 129),
                                    (256, 511), (32, 513), (33, 513), (31, 2047), (32, 2048), (32, 2049)])
@pytest.mark.parametrize("xt,yt", [(F32, F32), (BF16, F32), (BF16, BF16)])
def test_few_rows(lib, cuda, rows, D, xt, yt):
    """Fewer rows than CTAs, the rows' kernel and the sums' close together;
    three calls that add up give three times the sums."""
    c = Case(rows, D, xt, yt, seed=rows + D)
    bwd(lib, c, res=True, stats=False)
    check_bwd(c, res=True, stats=False)
    dw, db, dx = c.dw.clone(), c.db.clone(), c.dx.t.clone()
    for _ in range(2):
        bwd(lib, c, res=True, stats=False, acc=1)
        assert torch.equal(c.dx.t, dx)
    assert torch.equal(c.dw, (dw + dw) + dw) and torch.equal(c.db, (db + db) + db)


def test_gradient_against_differences(lib, cuda):
    """Along one direction: (f(x + t v) - f(x - t v)) / 2t of the forward, the
    sum taken in float64.  t = 2^-6: truncation ~ t^2, rounding ~ 2^-24 / t."""
    c = Case(4, 200)
    bwd(lib, c, stats=False)
    dx = c.dx.np()
    rng = np.random.default_rng(9)
    v = typed(rng.standard_normal((4, 200)) * 0.1, F32)
    t, f = 2.0 ** -6, []
    for sgn in (1, -1):
        c.x.set(c.xv + sgn * t * v)
        fwd(lib, c)
        f.append(float((c.y.np() * c.dyv).sum()))
    want = (f[0] - f[1]) / (2 * t)
    scale = np.abs(dx * v).sum()
    assert abs(float((dx * v).sum()) - want) <= (t * t + 2 ** -24 / t * 4) * scale, (want, (dx * v).sum())


def test_graph_capture_and_shared_workspace(lib, cuda):
    """Two graphs with one workspace, replayed one after the other with new
    inputs; capture without a workspace or in synchronous mode is refused."""
    cases = [Case(300, 513, seed=s) for s in (1, 2)]
    ws = torch.empty(lib.kmb_layernorm_workspace_bytes(byref(cases[0].args())), dtype=torch.uint8, device="cuda")
    calls = []
    for c in cases:
        a = c.args()
        a.dweight, a.dbias = c.dw.data_ptr(), c.db.data_ptr()
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        calls.append(a)
    stream = torch.cuda.Stream()
    graphs = []
    try:
        lib.kmb_set_sync(0)
        lib.kmb_set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            for a in calls:
                kb.check(lib, lib.kmb_layernorm_fwd(byref(a)))
                kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
        stream.synchronize()
        for a in calls:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                kb.check(lib, lib.kmb_layernorm_fwd(byref(a)))
                kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
                lib.kmb_set_sync(1)
                assert lib.kmb_layernorm_fwd(byref(a)) == kb.KMB_EINVAL
                assert b"capture" in lib.kmb_last_error()
                lib.kmb_set_sync(0)
                b = kb.KmbLayerNorm.from_buffer_copy(a)
                b.workspace, b.workspace_bytes = None, 0
                assert lib.kmb_layernorm_bwd(byref(b)) == kb.KMB_EINVAL
                assert b"capture" in lib.kmb_last_error()
            graphs.append(g)
        for c in cases:
            c.xv = typed(c.xv[::-1] * 1.5 + 0.25, F32)
            c.x.set(c.xv)
            c.dw.fill_(SENTINEL)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for g in graphs + graphs:
                g.replay()
        torch.cuda.synchronize()
    finally:
        lib.kmb_set_stream(None)
        lib.kmb_set_sync(1)
    for c in cases:
        (y, _, _), (ey, _, _) = ref.ln_fwd(c.xv, c.w, c.b, EPS)
        within("y", c.y.np(), y, ey)
        check_bwd(c, stats=False)


def test_few_rows_captured(lib, cuda):
    """A short backward, captured and replayed on new inputs."""
    c = Case(100, 384)
    a = c.args()
    a.dweight, a.dbias = c.dw.data_ptr(), c.db.data_ptr()
    ws = torch.empty(lib.kmb_layernorm_workspace_bytes(byref(a)), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    stream = torch.cuda.Stream()
    try:
        lib.kmb_set_sync(0)
        lib.kmb_set_stream(stream.cuda_stream)
        kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
        c.xv = typed(c.xv[::-1] * 1.5 + 0.25, F32)
        c.x.set(c.xv)
        c.dw.fill_(SENTINEL)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
            g.replay()
        torch.cuda.synchronize()
    finally:
        lib.kmb_set_stream(None)
        lib.kmb_set_sync(1)
    check_bwd(c, stats=False)


def test_rows_past_32_bits(lib, cuda):
    """A tensor of more than 2^32 elements between the first and last row."""
    D, rows = 256, 3
    ld = (1 << 31) + 8
    buf = torch.empty((rows - 1) * ld + D, dtype=BF16, device="cuda")
    x = buf.as_strided((rows, D), (ld, 1))
    rng = np.random.default_rng(0)
    xv = typed(rng.standard_normal((rows, D)), BF16)
    x.copy_(torch.from_numpy(xv).to(BF16))
    c = Case(rows, D, BF16, F32)
    c.xv = xv
    a = c.args()
    a.x, a.ld_x = x.data_ptr(), ld
    kb.check(lib, lib.kmb_layernorm_fwd(byref(a)))
    (y, _, _), (ey, _, _) = ref.ln_fwd(xv, c.w, c.b, EPS)
    within("y", c.y.np(), y, ey)


@pytest.mark.parametrize("D", [24, 96, 128])
@pytest.mark.parametrize("rows", [1, 5, 130, 9473])
@pytest.mark.parametrize("stats", [False, True])
def test_eps_zero(lib, cuda, rows, D, stats):
    """eps = 0 divides by the rows' own spread alone.  Lanes that share a warp
    with rows and have none (four rows a warp, up to 128 columns) add nothing
    to the sums, although zeros have no spread."""
    c = Case(rows, D, seed=rows + D)
    a = c.args()
    a.eps = 0.0
    if stats:
        (_, m, r), _ = ref.ln_fwd(c.xv, None, None, 0.0)
        c.mean, c.rstd = f32(m), f32(r)
        a.mean, a.rstd = c.mean.data_ptr(), c.rstd.data_ptr()
    a.dweight, a.dbias = c.dw.data_ptr(), c.db.data_ptr()
    kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
    m, r = (c.mean.double().cpu().numpy(), c.rstd.double().cpu().numpy()) if stats else (None, None)
    (dx, dw, db), (ex, ew, eb) = ref.ln_bwd(c.xv, c.w, c.dyv, 0.0, None, m, r)
    within("dx", c.dx.np(), dx, ex)
    within("dweight", c.dw.double().cpu().numpy(), dw, ew)
    within("dbias", c.db.double().cpu().numpy(), db, eb)
    a = c.args()
    a.eps = 0.0
    kb.check(lib, lib.kmb_layernorm_fwd(byref(a)))
    (y, _, _), (ey, _, _) = ref.ln_fwd(c.xv, c.w, c.b, 0.0)
    within("y", c.y.np(), y, ey)


@pytest.mark.parametrize("rows,D,xt", [(4097, 300, F32), (3001, 1537, BF16), (2500, 2048, F32), (1200, 5000, BF16)])
def test_expired_wait_is_reported(lib, cuda, rows, D, xt):
    """The error word set on the host, as by a wait that expired: the calls
    that find it return KMB_ETIMEOUT once, and end in order (rows through the
    ring: copies under way, no refill); the next ones are whole again."""
    c = Case(rows, D, xt, xt)
    for call, check in ((fwd, check_fwd), (bwd, check_bwd)):
        assert lib.kmb_layernorm_expire() == kb.KMB_OK
        with pytest.raises(RuntimeError, match="a wait for a row expired"):
            call(lib, c)
        torch.cuda.synchronize()
        assert lib.kmb_layernorm_check_error() == kb.KMB_OK
        call(lib, c)
        check(c)


@pytest.mark.parametrize("D", [(1 << 31) - 8, (1 << 31) - 3])
def test_one_row_of_almost_2_31_columns(lib, cuda, D):
    """x = 1, -1, 1, ..  dy has a few entries, at both ends; elsewhere dx is
    what the averages leave.

    Errors.  A thread's sum of x is a whole number of at most 2^22: exact.
    Across 32 lanes and 16 warps it passes 2^24: 5 + 16 additions of values
    whose absolute sum is D, so the mean is off by at most 21 U.  The centred
    squares are then within 42 U of 1.  A thread adds them to a sum below
    2^23, of which 1 is a whole number of steps: an addition is off by no more
    than the square's distance from 1, 42 U, and the sum of all by 42 + 42 +
    21 U; rstd by half of that and its own steps, 57 U; xhat by 21 + 57 + 2 U."""
    x = torch.ones(D, dtype=BF16, device="cuda")
    x[1::2] = -1
    y, mean, rstd = torch.empty_like(x), torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
    a = kb.KmbLayerNorm()
    a.x, a.y, a.mean, a.rstd = x.data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr()
    a.rows, a.D, a.eps, a.x_type, a.y_type = 1, D, EPS, kb.KMB_BF16, kb.KMB_BF16
    a.ld_x = a.ld_y = a.ld_dy = a.ld_dx = D
    kb.check(lib, lib.kmb_layernorm_fwd(byref(a)))
    m = (D % 2) / D
    r = (1 - m * m + EPS) ** -0.5
    assert abs(mean.item() - m) <= 21 * ref.U and abs(rstd.item() - r) <= 57 * ref.U
    assert torch.equal(y, x)  # (1 + 1e-5)^-1/2 rounds to 1
    del y
    at = torch.tensor([0, 3, D - 5000, D - 2, D - 1], device="cuda")
    v = torch.tensor([1.0, -2.0, 0.5, 4.0, -8.0], device="cuda")
    dy = torch.zeros_like(x)
    dy[at] = v.to(BF16)
    rest = 2 * 15.5 / D  # |rstd (avg g + xhat avg(g xhat))| <= 2 sum |g| / D
    for saved in (False, True):
        for sums in (False, True):
            dx = torch.full_like(x, SENTINEL)
            b = kb.KmbLayerNorm.from_buffer_copy(a)
            b.dy, b.dx = dy.data_ptr(), dx.data_ptr()
            if not saved:
                b.mean = b.rstd = None
            if sums:
                dw, db = (torch.full((D,), SENTINEL, device="cuda") for _ in range(2))
                ws = torch.empty(lib.kmb_layernorm_workspace_bytes(byref(b)), dtype=torch.uint8, device="cuda")
                b.dweight, b.dbias, b.workspace, b.workspace_bytes = dw.data_ptr(), db.data_ptr(), ws.data_ptr(), ws.numel()
            kb.check(lib, lib.kmb_layernorm_bwd(byref(b)))
            if sums:
                assert bool(((dw[at] - v * x[at] * r).abs() <= 82 * ref.U * v.abs()).all())
                assert torch.equal(db[at], v)
                dw[at] = db[at] = 0
                assert not bool(dw.any()) and not bool(db.any())
                del dw, db, ws
            assert bool(((dx[at].float() - v * r).abs() <= 2.0 ** -8 * v.abs()).all())
            dx[at] = 0
            assert dx.max().item() <= rest and dx.min().item() >= -rest
            del dx


# Enough rows for the ring of copies in both directions (more than a row for
# each warp, or CTA, of the resident grid).  Up to 1024 columns (backward 512)
# a warp has a row, above that several.  Whole pieces, vectors: rows that
# begin and end on 16 bytes.  Shared pieces, vectors: bf16 rows of a multiple
# of four columns beside fp32 ones.  Shared pieces, single values: the rest.
RING = [(2500, 512, 0, 0), (2500, 1024, 8, 8), (1300, 2048, 0, 0), (500, 8192, 0, 0), (400, 20000, 0, 0),
        (2500, 300, 0, 4), (2500, 388, 0, 0), (1300, 2052, 4, 4), (500, 5004, 0, 4),
        (2500, 257, 0, 0), (2500, 257, 3, 1), (2500, 771, 0, 1), (2500, 771, 5, 0), (2500, 1025, 0, 0),
        (2500, 1537, 5, 0), (2500, 1537, 5, 1), (2500, 1537, 0, 1), (1300, 2049, 0, 3), (1300, 2049, 7, 0),
        (500, 5001, 0, 0), (500, 5001, 3, 1), (500, 8191, 1, 1)]


@pytest.mark.parametrize("xt,yt", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,D,gap,shift", RING)
def test_ring(lib, cuda, rows, D, gap, shift, xt, yt):
    c = Case(rows, D, xt, yt, gap, shift, seed=rows + D)
    fwd(lib, c)
    check_fwd(c)
    for res, stats in ((False, True), (True, False)):
        bwd(lib, c, res=res, stats=stats)
        check_bwd(c, res=res, stats=stats)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("rows,D,gap,shift", [(2500, 512, 0, 0), (2500, 300, 0, 1), (2500, 771, 0, 1), (2500, 1537, 5, 1),
                                              (1300, 2048, 0, 0), (1300, 2049, 0, 3), (500, 5001, 0, 1)])
def test_ring_in_place(lib, cuda, rows, D, gap, shift, t):
    """Outputs over inputs whose later rows, and whose neighbours' bytes, are
    being copied meanwhile."""
    mk = lambda: Case(rows, D, t, t, gap, shift, seed=rows + D)  # noqa: E731
    c = mk()
    a = c.args()
    a.y = a.x
    kb.check(lib, lib.kmb_layernorm_fwd(byref(a)))
    (y, _, _), (ey, _, _) = ref.ln_fwd(c.xv, c.w, c.b, EPS)
    within("y", c.x.np(), y, ey, t)
    (dx, dw, db), (ex, ew, eb) = ref.ln_bwd(c.xv, c.w, c.dyv, EPS, c.resv)
    for target in ("x", "dy", "res"):
        c = mk()
        a = c.args()
        a.dres, a.ld_dres = c.res.t.data_ptr(), c.res.ld
        a.dweight, a.dbias = c.dw.data_ptr(), c.db.data_ptr()
        o = getattr(c, target)
        a.dx, a.ld_dx = o.t.data_ptr(), o.ld
        kb.check(lib, lib.kmb_layernorm_bwd(byref(a)))
        within("dx", o.np(), dx, ex, t)
        within("dweight", c.dw.double().cpu().numpy(), dw, ew)
        within("dbias", c.db.double().cpu().numpy(), db, eb)
        # what lies around the rows is as it was (NaN)
        f = o.flat.clone()
        f.as_strided(o.t.shape, o.t.stride(), o.t.storage_offset()).fill_(float("nan"))
        assert bool(f.isnan().all())
