"""The float64 definitions of the layer norm and the gated linear recurrence
(oracle/recurrent_ref.py) against central differences, and the argument
checks of their entry points (no GPU needed: every refusal comes before the
first CUDA launch)."""
import ctypes as C

import numpy as np
import pytest

import kmamba_b200 as kb
import recurrent_ref as ref


def diff(f, v, step=1e-5):
    """Central differences of the scalar f() over every entry of v."""
    g = np.empty_like(v)
    for k in np.ndindex(*v.shape):
        old = v[k]
        v[k] = old + step
        hi = f()
        v[k] = old - step
        lo = f()
        v[k] = old
        g[k] = (hi - lo) / (2 * step)
    return g


# central differences of step 1e-5 on values of order one: truncation step^2 ~
# 1e-10, rounding 1e-16 * |loss| / 1e-5 ~ 1e-10
TOL = 1e-7


def test_ln_gradients_match_differences():
    rng = np.random.default_rng(0)
    x, w, b, c = (rng.standard_normal(s) for s in ((3, 7), 7, 7, (3, 7)))
    (dx, dw, db), _ = ref.ln_bwd(x, w, c, 1e-5)
    f = lambda: float((ref.ln_fwd(x, w, b, 1e-5)[0][0] * c).sum())  # noqa: E731
    for name, v, g in (("x", x, dx), ("w", w, dw), ("b", b, db)):
        assert np.max(np.abs(diff(f, v) - g)) <= TOL, name


def test_glr_gradients_match_differences():
    rng = np.random.default_rng(1)
    D, seqs = 3, [(0, 4), (4, 4), (4, 9), (10, 11)]
    rows = 11
    x, gr, gi, cy = (rng.standard_normal((rows, D)) for _ in range(4))
    # a decaying channel, one near 1, and one that forgets within a step
    decay = np.array([-4.0, -9.0, 1.5])
    h0, cl = rng.standard_normal((4, D)), rng.standard_normal((4, D))

    def f():
        v, _ = ref.glr(x, gr, gi, decay, 8.0, seqs, h0)
        return float(np.nansum(v["y"] * cy) + (v["h_last"] * cl).sum())
    v, _ = ref.glr(x, gr, gi, decay, 8.0, seqs, h0, cy, cl)
    for name, t, g in (("x", x, v["dx"]), ("gate_r", gr, v["dgate_r"]), ("gate_i", gi, v["dgate_i"]),
                       ("decay", decay, v["ddecay"]), ("h0", h0, v["dh0"])):
        inside = ~np.isnan(g)
        assert np.max(np.abs(diff(f, t) - np.where(inside, g, 0.0))) <= TOL, name


# ---------------------------------------------------------------- refusals
BAD = 0x1000  # never dereferenced: the host's checks come first


def ln_args(**kw):
    a = kb.KmbLayerNorm()
    for k, n in enumerate(("x", "y", "dy", "dx", "dweight")):
        setattr(a, n, BAD + 4096 * k)
    a.rows, a.D, a.eps = 4, 8, 1e-5
    a.ld_x = a.ld_y = a.ld_dy = a.ld_dx = 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), b"sizes"), (dict(D=0), b"sizes"), (dict(x=None), b"x is required"),
    (dict(y=None), b"y is required"), (dict(ld_x=7), b"row stride"), (dict(ld_y=7), b"row stride"),
    (dict(x_type=2), b"type"), (dict(y_type=-1), b"type"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"), (dict(accumulate=2), b"accumulate"),
    (dict(x=BAD + 2), b"aligned"), (dict(y=BAD + 1, y_type=1), b"aligned"), (dict(weight=BAD + 1), b"aligned"),
    (dict(y=BAD, y_type=1), b"another type"), (dict(y=BAD, ld_y=9), b"another type"), (dict(), b"device memory")])
def test_layernorm_fwd_refuses(lib, kw, word):
    assert lib.kmb_layernorm_fwd(C.byref(ln_args(**kw))) == kb.KMB_EINVAL
    assert word in lib.kmb_last_error(), lib.kmb_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(dy=None), b"required"), (dict(dx=None), b"required"), (dict(mean=BAD), b"together"),
    (dict(rstd=BAD), b"together"), (dict(ld_dy=7), b"row stride"), (dict(ld_dx=7), b"row stride"),
    (dict(dres=BAD, ld_dres=7), b"row stride"), (dict(workspace=BAD, workspace_bytes=15), b"workspace"),
    (dict(workspace=BAD + 8, workspace_bytes=1 << 30), b"16-byte"), (dict(dbias=BAD + 2), b"aligned"),
    (dict(dx=BAD, ld_dx=9), b"another type"), (dict(dx=BAD + 4096 * 2, y_type=1), b"another type"),
    (dict(dres=BAD + 4096 * 3, ld_dres=9), b"another type"), (dict(), b"device memory")])
def test_layernorm_bwd_refuses(lib, kw, word):
    assert lib.kmb_layernorm_bwd(C.byref(ln_args(**kw))) == kb.KMB_EINVAL
    assert word in lib.kmb_last_error(), lib.kmb_last_error()


def test_layernorm_sizes(lib):
    assert lib.kmb_layernorm_bwd(None) == kb.KMB_EINVAL
    assert lib.kmb_layernorm_fwd(C.byref(ln_args(rows=1 << 31))) == kb.KMB_EUNSUPPORTED
    assert lib.kmb_layernorm_workspace_bytes(C.byref(ln_args(D=-1))) == 0
    assert lib.kmb_layernorm_workspace_bytes(C.byref(ln_args())) > 0


def glr_args(batch=2, L=5, D=8, **kw):
    a = kb.KmbGLR()
    a.batch, a.L, a.D, a.scale = batch, L, D, 8.0
    for k, n in enumerate(("x", "gate_r", "gate_i", "y", "dy", "dx", "dgate_r", "dgate_i")):
        setattr(a, n, kb.KmbRows(BAD + 4096 * k, D, L * D))
    a.decay = BAD
    for k, v in kw.items():
        setattr(a, k, v)
    return a


R = kb.KmbRows
FWD_BAD = [
    (dict(batch=-1), b"sizes"), (dict(L=-1), b"sizes"), (dict(D=0), b"sizes"), (dict(scale=0.0), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(type=2), b"type"),
    (dict(decay=None), b"decay"), (dict(decay=BAD + 2), b"aligned"), (dict(h_last=BAD + 1), b"aligned"),
    (dict(offsets=BAD + 4), b"aligned"), (dict(accumulate=-1), b"accumulate"),
    (dict(x=R(None, 8, 40)), b"x is required"), (dict(gate_r=R(BAD, 7, 40)), b"row stride of gate_r"),
    (dict(gate_i=R(BAD, 8, 7)), b"batch stride of gate_i"), (dict(x=R(BAD + 2, 8, 40)), b"x is not aligned"),
    (dict(), b"device memory")]


@pytest.mark.parametrize("kw,word", FWD_BAD + [(dict(y=R(BAD, 8, 39)), b"overlap"), (dict(y=R(BAD, 15, 8)), b"overlap"),
                                               (dict(y=R(None, 8, 40)), b"y is required"),
                                               (dict(y=R(BAD, 9, 45)), b"other strides")])
def test_glr_fwd_refuses(lib, kw, word):
    assert lib.kmb_glr_fwd(C.byref(glr_args(**kw))) == kb.KMB_EINVAL
    assert word in lib.kmb_last_error(), lib.kmb_last_error()


@pytest.mark.parametrize("kw,word", FWD_BAD + [(dict(dx=R(BAD, 8, 39)), b"overlap"), (dict(dy=R(None, 8, 40)), b"dy is required"),
                                               (dict(dgate_i=R(None, 8, 40)), b"dgate_i is required"),
                                               (dict(dx=R(BAD + 7 * 4096, 8, 40)), b"two outputs"),
                                               (dict(dgate_r=R(BAD, 8, 48)), b"other strides"),
                                               (dict(workspace=BAD, workspace_bytes=3), b"workspace"),
                                               (dict(workspace=BAD + 4, workspace_bytes=1 << 40), b"16-byte")])
def test_glr_bwd_refuses(lib, kw, word):
    assert lib.kmb_glr_bwd(C.byref(glr_args(**kw))) == kb.KMB_EINVAL
    assert word in lib.kmb_last_error(), lib.kmb_last_error()


def test_glr_sizes(lib):
    assert lib.kmb_glr_fwd(None) == kb.KMB_EINVAL and lib.kmb_glr_bwd(None) == kb.KMB_EINVAL
    assert lib.kmb_glr_fwd(C.byref(glr_args(batch=1 << 31))) == kb.KMB_EUNSUPPORTED
    assert lib.kmb_glr_fwd(C.byref(glr_args(batch=1 << 20, L=1 << 20))) == kb.KMB_EUNSUPPORTED
    assert lib.kmb_glr_ckpt_elems(C.byref(glr_args(batch=3, L=65, D=7))) == 3 * 3 * 7
    assert lib.kmb_glr_ckpt_elems(C.byref(glr_args(batch=3, L=57, D=7, type=kb.KMB_BF16))) == 3 * 2 * 7
    assert lib.kmb_glr_ckpt_elems(C.byref(glr_args(batch=3, L=65, D=7, offsets=BAD))) == 3 * 7
    assert lib.kmb_glr_ckpt_elems(C.byref(glr_args(batch=3, L=0, D=7))) == 0
    assert lib.kmb_glr_ckpt_elems(C.byref(glr_args(D=-1))) == 0
    # a time-major output passes the overlap check (and then fails on the pointers)
    lib.kmb_glr_fwd(C.byref(glr_args(y=R(BAD + 64, 16, 8))))
    assert b"device memory" in lib.kmb_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), b"sizes"), (dict(D=0), b"sizes"), (dict(state=None), b"state is required"),
    (dict(ld_state=7), b"state stride"), (dict(slots=None, n_states=3), b"fewer states"),
    (dict(slots=BAD + 4), b"slots"), (dict(scale=-1.0), b"scale"), (dict(type=7), b"type"),
    (dict(decay=None), b"decay"), (dict(x=R(None, 8, 0)), b"x is required"), (dict(y=R(BAD, 7, 0)), b"row stride"),
    (dict(state=BAD + 2), b"aligned"), (dict(), b"device memory")])
def test_glr_step_refuses(lib, kw, word):
    a = kb.KmbGLRStep()
    for n in ("x", "gate_r", "gate_i", "y"):
        setattr(a, n, kb.KmbRows(BAD, 8, 0))
    a.decay, a.state, a.slots, a.rows, a.n_states, a.D, a.ld_state, a.scale = BAD, BAD, BAD, 4, 6, 8, 8, 8.0
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.kmb_glr_step(C.byref(a)) == kb.KMB_EINVAL
    assert word in lib.kmb_last_error(), lib.kmb_last_error()
