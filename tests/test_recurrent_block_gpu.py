"""The operators as they are used together: a pre-norm recurrent block,
  n = LN(x);  [u | r | i] = n W^T;  h = GLR(u, r, i);  out = x + h V^T
on the library's layer norm, GEMM and gated linear recurrence, forward and
backward, against the same block in float64 torch with autograd.  The bf16
operands of both sides' GEMMs and the block's own bf16 tensors are rounded
where the library rounds them, so what is left is fp32 noise and single
roundings that fall to the neighbouring bf16 value: a value within fp32 noise
(2^-22 relative) of a boundary does so with probability 2^-22 / 2^-8 = 2^-14,
and moves by 2^-8; in the norm of a tensor that is 2^-8 * 2^-7 = 3e-5, here
through at most three roundings in a row and the recurrence's memory of about
ten steps: 1e-3."""
import ctypes as C

import numpy as np
import pytest
import torch

import kmamba_b200 as kb
from conftest import norm_err

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
TOL = 1e-3


def gemm(lib, A, B, out, M, N, K, a_mn=0, b_mn=0, residual=None):
    g = kb.KmbGemm()
    g.A, g.B, g.C = A.data_ptr(), B.data_ptr(), out.data_ptr()
    g.M, g.N, g.K = M, N, K
    g.lda, g.ldb, g.ldc, g.ldr = A.stride(0), B.stride(0), out.stride(0), out.stride(0)
    g.a_mn_major, g.b_mn_major, g.c_bf16 = a_mn, b_mn, int(out.dtype == BF)
    if residual is not None:
        g.residual = residual.data_ptr()
    kb.check(lib, lib.kmb_gemm_bf16(C.byref(g)))


class RoundBf(torch.autograd.Function):
    """bf16 rounding of a tensor and of its gradient."""

    @staticmethod
    def forward(ctx, x):
        return x.float().to(BF).double()

    @staticmethod
    def backward(ctx, g):
        return g.float().to(BF).double()


class RoundFwd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.float().to(BF).double()

    @staticmethod
    def backward(ctx, g):
        return g


class RoundGrad(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        return g.float().to(BF).double()


@pytest.mark.parametrize("batch,L,d", [(2, 130, 64), (1, 257, 128), (3, 48, 192)])
def test_block(lib, cuda, batch, L, d):
    rng = np.random.default_rng(d)
    T = batch * L
    t64 = lambda a: torch.from_numpy(np.asarray(a, np.float32)).double().cuda()  # noqa: E731
    x = t64(rng.standard_normal((T, d)))
    w, b = t64(1 + 0.1 * rng.standard_normal(d)), t64(0.1 * rng.standard_normal(d))
    W = t64(rng.standard_normal((3 * d, d)) / np.sqrt(d)).to(BF).double()
    V = t64(rng.standard_normal((d, d)) / np.sqrt(d)).to(BF).double()
    a_open = rng.uniform(0.5, 0.9, d)
    decay = t64(np.log(np.expm1(-np.log(a_open) / 8)))
    dout = t64(rng.standard_normal((T, d)))

    # ---- float64
    leaves = [v.clone().requires_grad_(True) for v in (x, w, b, W, V, decay)]
    X, ww, bb, WW, VV, dd = leaves
    c = X - X.mean(1, keepdim=True)
    n = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * ww + bb
    p = RoundBf.apply(RoundFwd.apply(n) @ WW.T).view(batch, L, 3 * d)
    u, r, i = p[..., :d], torch.sigmoid(p[..., d:2 * d]), torch.sigmoid(p[..., 2 * d:])
    e = 8 * torch.nn.functional.softplus(dd) * r
    a, inp = torch.exp(-e), torch.sqrt(-torch.expm1(-2 * e)) * i * u
    h, hs = torch.zeros(batch, d, dtype=torch.float64, device="cuda"), []
    for t in range(L):
        h = a[:, t] * h + inp[:, t]
        hs.append(h)
    hseq = RoundBf.apply(torch.stack(hs, 1).reshape(T, d))
    out = X + RoundGrad.apply(hseq @ VV.T)
    (out * dout).sum().backward()

    # ---- the library
    f = lambda v: v.float().contiguous()  # noqa: E731
    xg, wg, bg, dg, dog = f(x), f(w), f(b), f(decay), f(dout)
    Wg, Vg = W.to(BF).contiguous(), V.to(BF).contiguous()
    n16 = torch.empty(T, d, dtype=BF, device="cuda")
    mean, rstd = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    ln = kb.KmbLayerNorm()
    ln.x, ln.weight, ln.bias, ln.y, ln.mean, ln.rstd = (v.data_ptr() for v in (xg, wg, bg, n16, mean, rstd))
    ln.rows, ln.D, ln.ld_x, ln.ld_y, ln.eps, ln.y_type = T, d, d, d, 1e-5, kb.KMB_BF16
    kb.check(lib, lib.kmb_layernorm_fwd(C.byref(ln)))
    proj = torch.empty(T, 3 * d, dtype=BF, device="cuda")
    gemm(lib, n16, Wg, proj, T, 3 * d, d)
    hy = torch.empty(T, d, dtype=BF, device="cuda")
    g = kb.KmbGLR()
    part = lambda m, k: kb.KmbRows(m.data_ptr() + 2 * k * d, 3 * d, L * 3 * d)  # noqa: E731
    g.x, g.gate_r, g.gate_i = part(proj, 0), part(proj, 1), part(proj, 2)
    g.y = kb.KmbRows(hy.data_ptr(), d, L * d)
    g.decay, g.batch, g.L, g.D, g.scale, g.type = dg.data_ptr(), batch, L, d, 8.0, kb.KMB_BF16
    ckpt = torch.empty(lib.kmb_glr_ckpt_elems(C.byref(g)), device="cuda")
    g.ckpt = ckpt.data_ptr()
    kb.check(lib, lib.kmb_glr_fwd(C.byref(g)))
    og = torch.empty(T, d, device="cuda")
    gemm(lib, hy, Vg, og, T, d, d, residual=xg)
    # backward
    do16 = dog.to(BF)
    dh16 = torch.empty(T, d, dtype=BF, device="cuda")
    dV, dW = torch.empty(d, d, device="cuda"), torch.empty(3 * d, d, device="cuda")
    gemm(lib, do16, Vg, dh16, T, d, d, b_mn=1)
    gemm(lib, do16, hy, dV, d, d, T, a_mn=1, b_mn=1)
    dproj = torch.empty_like(proj)
    ddecay = torch.empty(d, device="cuda")
    g.dy = kb.KmbRows(dh16.data_ptr(), d, L * d)
    g.dx, g.dgate_r, g.dgate_i = part(dproj, 0), part(dproj, 1), part(dproj, 2)
    g.ddecay = ddecay.data_ptr()
    kb.check(lib, lib.kmb_glr_bwd(C.byref(g)))
    dn = torch.empty(T, d, device="cuda")
    gemm(lib, dproj, Wg, dn, T, d, 3 * d, b_mn=1)
    gemm(lib, dproj, n16, dW, 3 * d, d, T, a_mn=1, b_mn=1)
    dxg, dw, db = torch.empty(T, d, device="cuda"), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    lb = kb.KmbLayerNorm()
    lb.x, lb.weight, lb.mean, lb.rstd, lb.dy, lb.dres, lb.dx, lb.dweight, lb.dbias = (
        v.data_ptr() for v in (xg, wg, mean, rstd, dn, dog, dxg, dw, db))
    lb.rows, lb.D, lb.ld_x, lb.ld_dy, lb.ld_dres, lb.ld_dx, lb.eps = T, d, d, d, d, d, 1e-5
    kb.check(lib, lib.kmb_layernorm_bwd(C.byref(lb)))
    torch.cuda.synchronize()
    got = {"out": og, "x": dxg, "w": dw, "b": db, "W": dW, "V": dV, "decay": ddecay}
    want = {"out": out.detach()} | {k: v.grad for k, v in zip(("x", "w", "b", "W", "V", "decay"), leaves)}
    for k in got:
        err = norm_err(got[k].double().cpu().numpy(), want[k].cpu().numpy())
        assert err <= TOL, (k, err)
