"""GPU parity of the pre-norm Mamba-ND model (kmb_ndmodel_create_prenorm)
against its float64 torch restatement (oracle/ndmodel_ref.py): loss, every
parameter gradient, and one AdamW step, with the batch whole and as
micro-batches whose gradients accumulate.  Tolerances as in
test_ndmodel_gpu.py, whose reasons hold here: the GEMM operands of both sides
are rounded to bf16, and an operand within fp32 noise of a rounding boundary
goes to neighbouring values on the two sides."""
import ctypes as C

import numpy as np
import pytest

from conftest import norm_err, rel_err
from test_ndmodel_gpu import device_array, flatten, split

import kmamba_b200 as kb

pytestmark = pytest.mark.gpu
EPS = 1e-3


def config(dims, d, L, micro=0):
    cfg = kb.KmbNDModelConfig()
    for i in range(3):
        cfg.dims[i] = dims[i]
    cfg.dim, cfg.n_layers, cfg.vocab, cfg.seed, cfg.micro_batch = d, L, 256, 1234, micro
    return cfg


def split_norms(flat, d, L, V):
    """The flat layout with the norms behind the layers."""
    import torch
    n = 2 * (L + 1) * d
    tree = split(flat[:-n], d, L, V)
    norms = torch.tensor(flat[-n:].reshape(L + 1, 2, d), dtype=torch.float64)
    for i, part in enumerate(tree["layers"] + [tree]):
        part["norm_weight"], part["norm_bias"] = norms[i, 0].clone(), norms[i, 1].clone()
    return tree


@pytest.mark.parametrize("dims,d,L,batch,micro", [([3, 4, 5], 32, 2, 2, 0), ([6, 6, 6], 64, 2, 1, 0),
                                                  ([4, 5, 3], 32, 2, 3, 2)])
def test_loss_gradients_and_step(lib, cuda, dims, d, L, batch, micro):
    import torch
    import ndmodel_ref as ref
    V = 256
    plain = lib.kmb_ndmodel_create(C.byref(config(dims, d, L, micro)))
    m = lib.kmb_ndmodel_create_prenorm(C.byref(config(dims, d, L, micro)), EPS)
    assert m and plain, kb.last_error(lib)
    try:
        n = lib.kmb_ndmodel_param_count(m)
        n0 = lib.kmb_ndmodel_param_count(plain)
        assert n == n0 + 2 * (L + 1) * d
        start = device_array(lib.kmb_ndmodel_params(m), n)
        # the same weights as without norms, then ones and zeros
        assert np.array_equal(start[:n0], device_array(lib.kmb_ndmodel_params(plain), n0))
        assert np.array_equal(start[n0:].reshape(L + 1, 2, d)[:, 0], np.ones((L + 1, d)))
        assert np.array_equal(start[n0:].reshape(L + 1, 2, d)[:, 1], np.zeros((L + 1, d)))
        rng = np.random.default_rng(sum(dims) + d)
        # weights and biases that are not at their start
        norms = start[n0:].reshape(L + 1, 2, d) + 0.2 * rng.standard_normal((L + 1, 2, d)).astype(np.float32)
        rt = C.CDLL("libcudart.so.12")
        rt.cudaMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
        norms = np.ascontiguousarray(norms, np.float32)
        assert rt.cudaMemcpy(lib.kmb_ndmodel_params(m) + 4 * n0, norms.ctypes.data, norms.nbytes, 1) == 0
        P = int(np.prod(dims))
        tok = rng.integers(0, V, (batch, P), dtype=np.uint32)
        ttok = torch.from_numpy(tok.astype(np.int32)).cuda()
        loss = C.c_float()
        kb.check(lib, lib.kmb_ndmodel_backward(m, ttok.data_ptr(), batch, C.byref(loss)))
        flat = device_array(lib.kmb_ndmodel_params(m), n)
        grads = device_array(lib.kmb_ndmodel_grads(m), n)
        tree = split_norms(flat, d, L, V)
        leaves = flatten(tree)
        for part in tree["layers"] + [tree]:
            leaves += [part["norm_weight"], part["norm_bias"]]
        for t in leaves:
            t.requires_grad_(True)
        want = ref.forward_loss(tree, torch.from_numpy(tok.astype(np.int64)), dims, eps=EPS)
        want.backward()
        assert abs(loss.value - want.item()) <= 1e-4 * abs(want.item()), (loss.value, want.item())
        o = 0
        for k, t in enumerate(leaves):
            g_ref = t.grad.numpy().ravel()
            g = grads[o:o + g_ref.size]
            o += g_ref.size
            assert norm_err(g, g_ref) <= 5e-3, (k, norm_err(g, g_ref))
            assert rel_err(g, g_ref) <= 0.2, (k, rel_err(g, g_ref))
        assert o == n
        lr, wd = 1e-3, 0.01
        kb.check(lib, lib.kmb_ndmodel_step(m, lr, wd))
        new = device_array(lib.kmb_ndmodel_params(m), n)
        g = grads.astype(np.float64)
        upd = flat * (1 - lr * wd) - lr * g / (np.abs(g) + 1e-8)
        assert np.max(np.abs(new - upd)) <= 1e-4 * lr + 1e-6 * np.max(np.abs(flat))
        f = C.c_float()
        kb.check(lib, lib.kmb_ndmodel_forward(m, ttok.data_ptr(), batch, C.byref(f)))
        assert np.isfinite(f.value)
    finally:
        lib.kmb_ndmodel_free(m)
        lib.kmb_ndmodel_free(plain)


def test_refusals(lib):
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        assert not lib.kmb_ndmodel_create_prenorm(C.byref(config([4, 4, 4], 32, 1)), eps)
        assert b"norm_eps" in lib.kmb_last_error()
    assert not lib.kmb_ndmodel_create_prenorm(C.byref(config([4, 4, 4], 48, 1)), 1e-5)
    assert b"multiple of 32" in lib.kmb_last_error()


def test_expired_wait_is_reported(lib, cuda):
    """A layer norm whose wait gave up: the model's call that finds the word
    returns KMB_ETIMEOUT, and the next is as it was."""
    import torch
    m = lib.kmb_ndmodel_create_prenorm(C.byref(config([6, 6, 6], 256, 1)), EPS)
    plain = lib.kmb_ndmodel_create(C.byref(config([6, 6, 6], 256, 1)))
    assert m and plain, kb.last_error(lib)
    try:
        tok = torch.randint(0, 256, (2, 216), dtype=torch.int32, device="cuda")
        want, got = C.c_float(), C.c_float()
        kb.check(lib, lib.kmb_ndmodel_forward(m, tok.data_ptr(), 2, C.byref(want)))
        for call in (lambda: lib.kmb_ndmodel_forward(m, tok.data_ptr(), 2, C.byref(got)),
                     lambda: lib.kmb_ndmodel_backward(m, tok.data_ptr(), 2, C.byref(got))):
            assert lib.kmb_layernorm_expire() == kb.KMB_OK
            assert call() == kb.KMB_ETIMEOUT
            assert b"a wait for a row expired" in lib.kmb_last_error()
            kb.check(lib, call())
            assert got.value == want.value
        # a model without norms does not ask for the word
        assert lib.kmb_layernorm_expire() == kb.KMB_OK
        kb.check(lib, lib.kmb_ndmodel_forward(plain, tok.data_ptr(), 2, C.byref(got)))
    finally:
        lib.kmb_layernorm_check_error()
        lib.kmb_ndmodel_free(m)
        lib.kmb_ndmodel_free(plain)


def test_gradients_through_a_communicator(lib, cuda):
    """With a communicator of one rank, whose mean is the gradient itself:
    every gradient goes through the buckets once, the norms' among them.  Two
    backward passes differ by the order of atomic sums, some d = 2^-20 of a
    value, which sends a share d / 2^-8 of the bf16 operands behind them to the
    other neighbour, a step of 2^-8: sqrt(2^-8 d) = 2^-14 in norm for each of
    the rounded tensors on the way, up to 7 a layer, 2 layers and the head's 2:
    4 2^-14 when they add up as squares."""
    import torch
    cfg = config([6, 6, 6], 64, 2)
    uid = C.create_string_buffer(128)
    assert lib.kmb_dist_get_unique_id(uid) == kb.KMB_OK
    ctx = lib.kmb_dist_init_with_id(1, 0, torch.cuda.current_device(), uid)
    assert ctx, kb.last_error(lib)
    m = lib.kmb_ndmodel_create_prenorm(C.byref(cfg), EPS)
    assert m, kb.last_error(lib)
    try:
        n = lib.kmb_ndmodel_param_count(m)
        tok = torch.randint(0, 256, (2, 216), dtype=torch.int32, device="cuda")
        loss = C.c_float()
        kb.check(lib, lib.kmb_ndmodel_backward(m, tok.data_ptr(), 2, C.byref(loss)))
        want = device_array(lib.kmb_ndmodel_grads(m), n)
        kb.check(lib, lib.kmb_ndmodel_set_dist(m, ctx))
        first, last = C.c_ulonglong(), C.c_ulonglong()
        lib.kmb_dist_stats(ctx, None, C.byref(first))
        kb.check(lib, lib.kmb_ndmodel_backward(m, tok.data_ptr(), 2, C.byref(loss)))
        torch.cuda.synchronize()
        lib.kmb_dist_stats(ctx, None, C.byref(last))
        assert last.value - first.value == 4 * n
        got = device_array(lib.kmb_ndmodel_grads(m), n)
        norms = 2 * 3 * 64
        assert np.abs(want[-norms:]).max() > 0
        assert norm_err(got[-norms:], want[-norms:]) <= 2.0 ** -12 and norm_err(got, want) <= 2.0 ** -12
        kb.check(lib, lib.kmb_ndmodel_set_dist(m, None))
    finally:
        lib.kmb_ndmodel_free(m)
        lib.kmamba_distributed_fini_nccl(ctx)
