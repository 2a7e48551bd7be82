"""Cases of the layer norm and the gated linear recurrence: what a pass of
each costs, in the framework's kernels (`own`) or in elementary torch
operations.

Operators (D channels, every sum and state in 32 bits):

  ln_fwd   y = (x - mean) rstd weight + bias per row, and mean, rstd
  ln_bwd   dx (plus the residual stream's gradient), dweight, dbias
  glr_fwd  h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gate_i) x,
           a_t = exp(-scale softplus(decay) sigmoid(gate_r)), every h_t and
           the last one of each sequence
  glr_train  the same forward, then its adjoint: gradients of x, both gates,
           decay and the first state
  glr_step  one token for each row of a serving batch; states live in slots
"""
import math
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SCALE = 8.0
EPS = 1e-5


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step's norm: latency of a call
        {"name": "ln_fwd_token", "op": "ln_fwd", "rows": 4, "D": 1024, "xt": "f32", "yt": "bf16", "gap": 0},
        # the residual stream of one 64^3 volume at dim 1024, bf16 for the projections that follow
        {"name": "ln_fwd_volume", "op": "ln_fwd", "rows": 262144, "D": 1024, "xt": "f32", "yt": "bf16", "gap": 0},
        # a bf16 stream of odd width whose rows are slices of a wider matrix
        {"name": "ln_fwd_odd", "op": "ln_fwd", "rows": 16411, "D": 1537, "xt": "bf16", "yt": "bf16", "gap": 5},
        # backward of the volume's norm, joined with the residual stream's gradient
        {"name": "ln_bwd_volume", "op": "ln_bwd", "rows": 262144, "D": 1024, "xt": "f32", "yt": "f32", "gap": 0, "res": True},
        # a wide model's backward on few rows
        {"name": "ln_bwd_wide", "op": "ln_bwd", "rows": 2048, "D": 8192, "xt": "bf16", "yt": "bf16", "gap": 0, "res": False},
        # one short sequence (128 tokens, dim 384) in training: launches count
        {"name": "ln_bwd_small", "op": "ln_bwd", "rows": 128, "D": 384, "xt": "f32", "yt": "f32", "gap": 0, "res": False},
        # prefill of one long document
        {"name": "glr_fwd_long", "op": "glr_fwd", "batch": 1, "L": 65536, "D": 2048, "type": "bf16", "packed": False, "fused": False},
        # a batch of 8 x 4096 tokens at 1536 channels in fp32
        {"name": "glr_fwd_batch", "op": "glr_fwd", "batch": 8, "L": 4096, "D": 1536, "type": "f32", "packed": False, "fused": False},
        # training step of the same batch in bf16, inputs read from one fused projection
        {"name": "glr_train_batch", "op": "glr_train", "batch": 8, "L": 4096, "D": 1536, "type": "bf16", "packed": False, "fused": True},
        # training on packed ragged documents, odd width
        {"name": "glr_train_packed", "op": "glr_train", "batch": 37, "L": 24001, "D": 771, "type": "f32", "packed": True, "fused": True},
        # decoding: a handful of users
        {"name": "glr_step_small", "op": "glr_step", "rows": 4, "D": 1536, "type": "bf16", "slots": 16},
        # decoding: a full serving batch
        {"name": "glr_step_batch", "op": "glr_step", "rows": 512, "D": 4096, "type": "f32", "slots": 1024},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ln_fwd", "ln_bwd", "glr_fwd", "glr_train", "glr_step"))
    if op in ("ln_fwd", "ln_bwd"):
        D = _log(rng, 32, 20000)
        rows = _log(rng, 1, max(2, min(262144, (1 << 26) // D)))
        xt, yt = rng.choice((("f32", "bf16"), ("f32", "f32"), ("bf16", "bf16")))
        case = {"op": op, "rows": rows, "D": D, "xt": xt, "yt": yt, "gap": rng.choice((0, 0, 3, 8))}
        if op == "ln_bwd":
            case["res"] = rng.random() < 0.5
        return case
    if op == "glr_step":
        rows = _log(rng, 1, 512)
        return {"op": op, "rows": rows, "D": _log(rng, 64, 4096), "type": rng.choice(("f32", "bf16")),
                "slots": rows + _log(rng, 1, 512)}
    D = _log(rng, 64, 4096)
    rows = _log(rng, 64, max(65, min(65536, (1 << 25) // D)))
    packed = rng.random() < 0.4
    batch = _log(rng, 1, min(64, rows))
    return {"op": op, "batch": batch, "L": rows if packed else max(1, rows // batch), "D": D,
            "type": rng.choice(("f32", "bf16")), "packed": packed, "fused": rng.random() < 0.5}


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    op, D = case["op"], case["D"]
    s = {"case": case}
    if op in ("ln_fwd", "ln_bwd"):
        rows, ld = case["rows"], D + case["gap"]
        xt, yt = TYPES[case["xt"]], TYPES[case["yt"]]

        def strided(dtype):
            return torch.empty(rows, ld, dtype=dtype, device="cuda")[:, :D]

        # a residual stream: per-row scale and a common offset
        x = strided(xt)
        x.copy_(normal(rows, D) * (0.5 + 2.5 * torch.rand(rows, 1, generator=g, device="cuda")) + 0.3)
        s.update(x=x, weight=1 + 0.1 * normal(D), bias=0.1 * normal(D))
        if op == "ln_fwd":
            s.update(y=strided(yt), mean=torch.empty(rows, device="cuda"), rstd=torch.empty(rows, device="cuda"))
            return s
        f = x.float()
        mean = f.mean(1)
        s.update(mean=mean, rstd=torch.rsqrt((f - mean[:, None]).square().mean(1) + EPS))
        dy = strided(yt)
        dy.copy_(normal(rows, D))
        s.update(dy=dy, dx=strided(xt), dweight=torch.empty(D, device="cuda"), dbias=torch.empty(D, device="cuda"))
        if case["res"]:
            s["dres"] = strided(xt)
            s["dres"].copy_(normal(rows, D))
        return s
    t = TYPES[case["type"]]
    # decay so that a at a fully open gate is uniform in [0.9, 0.999]
    open_a = 0.9 + 0.099 * torch.rand(D, generator=g, device="cuda")
    s["decay"] = torch.log(torch.expm1(-torch.log(open_a) / SCALE))
    if op == "glr_step":
        rows, n = case["rows"], case["slots"]
        p = normal(rows, 3 * D, dtype=t)  # one projection of the batch
        slots = torch.randperm(n, generator=g, device="cuda")[:rows]
        if rows > 2:
            slots[rows // 2] = -1  # a padded row
        s.update(x=p[:, :D], gate_r=p[:, D:2 * D], gate_i=p[:, 2 * D:], slots=slots, state=normal(n, D),
                 y=torch.zeros(rows, D, dtype=t, device="cuda"))
        return s
    lead = (case["L"],) if case["packed"] else (case["batch"], case["L"])
    if case["fused"]:
        p = normal(*lead, 3 * D, dtype=t)
        s.update(x=p[..., :D], gate_r=p[..., D:2 * D], gate_i=p[..., 2 * D:])
    else:
        s.update(x=normal(*lead, D, dtype=t), gate_r=normal(*lead, D, dtype=t), gate_i=normal(*lead, D, dtype=t))
    n = case["batch"]
    s.update(h0=normal(n, D), h_last=torch.empty(n, D, device="cuda"), y=torch.empty(*lead, D, dtype=t, device="cuda"))
    if case["packed"]:
        # ragged documents: random cuts, so that lengths of zero and one occur
        cuts = torch.randint(0, case["L"] + 1, (n - 1,), generator=g, device="cuda").sort().values
        if n > 4:
            cuts[1] = cuts[0]
            cuts[3] = torch.minimum(cuts[2] + 1, cuts[3])
        ends = torch.tensor([0, case["L"]], device="cuda")
        s["offsets"] = torch.cat([ends[:1], cuts, ends[1:]])
    if op == "glr_train":
        s.update(dy=normal(*lead, D, dtype=t), dh_last=normal(n, D), dh0=torch.empty(n, D, device="cuda"),
                 ddecay=torch.empty(D, device="cuda"))
        d = torch.empty(*lead, 3 * D, dtype=t, device="cuda")  # gradient of the fused projection
        s.update(dx=d[..., :D], dgate_r=d[..., D:2 * D], dgate_i=d[..., 2 * D:])
    return s


# ------------------------------------------------------- the plain forms
def _plain_ln_fwd(s):
    x = s["x"].float()
    mean = x.mean(1)
    xc = x - mean[:, None]
    rstd = torch.rsqrt(xc.square().mean(1) + EPS)
    y = xc * rstd[:, None] * s["weight"] + s["bias"]
    return {"y": y.to(s["y"].dtype), "mean": mean, "rstd": rstd}


def _plain_ln_bwd(s):
    x, dy, rstd = s["x"].float(), s["dy"].float(), s["rstd"][:, None]
    xhat = (x - s["mean"][:, None]) * rstd
    wdy = dy * s["weight"]
    dx = (wdy - wdy.mean(1, keepdim=True) - xhat * (wdy * xhat).mean(1, keepdim=True)) * rstd
    if "dres" in s:
        dx = dx + s["dres"].float()
    # sums over all rows: in 64 bits
    return {"dx": dx.to(s["dx"].dtype), "dweight": (dy * xhat).sum(0, dtype=torch.float64).float(),
            "dbias": dy.sum(0, dtype=torch.float64).float()}


def _gates(x, gate_r, gate_i, decay):
    """(r, i, u, a, root, b): both gates, the log decay u = -log a, the decay, sqrt(1 - a^2) and the input term."""
    r, i = torch.sigmoid(gate_r.float()), torch.sigmoid(gate_i.float())
    u = SCALE * torch.nn.functional.softplus(decay) * r
    root = torch.sqrt(-torch.expm1(-2 * u))
    # next to one, where a long memory multiplies the error of a: its exponential in 64 bits, rounded once
    a = torch.exp(-u.double()).float()
    return r, i, u, a, root, root * i * x.float()


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h = 0, by doubling the reach of each entry."""
    reach, L = 1, a.shape[1]
    while reach < L:
        b = torch.cat([b[:, :reach], b[:, reach:] + a[:, reach:] * b[:, :-reach]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return b


def _edges(s):
    """Rows where sequences begin and end (flat over batch and time) and the sequences that have rows."""
    n, L = s["case"]["batch"], s["case"]["L"]
    off = s["offsets"] if "offsets" in s else torch.arange(n + 1, device="cuda") * L
    some = (off[1:] > off[:-1]).nonzero()[:, 0]
    return off[some], off[some + 1] - 1, some


def _plain_glr(s, train):
    D, dt = s["case"]["D"], s["y"].dtype
    first, last, some = _edges(s)
    shape = s["x"].shape if s["x"].dim() == 3 else (1, *s["x"].shape)
    r, i, u, a, root, b = _gates(s["x"], s["gate_r"], s["gate_i"], s["decay"])

    def flat(v):
        return v.reshape(-1, D)

    # a sequence's first row takes its h0 and nothing of the row before it
    before = torch.zeros_like(flat(a))
    before[first] = s["h0"][some]
    carry = flat(a).clone()
    carry[first] = 0
    h = flat(_scan(carry.view(shape), (flat(b) + flat(a) * before).view(shape)))
    h_last = s["h0"].clone()
    h_last[some] = h[last]
    y = h.to(dt).view(s["y"].shape)
    if not train:
        return {"y": y, "h_last": h_last}
    # adjoint: G_t = dy_t + a_{t+1} G_{t+1}
    dy = flat(s["dy"].float()).clone()
    dy[last] += s["dh_last"][some]
    carry = torch.cat([flat(a)[1:], torch.zeros_like(flat(a)[:1])])
    carry[last] = 0
    G = flat(_scan(carry.view(shape).flip(1), dy.view(shape).flip(1)).flip(1))
    prev = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    prev[first] = s["h0"][some]
    r, i, u, a, root, b = (flat(v) for v in (r, i, u, a, root, b))
    dh0 = s["dh_last"].clone()
    dh0[some] = (a * G)[first]
    # u dL/du = G (u a^2 / (1 - a^2) b - u a h_{t-1})
    udu = G * (u * a * a / (-torch.expm1(-2 * u)) * b - u * a * prev)
    ratio = torch.sigmoid(s["decay"]) / torch.nn.functional.softplus(s["decay"])
    to = (s["dx"].shape, dt)
    return {"y": y, "h_last": h_last, "dh0": dh0,
            "dx": (G * root * i).to(to[1]).view(to[0]),
            "dgate_r": (udu * (1 - r)).to(to[1]).view(to[0]),
            "dgate_i": (G * b * (1 - i)).to(to[1]).view(to[0]),
            "ddecay": (udu.sum(0, dtype=torch.float64) * ratio).float()}


def _plain_step(s):
    live = (s["slots"] >= 0)[:, None]
    at = s["slots"].clamp(min=0)
    _, _, _, a, _, b = _gates(s["x"], s["gate_r"], s["gate_i"], s["decay"])
    h = a * s["state"][at] + b
    # padded rows write to no slot: they are sent behind the last one
    grown = torch.cat([s["state"], torch.zeros_like(s["state"][:1])])
    grown[torch.where(s["slots"] >= 0, s["slots"], s["state"].shape[0])] = h
    s["state"].copy_(grown[:-1])
    return {"y": torch.where(live, h, 0.0).to(s["y"].dtype), "state": s["state"]}


# ------------------------------------------------- the framework's kernels
_framework = None


def _lib():
    """(library, its Python declarations), asynchronous on torch's stream."""
    global _framework
    if _framework is None:
        sys.path.insert(0, "k-mamba_b200")
        import kmamba_b200 as kb
        lib = kb.load()
        lib.kmb_set_sync(0)
        _framework = (lib, kb)
    lib, kb = _framework
    lib.kmb_set_stream(torch.cuda.current_stream().cuda_stream)
    return lib, kb


def _rows(kb, t):
    return kb.KmbRows(t.data_ptr(), t.stride(-2), t.stride(0) if t.dim() == 3 else 0)


def _ln_args(s):
    import ctypes
    lib, kb = _lib()
    a, c = kb.KmbLayerNorm(), s["case"]
    for name in ("x", "weight", "bias", "y", "mean", "rstd", "dy", "dres", "dx", "dweight", "dbias"):
        if name in s:
            setattr(a, name, s[name].data_ptr())
    for name in ("x", "y", "dy", "dres", "dx"):
        if name in s:
            setattr(a, "ld_" + name, s[name].stride(0))
    a.rows, a.D, a.eps = c["rows"], c["D"], EPS
    a.x_type = kb.KMB_BF16 if c["xt"] == "bf16" else kb.KMB_F32
    a.y_type = kb.KMB_BF16 if c["yt"] == "bf16" else kb.KMB_F32
    if c["op"] == "ln_bwd":
        s["workspace"] = torch.empty(lib.kmb_layernorm_workspace_bytes(ctypes.byref(a)), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    return a


def _glr_args(s):
    import ctypes
    lib, kb = _lib()
    a, c = kb.KmbGLR(), s["case"]
    for name in ("x", "gate_r", "gate_i", "y", "dy", "dx", "dgate_r", "dgate_i"):
        if name in s:
            setattr(a, name, _rows(kb, s[name]))
    for name in ("decay", "h0", "h_last", "dh_last", "dh0", "ddecay", "offsets"):
        if name in s:
            setattr(a, name, s[name].data_ptr())
    a.batch, a.L, a.D, a.scale = c["batch"], c["L"], c["D"], SCALE
    a.type = kb.KMB_BF16 if c["type"] == "bf16" else kb.KMB_F32
    train = int(c["op"] == "glr_train")
    if train:
        s["ckpt"] = torch.empty(lib.kmb_glr_ckpt_elems(ctypes.byref(a)), device="cuda")
        a.ckpt = s["ckpt"].data_ptr()
    s["workspace"] = torch.empty(max(1, lib.kmb_glr_workspace_bytes(ctypes.byref(a), train)), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    return a


def _step_args(s):
    _, kb = _lib()
    a, c = kb.KmbGLRStep(), s["case"]
    for name in ("x", "gate_r", "gate_i", "y"):
        setattr(a, name, _rows(kb, s[name]))
    a.decay, a.state, a.slots = s["decay"].data_ptr(), s["state"].data_ptr(), s["slots"].data_ptr()
    a.rows, a.n_states, a.D, a.ld_state, a.scale = c["rows"], c["slots"], c["D"], s["state"].stride(0), SCALE
    a.type = kb.KMB_BF16 if c["type"] == "bf16" else kb.KMB_F32
    return a


ARGS = {"ln_fwd": _ln_args, "ln_bwd": _ln_args, "glr_fwd": _glr_args, "glr_train": _glr_args, "glr_step": _step_args}
CALLS = {"ln_fwd": ("kmb_layernorm_fwd",), "ln_bwd": ("kmb_layernorm_bwd",), "glr_fwd": ("kmb_glr_fwd",),
         "glr_train": ("kmb_glr_fwd", "kmb_glr_bwd"), "glr_step": ("kmb_glr_step",)}
OUTPUTS = {"ln_fwd": ("y", "mean", "rstd"), "ln_bwd": ("dx", "dweight", "dbias"), "glr_fwd": ("y", "h_last"),
           "glr_train": ("y", "h_last", "dh0", "dx", "dgate_r", "dgate_i", "ddecay"), "glr_step": ("y", "state")}


def _own(s):
    import ctypes
    lib, kb = _lib()
    op = s["case"]["op"]
    if "args" not in s:  # the argument struct, its workspace and checkpoints stay with the buffers
        s["args"] = ARGS[op](s)
    for name in CALLS[op]:
        kb.check(lib, getattr(lib, name)(ctypes.byref(s["args"])))
    return {k: s[k] for k in OUTPUTS[op]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "ln_fwd":
        return _plain_ln_fwd(state)
    if op == "ln_bwd":
        return _plain_ln_bwd(state)
    if op == "glr_step":
        return _plain_step(state)
    return _plain_glr(state, op == "glr_train")


# ------------------------------------------------------------------- work
def work(case):
    op, D = case["op"], case["D"]
    size = {"f32": 4, "bf16": 2}
    if op in ("ln_fwd", "ln_bwd"):
        n, xs, ys = case["rows"] * D, size[case["xt"]], size[case["yt"]]
        if op == "ln_fwd":
            return {"bytes": n * (xs + ys) + 8 * case["rows"] + 8 * D, "flops": 8 * n}
        return {"bytes": n * ((3 if case["res"] else 2) * xs + ys) + 8 * case["rows"] + 12 * D, "flops": 14 * n}
    es = size[case["type"]]
    if op == "glr_step":
        n = case["rows"] * D
        return {"bytes": n * (4 * es + 8) + 8 * case["rows"] + 4 * D, "flops": 20 * n}
    rows = case["L"] if case["packed"] else case["batch"] * case["L"]
    n, ends = rows * D, 8 * case["batch"] * D
    if op == "glr_fwd":
        return {"bytes": 4 * es * n + ends + 4 * D, "flops": 20 * n}
    # forward and backward: the inputs are needed once in each
    return {"bytes": (4 + 7) * es * n + 2 * ends + 12 * D, "flops": 60 * n}


# ------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    own_state = prepare(case, seed)
    v = {k: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for k, t in own_state.items()}
    op, D = case["op"], case["D"]
    if op == "ln_fwd":
        var, mean = torch.var_mean(v["x"], dim=1, correction=0)
        rstd = 1 / (var + EPS).sqrt()
        return {"y": torch.addcmul(v["bias"], (v["x"] - mean.unsqueeze(1)) * rstd.unsqueeze(1), v["weight"]), "mean": mean, "rstd": rstd}
    if op == "ln_bwd":
        xhat = (v["x"] - v["mean"].unsqueeze(1)) * v["rstd"].unsqueeze(1)
        along = torch.einsum("nd,nd,d->n", v["dy"], xhat, v["weight"]) / D
        flat = torch.mv(v["dy"], v["weight"]) / D
        dx = v["rstd"].unsqueeze(1) * (v["dy"] * v["weight"] - flat.unsqueeze(1) - xhat * along.unsqueeze(1))
        return {"dx": dx + v["dres"] if case["res"] else dx, "dweight": torch.einsum("nd,nd->d", v["dy"], xhat), "dbias": v["dy"].sum(0)}

    rate = SCALE * torch.where(v["decay"] > 30, v["decay"], torch.log1p(v["decay"].exp()))
    r, i = 1 / (1 + (-v["gate_r"]).exp()), 1 / (1 + (-v["gate_i"]).exp())
    a = (-rate * r).exp()
    root = (-(-2 * rate * r).expm1()).sqrt()
    if op == "glr_step":
        y, state = torch.zeros_like(v["x"]), v["state"].clone()
        for k, slot in enumerate(case_slots := v["slots"].tolist()):
            if case_slots[k] >= 0:
                state[slot] = y[k] = a[k] * state[slot] + root[k] * i[k] * v["x"][k]
        return {"y": y, "state": state}

    # token by token; a packed batch is one row of documents, time runs along dim 0
    packed = case["packed"]
    turn = (lambda t: t) if packed else (lambda t: t.transpose(0, 1))
    at, bt = turn(a), turn(root * i * v["x"])
    L = case["L"]
    starts, ends = {}, {}
    if packed:
        off = v["offsets"].tolist()
        for k in range(case["batch"]):
            if off[k + 1] > off[k]:
                starts[off[k]], ends[off[k + 1] - 1] = k, k
    before, hs = torch.empty_like(at), torch.empty_like(at)
    h, h_last = v["h0"], v["h0"].clone()
    for t in range(L):
        if t in starts:
            h = v["h0"][starts[t]]
        before[t] = h
        h = torch.addcmul(bt[t], at[t], h, out=hs[t])
        if t in ends:
            h_last[ends[t]] = h
    if not packed:
        h_last = h
    out = {"y": turn(hs), "h_last": h_last}
    if op == "glr_fwd":
        return out
    dyt, G = turn(v["dy"]), torch.empty_like(at)
    g, dh0 = v["dh_last"], v["dh_last"].clone()
    for t in range(L - 1, -1, -1):
        if t in ends:
            g = v["dh_last"][ends[t]]
        torch.add(dyt[t], g, out=G[t])
        g = at[t] * G[t]
        if t in starts:
            dh0[starts[t]] = g
    G, before = turn(G), turn(before)
    dr = G * (i * v["x"] * a * a / root - a * before) * rate
    dims = (0,) if packed else (0, 1)
    out.update(dh0=dh0 if packed else g, dx=G * root * i, dgate_r=dr * r * (1 - r), dgate_i=G * root * v["x"] * i * (1 - i),
               ddecay=(dr / rate * r).sum(dims) * SCALE / (1 + (-v["decay"]).exp()))
    return out
