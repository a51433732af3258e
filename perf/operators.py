"""The operators of a language model's training step, as they are measured: each in its plain form (elementary torch operations)
and as the calls that a program makes of this library.

The model they belong to is a recurrent one: token embedding, blocks of RMS norm with the residual's addition, Linear layers with
bias, activation and residual in the product's epilogue, a gated linear recurrence along the sequence, and the clipping of all
gradients by their global norm in front of the optimizer.  All tensors are f32 or f64 as everywhere in the library, token ids are
int64.
"""
import math

import numpy as np
import torch

own = False

_EPS = 1e-6
_ACTS = ("none", "relu", "gelu", "silu")
_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        from ferrox_amd import capi
        _ctx = capi.Context(0)
    return _ctx


def _dev(t):
    """A tensor in the form the library's calls take: its device pointer with a shape (non-owning)."""
    from ferrox_amd import capi
    return capi.DeviceArray(_context(), tuple(t.shape), {torch.float32: np.float32, torch.float64: np.float64, torch.int64: np.int64}[t.dtype],
                            t.data_ptr(), 0, None)


# ---- the cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the input layer of a training step: 32 sequences of 512 tokens, 2 % of them padding (-1), a vocabulary of 32000
        {"name": "embed_fwd_f32", "op": "embed", "back": False, "dtype": "f32", "n": 16384, "vocab": 32000, "dim": 1024},
        # its dense weight gradient; token frequencies fall like 1 / rank, so a few rows collect thousands of tokens
        {"name": "embed_bwd_f32", "op": "embed", "back": True, "dtype": "f32", "n": 16384, "vocab": 32000, "dim": 1024},
        # the norm in front of a block, with the residual stream's update; f64 at a width that fills no whole vector of threads
        {"name": "rmsnorm_fwd_f64", "op": "rmsnorm", "back": False, "dtype": "f64", "rows": 4099, "dim": 1001, "res": True},
        # its backward pass with the gradient that arrives along the residual stream
        {"name": "rmsnorm_bwd_f32", "op": "rmsnorm", "back": True, "dtype": "f32", "rows": 16384, "dim": 1024, "res": True},
        # the 784 x 256 layer of a small classifier at batch 256, where the launch is what costs
        {"name": "linear_fwd_small_f32", "op": "linear", "back": False, "dtype": "f32", "batch": 256, "in": 784, "out": 256, "act": "gelu",
         "bias": True, "res": False, "pre": True},
        # the projection back onto the residual stream: a deep product with the residual in its epilogue
        {"name": "linear_fwd_res_f32", "op": "linear", "back": False, "dtype": "f32", "batch": 4096, "in": 4096, "out": 1024, "act": "none",
         "bias": True, "res": True, "pre": False},
        # the backward pass of the widening layer in front of it
        {"name": "linear_bwd_f32", "op": "linear", "back": True, "dtype": "f32", "batch": 4096, "in": 1024, "out": 4096, "act": "gelu",
         "bias": True, "res": False, "pre": True},
        # one token of each of 64 streams: the recurrence as a program that generates runs it
        {"name": "recurrence_step_f32", "op": "recurrence", "back": False, "dtype": "f32", "batch": 64, "steps": 1, "dim": 1024, "h0": True},
        # two long sequences: few channels, many steps
        {"name": "recurrence_fwd_long_f32", "op": "recurrence", "back": False, "dtype": "f32", "batch": 2, "steps": 8192, "dim": 1024, "h0": False},
        # an ordinary training batch backwards, f64, at an odd length
        {"name": "recurrence_bwd_f64", "op": "recurrence", "back": True, "dtype": "f64", "batch": 16, "steps": 511, "dim": 1000, "h0": True},
        # the eleven gradients of a small model, where the launches are what costs
        {"name": "clip_small_f32", "op": "clip", "dtype": "f32", "layers": 2, "dim": 64, "vocab": 1001, "clipped": True},
        # the 61 gradients of a model of 133 million parameters
        {"name": "clip_large_f32", "op": "clip", "dtype": "f32", "layers": 12, "dim": 1024, "vocab": 32000, "clipped": True},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi):
    """A feature width: half of them multiples of 8, the others as they come."""
    w = _log(rng, lo, hi)
    return max(lo, min(hi, (w + 7) // 8 * 8)) if rng.random() < 0.5 else w


def draw(rng):
    op = rng.choice(("embed", "rmsnorm", "linear", "recurrence", "clip"))
    dtype = rng.choice(("f32", "f32", "f64"))
    most = 1 << (24 if dtype == "f32" else 23)
    if op == "embed":
        dim = _width(rng, 8, 2048)
        return {"op": op, "back": rng.random() < 0.5, "dtype": dtype, "n": _log(rng, 1, min(32768, most // dim)),
                "vocab": _log(rng, 16, min(65536, 2 * most // dim)), "dim": dim}
    if op == "rmsnorm":
        dim = _width(rng, 8, 8192)
        return {"op": op, "back": rng.random() < 0.5, "dtype": dtype, "rows": _log(rng, 1, most // dim), "dim": dim, "res": rng.random() < 0.7}
    if op == "linear":
        back = rng.random() < 0.5
        act = rng.choice(_ACTS)
        inn, out = _width(rng, 32, 4096), _width(rng, 32, 4096)
        batch = _log(rng, 1, 4096)
        while batch * inn * out > (1 << (33 if dtype == "f32" else 32)):  # keeps a drawn product below the largest listed one
            batch = (batch + 1) // 2
        return {"op": op, "back": back, "dtype": dtype, "batch": batch, "in": inn, "out": out, "act": act, "bias": rng.random() < 0.8,
                "res": (not back) and rng.random() < 0.5, "pre": back or rng.random() < 0.5}
    if op == "recurrence":
        dim = _width(rng, 8, 2048)
        steps = _log(rng, 1, 8192)
        return {"op": op, "back": rng.random() < 0.5, "dtype": dtype, "batch": _log(rng, 1, max(1, min(256, most // (dim * steps)))),
                "steps": steps, "dim": dim, "h0": rng.random() < 0.5}
    return {"op": op, "dtype": dtype, "layers": rng.randint(1, 12), "dim": _width(rng, 16, 768), "vocab": _log(rng, 16, 32000),
            "clipped": rng.random() < 0.7}


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def _clip_shapes(case):
    d = case["dim"]
    shapes = [(case["vocab"], d)]
    for _ in range(case["layers"]):
        shapes += [(d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)]
    return shapes


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = torch.float32 if case["dtype"] == "f32" else torch.float64

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=gen, device=dev, dtype=dt) * std + mean

    def empty(*shape):
        return torch.empty(shape, device=dev, dtype=dt)

    s = {"case": case}
    op = case["op"]
    if op == "embed":
        n, vocab, dim = case["n"], case["vocab"], case["dim"]
        u = torch.rand((n,), generator=gen, device=dev, dtype=torch.float64)
        ids = torch.exp(u * math.log(vocab + 1.0)).floor().long() - 1  # P(id) falls like 1 / (id + 1)
        ids = ids.clamp_(0, vocab - 1)
        perm = torch.randperm(vocab, generator=gen, device=dev)
        ids = perm[ids]
        pad = torch.rand((n,), generator=gen, device=dev) < 0.02
        s["ids"] = torch.where(pad, torch.full_like(ids, -1), ids)
        s["scale"] = math.sqrt(dim)
        if case["back"]:
            s["g"], s["out"] = normal(n, dim, std=0.02), [empty(vocab, dim)]
        else:
            s["w"], s["out"] = normal(vocab, dim, std=0.02), [empty(n, dim)]
    elif op == "rmsnorm":
        rows, dim = case["rows"], case["dim"]
        s["w"] = normal(dim, std=0.1, mean=1.0)
        if case["back"]:
            s["h"] = normal(rows, dim, std=2.0)
            s["rstd"] = ((s["h"] * s["h"]).double().mean(1) + _EPS).rsqrt().to(dt)  # saved by the forward pass
            s["dy"] = normal(rows, dim)
            s["dh"] = normal(rows, dim) if case["res"] else None
            s["out"] = [empty(rows, dim), empty(dim)]
        else:
            s["x"] = normal(rows, dim)
            s["res"] = normal(rows, dim, std=2.0) if case["res"] else None
            s["out"] = [empty(rows, dim) if case["res"] else None, empty(rows, dim), empty(rows)]
    elif op == "linear":
        b, i, o = case["batch"], case["in"], case["out"]
        s["x"], s["w"] = normal(b, i), normal(o, i, std=1.0 / math.sqrt(i))
        if case["back"]:
            s["pre"] = normal(b, o)  # saved by the forward pass
            s["dy"] = normal(b, o)
            s["out"] = [empty(b, i), empty(o, i), empty(o) if case["bias"] else None, empty(b, o)]
        else:
            s["bias"] = normal(o, std=0.1) if case["bias"] else None
            s["res"] = normal(b, o, std=2.0) if case["res"] else None
            s["out"] = [empty(b, o), empty(b, o) if case["pre"] else None]
    elif op == "recurrence":
        b, t, d = case["batch"], case["steps"], case["dim"]
        s["z"], s["x"] = normal(b, t, d, std=2.0, mean=2.0), normal(b, t, d)
        s["h0"] = normal(b, d) if case["h0"] else None
        if case["back"]:
            s["h"] = _scan(s["z"], s["x"], s["h0"])  # saved by the forward pass
            s["dh"] = normal(b, t, d)
            s["out"] = [empty(b, t, d), empty(b, t, d), empty(b, d) if case["h0"] else None]
        else:
            s["out"] = [empty(b, t, d)]
    else:
        s["g"] = [normal(*shape, std=0.01) for shape in _clip_shapes(case)]
        count = sum(g.numel() for g in s["g"])
        s["max_norm"] = 0.01 * math.sqrt(count) * (0.5 if case["clipped"] else 2.0)
        s["out"] = [torch.empty_like(g) for g in s["g"]] + [empty(1)]
    if own:  # the same memory as the library's calls take it
        s["dev"] = {k: _dev(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        s["dev_out"] = [None if t is None else _dev(t) for t in s["out"]]
        s["dev_g"] = [_dev(t) for t in s["g"]] if isinstance(s.get("g"), list) else None
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------------
def _act(v, name):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _act_grad(v, name):
    if name == "relu":
        return (v > 0).to(v.dtype)
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "silu":
        f = 1.0 / (1.0 + torch.exp(-v))
        return f * (1.0 + v * (1.0 - f))
    return torch.ones_like(v)


def _linear_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from h_{-1} = 0, by doubling: after step k every element holds 2^k terms."""
    d, steps = 1, a.shape[1]
    while d < steps:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def _scan(z, x, h0):
    f, k = 1.0 / (1.0 + torch.exp(-z)), 1.0 / (1.0 + torch.exp(z))
    b = k * x
    if h0 is not None:
        b[:, 0] += f[:, 0] * h0
    return _linear_scan(f, b)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "embed":
        ids = s["ids"]
        live = ((ids >= 0) & (ids < case["vocab"])).to(torch.float32 if case["dtype"] == "f32" else torch.float64)
        at = ids.clamp(0, case["vocab"] - 1)
        if case["back"]:
            dw = torch.zeros((case["vocab"], case["dim"]), device=ids.device, dtype=s["g"].dtype)
            return [dw.index_add_(0, at, s["g"] * (live * s["scale"])[:, None])]
        return [s["w"][at] * (live * s["scale"])[:, None]]
    if op == "rmsnorm":
        if case["back"]:
            h, rstd, dy, w = s["h"], s["rstd"][:, None], s["dy"], s["w"]
            wdy = dy * w
            dx = rstd * (wdy - h * (rstd * rstd * (wdy * h).mean(1, keepdim=True)))
            if s["dh"] is not None:
                dx = dx + s["dh"]
            return [dx, (dy * (h * rstd)).sum(0)]
        h = s["x"] if s["res"] is None else s["x"] + s["res"]
        rstd = 1.0 / torch.sqrt((h * h).mean(1) + _EPS)
        return [None if s["res"] is None else h, h * rstd[:, None] * s["w"], rstd]
    if op == "linear":
        if case["back"]:
            dpre = s["dy"] * _act_grad(s["pre"], case["act"])
            return [dpre @ s["w"], dpre.t() @ s["x"], dpre.sum(0) if case["bias"] else None, dpre]
        pre = s["x"] @ s["w"].t()
        if s["bias"] is not None:
            pre = pre + s["bias"]
        y = _act(pre, case["act"])
        if s["res"] is not None:
            y = y + s["res"]
        return [y, pre if case["pre"] else None]
    if op == "recurrence":
        if not case["back"]:
            return [_scan(s["z"], s["x"], s["h0"])]
        f, k = 1.0 / (1.0 + torch.exp(-s["z"])), 1.0 / (1.0 + torch.exp(s["z"]))
        # D_t = dh_t + f_{t+1} D_{t+1}: the same recurrence from the other end, with the gates one step on
        nxt = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], 1)
        total = _linear_scan(nxt.flip(1), s["dh"].flip(1)).flip(1)
        first = s["h0"] if s["h0"] is not None else torch.zeros_like(s["x"][:, 0])
        before = torch.cat([first[:, None], s["h"][:, :-1]], 1)
        return [total * (before - s["x"]) * (f * k), total * k, f[:, 0] * total[:, 0] if case["h0"] else None]
    norm = torch.sqrt(torch.stack([(g * g).sum(dtype=torch.float64) for g in s["g"]]).sum())
    coef = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).to(s["g"][0].dtype)
    return [g * coef for g in s["g"]] + [norm.to(s["g"][0].dtype).reshape(1)]


# ---- the library's calls ---------------------------------------------------------------------------------------------------
def _calls(s):
    case, d, out = s["case"], s["dev"], s["dev_out"]
    ctx, op = _ctx, s["case"]["op"]
    if op == "embed":
        if case["back"]:
            ctx.embedding_bwd(d["g"], d["ids"], case["vocab"], s["scale"], out=out[0])
        else:
            ctx.embedding_fwd(d["w"], d["ids"], s["scale"], out=out[0])
    elif op == "rmsnorm":
        if case["back"]:
            ctx.rmsnorm_bwd(d["dy"], d["h"], d["w"], d["rstd"], dh=d.get("dh"), out=out)
        else:
            ctx.rmsnorm_fwd(d["x"], d["w"], _EPS, res=d.get("res"), out=out)
    elif op == "linear":
        if case["back"]:
            ctx.linear_act_bwd(d["dy"], d["w"], d["x"], d["pre"], case["act"], want_db=case["bias"], out=out)
        else:
            ctx.gemm_bias_act_residual(d["x"], d["w"], tb=True, bias=d.get("bias"), act=case["act"], residual=d.get("res"), pre=out[1], out=out[0])
    elif op == "recurrence":
        if case["back"]:
            ctx.gated_recurrence_bwd(d["dh"], d["z"], d["x"], d["h"], h0=d.get("h0"), out=out)
        else:
            ctx.gated_recurrence_fwd(d["z"], d["x"], h0=d.get("h0"), out=out[0])
    else:
        ctx.clip_grad_norm(s["dev_g"], s["max_norm"], outs=out[:-1], norm=out[-1])
    return s["out"]


def run(state):
    return _calls(state) if own else _plain(state)


def work(case):
    e = 4 if case["dtype"] == "f32" else 8
    op = case["op"]
    if op == "embed":
        n, v, d = case["n"], case["vocab"], case["dim"]
        p = np.diff(np.log(np.arange(1, v + 2))) / math.log(v + 1.0)
        rows = float((1.0 - (1.0 - p) ** (0.98 * n)).sum())  # distinct tokens to be expected: the rows of the table that have to be read
        return {"bytes": (n * d + v * d if case["back"] else rows * d + n * d) * e + 8 * n, "flops": n * d}
    if op == "rmsnorm":
        n, d = case["rows"], case["dim"]
        if case["back"]:
            return {"bytes": ((4 if case["res"] else 3) * n * d + n + 2 * d) * e, "flops": 9 * n * d}
        return {"bytes": ((4 if case["res"] else 2) * n * d + n + d) * e, "flops": 5 * n * d}
    if op == "linear":
        b, i, o = case["batch"], case["in"], case["out"]
        if case["back"]:  # x, w, dy, pre read; dx, dw, db, dpre written
            return {"bytes": (2 * b * i + 2 * i * o + 3 * b * o + (o if case["bias"] else 0)) * e, "flops": 4 * b * i * o}
        extra = (1 if case["res"] else 0) + (1 if case["pre"] else 0)
        return {"bytes": (b * i + i * o + (1 + extra) * b * o + (o if case["bias"] else 0)) * e, "flops": 2 * b * i * o}
    if op == "recurrence":
        n, b = case["batch"] * case["steps"] * case["dim"], case["batch"] * case["dim"]
        ends = (b * (2 if case["back"] else 1)) if case["h0"] else 0
        return {"bytes": ((6 if case["back"] else 3) * n + ends) * e, "flops": (20 if case["back"] else 10) * n}
    n = sum(int(np.prod(shape)) for shape in _clip_shapes(case))
    return {"bytes": 2 * n * e, "flops": 3 * n}


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    up = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.dtype.is_floating_point}
    op = case["op"]
    if op == "embed":
        ids = s["ids"].cpu().numpy()
        live = np.flatnonzero((ids >= 0) & (ids < case["vocab"]))
        if case["back"]:
            dw = np.zeros((case["vocab"], case["dim"]))
            if live.size:
                order = live[np.argsort(ids[live], kind="stable")]
                keys = ids[order]
                starts = np.flatnonzero(np.concatenate([[True], keys[1:] != keys[:-1]]))
                dw[keys[starts]] = np.add.reduceat(up["g"].cpu().numpy()[order], starts, axis=0) * s["scale"]
            return [dw]
        w = up["w"].cpu().numpy()
        out = np.zeros((case["n"], case["dim"]))
        out[live] = w[ids[live]] * s["scale"]
        return [out]
    if op == "rmsnorm":
        if case["back"]:
            # of y_j = w_j h_j r, r = (mean h^2 + eps)^(-1/2) as the forward pass saved it: dL/dh_j = w_j dy_j r - h_j r^3 sum_k(w_k dy_k h_k) / dim
            h, r, dy = up["h"], up["rstd"].unsqueeze(1), up["dy"]
            g = torch.einsum("nd,d->nd", dy, up["w"])
            dx = g * r - h * r.pow(3) * torch.einsum("nd,nd->n", g, h).unsqueeze(1) / case["dim"]
            if s["dh"] is not None:
                dx = dx + up["dh"]
            return [dx, torch.einsum("nd,nd->d", dy, h * r)]
        # the sum with the residual is stored in the tensors' own type; the norm is taken of what is stored
        h = up["x"] if s["res"] is None else (s["x"] + s["res"]).double()
        r = (h.pow(2).sum(1) / case["dim"] + _EPS).pow(-0.5)
        return [None if s["res"] is None else up["x"] + up["res"], torch.einsum("nd,n,d->nd", h, r, up["w"]), r]
    if op == "linear":
        act = case["act"]
        if case["back"]:
            p = up["pre"].clone().requires_grad_(True)
            y = {"none": lambda v: v, "relu": torch.relu, "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2.0)),
                 "silu": lambda v: v * torch.sigmoid(v)}[act](p)
            (dpre,) = torch.autograd.grad(y, p, up["dy"])
            dpre = dpre.detach()
            return [dpre.mm(up["w"]), dpre.t().contiguous().mm(up["x"]), dpre.sum(0) if case["bias"] else None, dpre]
        pre = torch.mm(up["x"], up["w"].t().contiguous())
        if s["bias"] is not None:
            pre = pre + up["bias"]
        y = {"none": lambda v: v, "relu": torch.relu, "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2.0)),
             "silu": lambda v: v * torch.sigmoid(v)}[act](pre)
        if s["res"] is not None:
            y = y + up["res"]
        return [y, pre if case["pre"] else None]
    if op == "recurrence":
        f, k = torch.sigmoid(up["z"]), torch.sigmoid(-up["z"])
        steps = case["steps"]
        if not case["back"]:
            state = up["h0"] if case["h0"] else torch.zeros_like(up["x"][:, 0])
            h = torch.empty_like(up["x"])
            for t in range(steps):
                state = f[:, t] * state + k[:, t] * up["x"][:, t]
                h[:, t] = state
            return [h]
        carry = torch.zeros_like(up["x"][:, 0])
        dz, dx = torch.empty_like(up["x"]), torch.empty_like(up["x"])
        for t in reversed(range(steps)):
            carry = carry + up["dh"][:, t]
            before = up["h"][:, t - 1] if t else (up["h0"] if case["h0"] else torch.zeros_like(carry))
            dz[:, t] = carry * (before - up["x"][:, t]) * f[:, t] * k[:, t]
            dx[:, t] = carry * k[:, t]
            carry = carry * f[:, t]
        return [dz, dx, carry if case["h0"] else None]
    norm = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in s["g"]))
    coef = min(1.0, s["max_norm"] / norm) if norm > 0 else 1.0
    return [g.double() * coef for g in s["g"]] + [torch.tensor([norm], dtype=torch.float64)]
