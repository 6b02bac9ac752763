"""Cases of the sequence-layer operators: the gated linear recurrence, the
group norm with an activation (channels last) and the AdamW step, each with its
plain form in elementary torch operations and its definition in 64 bits.

``own`` false: the plain forms.  ``own`` true: the calls of ``pacho_b200``.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f64": torch.float64}
_BETAS, _EPS_ADAM, _DECAY, _RATE, _STEP = (0.9, 0.95), 1e-8, 0.1, 3e-4, 1000
_EPS_NORM = 1e-5
_backend = None


def _device():
    """The backend that every state of this process shares (a user's program
    keeps one per GPU)."""
    global _backend
    if _backend is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "open-pacho_b200"))
        from pacho_b200 import B200Backend

        _backend = B200Backend(0)
    return _backend


def listed():
    return [
        # One new token for each of 32 streams being served: the state is updated in place.
        dict(name="recurrence_token", op="recurrence", batch=32, steps=1, width=2048, dtype="f32",
             gate="sigmoid", step=True),
        # A long prompt of one user, an odd number of tokens, read into the state.
        dict(name="recurrence_prompt", op="recurrence", batch=1, steps=16381, width=1024, dtype="f32",
             gate="linear", step=False),
        # The forward pass of a training step.
        dict(name="recurrence_train", op="recurrence", batch=8, steps=4096, width=2048, dtype="f32",
             gate="sigmoid", step=False),
        # The backward pass of the same training step.
        dict(name="recurrence_train_grad", op="recurrence_grad", batch=8, steps=4096, width=2048,
             dtype="f32", gate="sigmoid", final=False),
        # Gradients in float64 (a numerical study of a small model, ragged sizes, gradient of the final state).
        dict(name="recurrence_f64_grad", op="recurrence_grad", batch=3, steps=1000, width=515, dtype="f64",
             gate="linear", final=True),
        # Per-head normalisation of one token for each of 32 streams.
        dict(name="norm_token", op="norm", n=32, s=1, channels=2048, groups=16, dtype="f32", act="silu",
             affine=True),
        # A feature map inside an image model.
        dict(name="norm_image", op="norm", n=8, s=4096, channels=320, groups=32, dtype="f32", act="silu",
             affine=True),
        # Per-head normalisation of every token of a training batch, backward.
        dict(name="norm_tokens_grad", op="norm_grad", n=16384, s=1, channels=2048, groups=16, dtype="f32",
             act="silu", affine=True),
        # A decoder's full-resolution feature map, backward.
        dict(name="norm_image_grad", op="norm_grad", n=4, s=65536, channels=128, groups=32, dtype="f32",
             act="silu", affine=True),
        # Gradients in float64 at ragged sizes.
        dict(name="norm_f64_grad", op="norm_grad", n=3, s=37 * 41, channels=90, groups=9, dtype="f64",
             act="gelu", affine=True),
        # The parameters of one small layer.
        dict(name="adamw_layer", op="adamw", tensors=11, total=1 << 20, dtype="f32", scaled=True),
        # A whole model's parameters: large matrices, and many short vectors.
        dict(name="adamw_model", op="adamw", tensors=146, total=100_000_000, dtype="f32", scaled=True),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """Sizes, types and options of the same ranges as the listed cases'."""
    op = rng.choice(["recurrence", "recurrence_grad", "norm", "norm_grad", "adamw"])
    dtype = rng.choice(["f32", "f32", "f64"])
    most = 1 << (26 if dtype == "f32" else 25)
    if op.startswith("recurrence"):
        width = _log_uniform(rng, 8, 4096)
        batch = _log_uniform(rng, 1, 32)
        steps = _log_uniform(rng, 1, min(16384, max(1, most // (width * batch))))
        case = dict(op=op, batch=batch, steps=steps, width=width, dtype=dtype,
                    gate=rng.choice(["linear", "sigmoid"]))
        case["step" if op == "recurrence" else "final"] = rng.random() < 0.5
        return case
    if op.startswith("norm"):
        most >>= 1
        groups = _log_uniform(rng, 1, 64)
        act = rng.choice(["none", "relu", "silu", "gelu"])
        if rng.random() < 0.5:  # each token by itself: groups of at least 8 values
            channels = groups * _log_uniform(rng, 8, 256)
            n, s = _log_uniform(rng, 1, min(32768, max(1, most // channels))), 1
        else:
            channels = groups * _log_uniform(rng, 1, 64)
            n = _log_uniform(rng, 1, 16)
            s = _log_uniform(rng, 16, min(65536, max(16, most // (n * channels))))
        return dict(op=op, n=n, s=s, channels=channels, groups=groups, dtype=dtype, act=act,
                    affine=rng.random() < 0.75)
    return dict(op=op, tensors=_log_uniform(rng, 1, 300), total=_log_uniform(rng, 1000, 50_000_000), dtype=dtype,
                scaled=rng.random() < 0.5)


def _offsets(case):
    """(offset, length) of each tensor in the flat parameter buffer: one length
    in four is a matrix's, the others vectors'; each starts on 16 bytes."""
    count, total = case["tensors"], case["total"]
    weights = [1.0 if i % 4 == 0 else 1e-4 * (1 + i % 7) for i in range(count)]
    scale = total / sum(weights)
    spans, at = [], 0
    for w in weights:
        n = max(1, int(w * scale))
        spans.append((at, n))
        at += -(-n // 4) * 4
    return spans, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=t)

    s = {"case": case}
    if case["op"].startswith("recurrence"):
        shape = (case["batch"], case["steps"], case["width"])
        gate = normal(*shape).add_(2.0)  # logits: decays around 0.88
        s["a"] = gate if case["gate"] == "sigmoid" else torch.sigmoid(gate)
        s["b"] = normal(*shape)
        s["state"] = normal(shape[0], shape[2])
        if case["op"] == "recurrence":
            s["h"] = torch.empty_like(s["b"])
            s["final"] = s["state"] if case["step"] else torch.empty_like(s["state"])
        else:
            s["h"] = _recurrence(s["a"], s["b"], s["state"], case["gate"])
            s["dh"] = normal(*shape)
            s["dfinal"] = normal(shape[0], shape[2]) if case["final"] else None
            s["da"], s["db"], s["dstate"] = (torch.empty_like(s[k]) for k in ("a", "b", "state"))
    elif case["op"].startswith("norm"):
        n, sp, c = case["n"], case["s"], case["channels"]
        s["x"] = normal(n, sp, c).mul_(1.5).add_(0.3)
        s["weight"] = normal(c).mul_(0.2).add_(1.0) if case["affine"] else None
        s["bias"] = normal(c).mul_(0.2) if case["affine"] else None
        if case["op"] == "norm":
            s["y"] = torch.empty_like(s["x"])
            s["mean"], s["rstd"] = (torch.empty(n, case["groups"], device="cuda", dtype=t) for _ in range(2))
        else:
            s["mean"], s["rstd"] = _statistics(s["x"], case["groups"])
            s["dy"] = normal(n, sp, c)
            s["dx"] = torch.empty_like(s["x"])
            if case["affine"]:
                s["dweight"], s["dbias"] = torch.empty_like(s["weight"]), torch.empty_like(s["bias"])
    else:
        spans, size = _offsets(case)
        live = torch.zeros(size, device="cuda", dtype=t)
        for at, n in spans:
            live[at:at + n] = 1
        s["p"] = normal(size).mul_(0.02).mul_(live)
        s["g"] = normal(size).mul_(0.01).mul_(live)
        s["m"] = normal(size).mul_(0.002).mul_(live)
        s["v"] = normal(size).square_().mul_(1e-4).mul_(live)
        s["scale"] = torch.rand(1, generator=gen, device="cuda", dtype=t) if case["scaled"] else None
    if own:
        # The same tensors as the framework's arrays (no copy), as its user holds them.
        backend = _device()
        if case["op"] == "adamw":
            s["dev"] = {k: [backend.view(s[k][at:at + n]) for at, n in spans] for k in ("p", "g", "m", "v")}
            s["dev"]["scale"] = backend.view(s["scale"]) if case["scaled"] else None
        else:
            s["dev"] = {k: backend.view(x) for k, x in s.items() if isinstance(x, torch.Tensor)}
    return s


# ----------------------------------------------------------- plain forms --


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t from h_{-1} = 0 along axis 1: doubling, log2(steps) passes."""
    k = 1
    while k < a.shape[1]:
        b = torch.cat([b[:, :k], torch.addcmul(b[:, k:], a[:, k:], b[:, :-k])], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _recurrence(a, b, state, gate):
    if gate == "sigmoid":
        a, b = torch.sigmoid(a), torch.sigmoid(-a) * b
    b = torch.cat([torch.addcmul(b[:, :1], a[:, :1], state[:, None]), b[:, 1:]], 1)
    return _scan(a, b)


def _recurrence_grad(s):
    gate = s["case"]["gate"]
    alpha = torch.sigmoid(s["a"]) if gate == "sigmoid" else s["a"]
    dh = s["dh"]
    if s["dfinal"] is not None:
        dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dfinal"][:, None]], 1)
    after = torch.cat([alpha[:, 1:], torch.zeros_like(alpha[:, :1])], 1)
    grad = _scan(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([s["state"][:, None], s["h"][:, :-1]], 1)
    dstate = alpha[:, 0] * grad[:, 0]
    if gate == "linear":
        return grad * before, grad, dstate
    rest = torch.sigmoid(-s["a"])
    return grad * (before - s["b"]) * alpha * rest, grad * rest, dstate


def _statistics(x, groups):
    n, sp, c = x.shape
    x = x.reshape(n, sp, groups, c // groups)
    mean = x.mean((1, 3), dtype=torch.float64)
    var = (x - mean[:, None, :, None]).square().mean((1, 3))
    return mean.to(x.dtype), torch.rsqrt(var + _EPS_NORM).to(x.dtype)


def _activate(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    return torch.clamp(z, min=0) if act == "relu" else z


def _slope(z, act):
    if act == "silu":
        q = torch.sigmoid(z)
        return q * (1 + z * (1 - q))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return (z > 0).to(z.dtype) if act == "relu" else torch.ones_like(z)


def _normalised(s):
    x, groups = s["x"], s["case"]["groups"]
    m = x.shape[2] // groups
    mean, rstd = (s[k].repeat_interleave(m, 1)[:, None] for k in ("mean", "rstd"))
    xhat = (x - mean) * rstd
    return xhat, rstd, xhat * s["weight"] + s["bias"] if s["case"]["affine"] else xhat


def _norm(s):
    mean, rstd = _statistics(s["x"], s["case"]["groups"])
    s = {**s, "mean": mean, "rstd": rstd}
    return _activate(_normalised(s)[2], s["case"]["act"]), mean, rstd


def _norm_grad(s):
    groups = s["case"]["groups"]
    n, sp, c = s["x"].shape
    xhat, rstd, z = _normalised(s)
    dz = s["dy"] * _slope(z, s["case"]["act"])
    wdz = dz * s["weight"] if s["case"]["affine"] else dz

    def average(v):
        v = v.reshape(n, sp, groups, c // groups).mean((1, 3), dtype=torch.float64).to(v.dtype)
        return v.repeat_interleave(c // groups, 1)[:, None]

    dx = rstd * (wdz - average(wdz) - xhat * average(wdz * xhat))
    if not s["case"]["affine"]:
        return (dx,)
    total = [(dz * f).sum((0, 1), dtype=torch.float64).to(dz.dtype) for f in (xhat, 1)]
    return dx, total[0], total[1]


def _adamw(s):
    g = s["g"] * s["scale"] if s["scale"] is not None else s["g"]
    s["m"].mul_(_BETAS[0]).add_(g, alpha=1 - _BETAS[0])
    s["v"].mul_(_BETAS[1]).add_(g * g, alpha=1 - _BETAS[1])
    root = torch.sqrt(s["v"] / (1 - _BETAS[1] ** _STEP)) + _EPS_ADAM
    s["p"].mul_(1 - _RATE * _DECAY).sub_(s["m"] / root, alpha=_RATE / (1 - _BETAS[0] ** _STEP))
    return s["p"], s["m"], s["v"]


def run(s):
    case = s["case"]
    if own:
        return _run_own(s)
    if case["op"] == "recurrence":
        h = _recurrence(s["a"], s["b"], s["state"], case["gate"])
        if case["step"]:
            s["state"].copy_(h[:, -1])
        return {"h": h, "final": s["state"] if case["step"] else h[:, -1].clone()}
    if case["op"] == "recurrence_grad":
        return dict(zip(("da", "db", "dstate"), _recurrence_grad(s)))
    if case["op"] == "norm":
        return dict(zip(("y", "mean", "rstd"), _norm(s)))
    if case["op"] == "norm_grad":
        return dict(zip(("dx", "dweight", "dbias"), _norm_grad(s)))
    return dict(zip(("p", "m", "v"), _adamw(s)))


def _run_own(s):
    import pacho_b200 as pb

    case, d = s["case"], s["dev"]
    act = None if case.get("act") == "none" else case.get("act")
    if case["op"] == "recurrence":
        pb.linear_recurrence(d["a"], d["b"], state=d["state"], gate=case["gate"], out=d["h"], final=d["final"])
        return {"h": s["h"], "final": s["final"]}
    if case["op"] == "recurrence_grad":
        pb.linear_recurrence_backward(d["a"], d["b"], d["h"], d["dh"], state=d["state"], dfinal=d.get("dfinal"),
                                      gate=case["gate"], out=(d["da"], d["db"], d["dstate"]))
        return {k: s[k] for k in ("da", "db", "dstate")}
    if case["op"] == "norm":
        pb.group_norm(d["x"], case["groups"], d.get("weight"), d.get("bias"), eps=_EPS_NORM, activation=act,
                      out=(d["y"], d["mean"], d["rstd"]))
        return {k: s[k] for k in ("y", "mean", "rstd")}
    if case["op"] == "norm_grad":
        pb.group_norm_backward(d["dy"], d["x"], case["groups"], d["mean"], d["rstd"], d.get("weight"),
                               d.get("bias"), activation=act, out=(d["dx"], d.get("dweight"), d.get("dbias")))
        return {k: s[k] for k in (("dx", "dweight", "dbias") if case["affine"] else ("dx",))}
    pb.adamw_step(d["p"], d["g"], d["m"], d["v"], step=_STEP, lr=_RATE, betas=_BETAS, eps=_EPS_ADAM,
                  weight_decay=_DECAY, grad_scale=d["scale"])
    return {k: s[k] for k in ("p", "m", "v")}


# ------------------------------------------------------------------ work --


def work(case):
    item = 4 if case["dtype"] == "f32" else 8
    if case["op"].startswith("recurrence"):
        n, states = case["batch"] * case["steps"] * case["width"], case["batch"] * case["width"]
        if case["op"] == "recurrence":
            return {"bytes": item * (3 * n + 2 * states), "flops": (2 if case["gate"] == "linear" else 6) * n}
        streams, flops = (5, 3) if case["gate"] == "linear" else (6, 10)
        return {"bytes": item * (streams * n + (3 if case["final"] else 2) * states), "flops": flops * n}
    if case["op"].startswith("norm"):
        n = case["n"] * case["s"] * case["channels"]
        stats, affine = 2 * case["n"] * case["groups"], case["channels"] if case["affine"] else 0
        if case["op"] == "norm":
            return {"bytes": item * (2 * n + stats + 2 * affine), "flops": 10 * n}
        return {"bytes": item * (3 * n + stats + 4 * affine), "flops": 25 * n}
    n = sum(length for _, length in _offsets(case)[0])
    return {"bytes": item * 7 * n, "flops": 12 * n}


# ------------------------------------------- the definitions, in 64 bits --


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    d = {k: x.double() for k, x in s.items() if isinstance(x, torch.Tensor)}
    if case["op"] == "recurrence":
        return _exact_recurrence(case, d)
    if case["op"] == "recurrence_grad":
        return _exact_recurrence_grad(case, d)
    if case["op"].startswith("norm"):
        return _exact_norm(case, d)
    g = d["g"] * d["scale"] if case["scaled"] else d["g"]
    m = _BETAS[0] * d["m"] + (1 - _BETAS[0]) * g
    v = _BETAS[1] * d["v"] + (1 - _BETAS[1]) * g ** 2
    fixed = [1 - np.float64(b) ** _STEP for b in _BETAS]
    p = d["p"] - _RATE * (_DECAY * d["p"] + (m / float(fixed[0])) / ((v / float(fixed[1])) ** 0.5 + _EPS_ADAM))
    return {"p": p, "m": m, "v": v}


def _exact_recurrence(case, d):
    """Step by step."""
    alpha, put = d["a"], d["b"]
    if case["gate"] == "sigmoid":
        alpha = 1 / (1 + torch.exp(-d["a"]))
        put = d["b"] / (1 + torch.exp(d["a"]))
    h, now = torch.empty_like(put), d["state"]
    for t in range(case["steps"]):
        now = alpha[:, t] * now + put[:, t]
        h[:, t] = now
    return {"h": h, "final": now}


def _exact_recurrence_grad(case, d):
    """The chain rule, step by step from the last one back, with the h that was given."""
    da, db = torch.empty_like(d["a"]), torch.empty_like(d["b"])
    back = d["dfinal"] if case["final"] else torch.zeros_like(d["state"])
    for t in reversed(range(case["steps"])):
        grad = d["dh"][:, t] + back
        last = d["h"][:, t - 1] if t else d["state"]
        if case["gate"] == "linear":
            da[:, t], db[:, t], back = grad * last, grad, grad * d["a"][:, t]
        else:
            e = torch.exp(-d["a"][:, t])
            keep = 1 / (1 + e)
            da[:, t] = grad * (last - d["b"][:, t]) * keep * (e * keep)
            db[:, t], back = grad * (e * keep), grad * keep
    return {"da": da, "db": db, "dstate": back}


def _exact_norm(case, d):
    """The definition, and its derivatives by torch's differentiation."""
    n, sp, c, groups = case["n"], case["s"], case["channels"], case["groups"]
    x = d["x"].requires_grad_(case["op"] == "norm_grad")
    parts = x.reshape(n, sp, groups, -1)
    mean = parts.mean((1, 3), keepdim=True)
    var = ((parts - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((parts - mean) / torch.sqrt(var + _EPS_NORM)).reshape(n, sp, c)
    if case["affine"]:
        w, b = (d[k].requires_grad_(case["op"] == "norm_grad") for k in ("weight", "bias"))
        z = z * w + b
    y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)),
         "silu": lambda: z / (1 + torch.exp(-z)),
         "gelu": lambda: z * torch.special.ndtr(z)}[case["act"]]()
    if case["op"] == "norm":
        return {"y": y, "mean": mean.reshape(n, groups), "rstd": ((var + _EPS_NORM) ** -0.5).reshape(n, groups)}
    wanted = [x, w, b] if case["affine"] else [x]
    return dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, wanted, d["dy"])))
