"""Measured operators of a transformer block in training and serving: expert
routing with its balance loss and counts, the norms before and after a block
fused with its gate and residual scale, and the gated activation and linear
layer whose inputs wait for the backward pass in 8 bits; through the framework's
public entry points (``own``) and in plain torch operations.
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-torchtpu_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

DEV = "cuda"
BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
EPS = 1e-6


def listed():
    return [
        # expert counts and balance of a decode batch of 8, as a server watches them: latency
        dict(name="balance_watch_8", op="balance", T=8, E=128, k=4, logits="bf16", route="softmax", pad=0, train=False),
        # a short fine-tuning batch (odd count) with padding: routing, loss, counts and the logits' gradient
        dict(name="balance_train_777", op="balance", T=777, E=128, k=4, logits="bf16", route="softmax", pad=100,
             train=True),
        # a training batch, grouped sigmoid routing with a correction bias
        dict(name="balance_train_16384", op="balance", T=16384, E=256, k=8, logits="f32", route="grouped", pad=0,
             train=True),
        # a decode step of one token between two blocks: residual added, next norm
        dict(name="residual_serve_1", op="residual", T=1, H=7168, res="bf16", post=False, gate="none", next=True,
             train=False),
        # a prompt: post-norm, a gate per channel, residual, next norm
        dict(name="residual_serve_1024", op="residual", T=1024, H=4096, res="bf16", post=True, gate="channel",
             next=True, train=False),
        # a short training batch with a float32 residual stream, a gate per token
        dict(name="residual_train_777", op="residual", T=777, H=2880, res="f32", post=True, gate="token", next=True,
             train=True),
        # a training batch: post-norm, gate per channel, residual, next norm, all gradients
        dict(name="residual_train_8192", op="residual", T=8192, H=7168, res="bf16", post=True, gate="channel",
             next=True, train=True),
        # a short training batch through the activation of biased experts (odd count)
        dict(name="act_train_777", op="act", T=777, I=2880, act="swigluoai"),
        # a training batch through a wide gated MLP
        dict(name="act_train_8192", op="act", T=8192, I=14336, act="silu"),
        # a handful of tokens through a down projection: one read of the weights per product
        dict(name="linear_train_19", op="linear", T=19, K=2880, N=2880, bias=True),
        # a fine-tuning batch (odd count) through an attention block's output projection
        dict(name="linear_train_777", op="linear", T=777, K=4096, N=4096, bias=False),
        # a training batch through a wide MLP's gate and up projection
        dict(name="linear_train_4096", op="linear", T=4096, K=4096, N=28672, bias=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(["balance", "balance", "residual", "residual", "act", "linear", "linear"])
    if op == "balance":
        route = rng.choice(["softmax", "sigmoid", "grouped"])
        E, k = rng.choice([16, 32, 60, 64, 128, 256, 384]), rng.choice([1, 2, 4, 6, 8])
        T = _log_int(rng, 1, 16384)
        return dict(op=op, T=T, E=64 if route == "grouped" and E == 60 else E, k=k, logits=rng.choice(["bf16", "f32"]),
                    route=route, pad=rng.choice([0, rng.randint(0, T // 2)]), train=rng.random() < 0.7)
    if op == "residual":
        return dict(op=op, T=_log_int(rng, 1, 8192), H=8 * _log_int(rng, 16, 896), res=rng.choice(["bf16", "f32"]),
                    post=rng.random() < 0.7, gate=rng.choice(["none", "channel", "token", "full"]),
                    next=rng.random() < 0.8, train=rng.random() < 0.7)
    if op == "act":
        return dict(op=op, T=_log_int(rng, 1, 8192), I=8 * _log_int(rng, 16, 1792),
                    act=rng.choice(["silu", "swigluoai", "gelu"]))
    K, N = 32 * _log_int(rng, 8, 448), 8 * _log_int(rng, 32, 3584)
    return dict(op=op, T=_log_int(rng, 1, min(8192, 4096 * 4096 * 28672 // (K * N))), K=K, N=N, bias=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(shape, g, std=1.0, dtype=BF16, mean=0.0):
    return torch.empty(shape, device=DEV, dtype=dtype).normal_(mean, std, generator=g)


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    T = case["T"]
    if case["op"] == "balance":
        E, k = case["E"], case["k"]
        grouped = case["route"] == "grouped"
        # some experts are more wanted than others
        st["logits"] = (_normal((T, E), g, 1.0, F32) + _normal((E,), g, 0.5, F32)).to(_TYPES[case["logits"]])
        st["correction"] = _normal((E,), g, 0.1, F32) if grouped else None
        st["mask"] = torch.arange(T, device=DEV) < T - case["pad"] if case["pad"] else None
        st["routing"] = dict(scoring_func="softmax" if case["route"] == "softmax" else "sigmoid", renormalize=True,
                             routed_scaling_factor=2.5 if grouped else 1.0, num_expert_group=8 if grouped else 1,
                             topk_group=4 if grouped else 1)
        st["g_weights"], st["g_loss"] = _normal((T, k), g, 0.1, F32), torch.full((), 0.01, device=DEV)
    elif case["op"] == "residual":
        H, rt = case["H"], _TYPES[case["res"]]
        st["y"], st["residual"] = _normal((T, H), g), _normal((T, H), g, 2.0, rt)
        st["norm_weight"] = _normal((H,), g, 0.1, rt, 1.0) if case["post"] else None
        st["next_weight"] = _normal((H,), g, 0.1, rt, 1.0) if case["next"] else None
        shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[case["gate"]]
        st["gate"] = None if shape is None else _normal(shape, g, 0.3, BF16 if shape == (T, H) else rt, 0.5)
        st["scale"] = 0.5
        if case["train"]:
            st["g_h"] = _normal((T, H), g, 1e-3, rt)
            st["g_z"] = _normal((T, H), g, 1e-3) if case["next"] else None
    elif case["op"] == "act":
        st["x"], st["grad"] = _normal((T, 2 * case["I"]), g, 2.0), _normal((T, case["I"]), g, 1e-3)
    else:
        K, N = case["K"], case["N"]
        # a few channels are far larger than the rest
        st["x"] = _normal((T, K), g) * (1.0 + 15.0 * (torch.rand((K,), generator=g, device=DEV) < 0.01)).to(BF16)
        st["weight"], st["grad"] = _normal((N, K), g, 0.02), _normal((T, N), g, 1e-3)
        st["bias"] = _normal((N,), g, 0.1, F32) if case["bias"] else None
    return st


_TYPES = {"bf16": BF16, "f32": F32}


# ---------------------------------------------------------------- one pass


def run(st):
    op = st["case"]["op"]
    if op == "balance":
        return _balance_own(st) if own else _balance(st)
    if op == "residual":
        return _residual_own(st) if own else _residual(st)
    if op == "act":
        return _act_own(st) if own else _act(st)
    return _linear_own(st) if own else _linear(st)


def _balance_own(st):
    from qmoe.layers.moe_routing import balanced_experts

    c = st["case"]
    lg = st["logits"].detach().requires_grad_(c["train"])
    w, ids, loss, counts = balanced_experts(lg, c["k"], e_score_correction_bias=st["correction"], token_mask=st["mask"],
                                            **st["routing"])
    if not c["train"]:
        return w, ids, loss, counts
    (dl,) = torch.autograd.grad((w, loss), lg, (st["g_weights"], st["g_loss"]))
    return w.detach(), ids, loss.detach(), counts, dl


def _residual_own(st):
    from qmoe.layers.block import block_residual

    c = st["case"]
    names = ("y", "residual", "gate", "norm_weight", "next_weight")
    a = {n: st[n] if st[n] is None else st[n].detach().requires_grad_(c["train"]) for n in names}
    out = block_residual(scale=st["scale"], eps=EPS, **a)
    out = out if c["next"] else (out,)
    if not c["train"]:
        return out
    leaves = [t for t in a.values() if t is not None]
    grads = torch.autograd.grad(out, leaves, (st["g_h"], st["g_z"])[: len(out)])
    return (*(t.detach() for t in out), *grads)


def _act_own(st):
    from qmoe.layers.block import checkpointed_activation

    x = st["x"].detach().requires_grad_()
    h = checkpointed_activation(x, st["case"]["act"])
    return h.detach(), torch.autograd.grad(h, x, st["grad"])[0]


def _linear_own(st):
    from qmoe.layers.block import checkpointed_linear

    leaves = [st[n].detach().requires_grad_() for n in ("x", "weight", "bias") if st[n] is not None]
    y = checkpointed_linear(*leaves)
    return (y.detach(), *torch.autograd.grad(y, leaves, st["grad"]))


# ---- plain forms (float32, rounded once at the end)


def _scores(st):
    x = st["logits"].double()  # scores next to each other decide the choice
    if st["routing"]["scoring_func"] == "softmax":
        e = (x - x.amax(-1, keepdim=True)).exp()
        return (e / e.sum(-1, keepdim=True)).float()
    return (1.0 / (1.0 + (-x).exp())).float()


def _choose(st, score):
    """Experts [T, k]; ties go to the lowest expert."""
    c, r = st["case"], st["routing"]
    choice = score if st["correction"] is None else score + st["correction"]
    if r["num_expert_group"] > 1:
        per = choice.view(c["T"], r["num_expert_group"], -1)
        rank = per.sort(dim=-1, descending=True)[0][..., :2].sum(-1).sort(dim=-1, descending=True, stable=True)[1]
        kept = torch.zeros(per.shape[:2], dtype=torch.bool, device=DEV).scatter_(1, rank[:, : r["topk_group"]], True)
        choice = torch.where(kept[..., None], per, torch.full_like(per, -math.inf)).view(c["T"], -1)
    return choice.sort(dim=-1, descending=True, stable=True)[1][:, : c["k"]]


def _balance(st):
    c, rsf = st["case"], st["routing"]["routed_scaling_factor"]
    T, E, k = c["T"], c["E"], c["k"]
    s = _scores(st)
    ids = _choose(st, s)
    live = torch.ones(T, device=DEV) if st["mask"] is None else st["mask"].float()
    top = s.gather(1, ids)
    total = top.sum(-1, keepdim=True)
    w = rsf * top / total * live[:, None]
    counts = torch.zeros(E, device=DEV).index_add_(0, ids.flatten(), live.repeat_interleave(k))
    softmax = st["routing"]["scoring_func"] == "softmax"
    row = s.sum(-1, keepdim=True)
    p = s if softmax else s / row
    n = live.sum()
    coef = counts * E / (k * n * n)  # d loss / d p of a counted token
    loss = (coef * (p * live[:, None]).sum(0)).sum()
    if not c["train"]:
        return w, ids.int(), loss, counts.int()
    gw = st["g_weights"] * live[:, None]
    gp = st["g_loss"] * coef * live[:, None]
    gs = gp if softmax else (gp - (gp * p).sum(-1, keepdim=True)) / row
    gs = gs.scatter_add(1, ids, rsf * (gw - (gw * top).sum(-1, keepdim=True) / total) / total)
    d = s * (gs - (gs * s).sum(-1, keepdim=True)) if softmax else gs * s * (1.0 - s)
    return w, ids.int(), loss, counts.int(), d.to(st["logits"].dtype)


def _rstd(a):
    return ((a * a).mean(-1, keepdim=True) + EPS).rsqrt()


def _norm_grad(a, r, w, g):
    """Gradients of a * r * w (r: _rstd(a)) for a gradient g: of a, and of w per element."""
    n, gw = a * r, g * w
    return (gw - n * (gw * n).mean(-1, keepdim=True)) * r, g * n


def _residual(st):
    c, rt = st["case"], st["residual"].dtype
    y, gate = st["y"].float(), None if st["gate"] is None else st["gate"].float()
    ry = _rstd(y)
    b = y * ry * st["norm_weight"].float() if c["post"] else y
    h = (st["residual"].float() + st["scale"] * (b if gate is None else gate * b)).to(rt)
    out = [h]
    hf = h.float()  # the next norm is that of h as it is stored
    if c["next"]:
        rh = _rstd(hf)
        out.append((hf * rh * st["next_weight"].float()).to(BF16))
    if not c["train"]:
        return out
    g, dnext = st["g_h"].float(), None
    if c["next"]:
        d, dnext = _norm_grad(hf, rh, st["next_weight"].float(), st["g_z"].float())
        g = g + d
    dgate = st["scale"] * g * b
    if c["gate"] in ("channel", "token"):
        dgate = dgate.sum(0) if c["gate"] == "channel" else dgate.sum(-1, keepdim=True)
    db, dpost = st["scale"] * (g if gate is None else g * gate), None
    if c["post"]:
        db, dpost = _norm_grad(y, ry, st["norm_weight"].float(), db)
    out += [db.to(BF16), g.to(rt)]
    if gate is not None:
        out.append(dgate.to(st["gate"].dtype))
    return out + [d.sum(0).to(rt) for d in (dpost, dnext) if d is not None]


def _eight_bits(x):
    """x as 8 bits hold it: e4m3 times the least power of two that keeps 32 columns within 448."""
    n = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -n % 32)).unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -119)
    m = torch.frexp(top)[0]
    s = top / m * torch.where(m > 0.875, 2.0 ** -8, 2.0 ** -9)  # (top / m is a power of two, exactly)
    return ((v / s).to(F8).float() * s).flatten(-2)[..., :n]


def _act(st):
    act, x = st["case"]["act"], st["x"].float()
    I = st["case"]["I"]
    gate, up = x[:, :I], x[:, I:]
    h = _activate(act, gate, up)[0]
    _, dg, du = _activate(act, _eight_bits(st["x"][:, :I]), _eight_bits(st["x"][:, I:]))
    g = st["grad"].float()
    return h.to(BF16), torch.cat((g * dg, g * du), -1).to(BF16)


def _activate(act, g, u):
    """(value, derivative by the gate, by the up value)"""
    if act == "swigluoai":
        gc, uc = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        s = torch.sigmoid(1.702 * gc)
        return ((uc + 1.0) * gc * s, (uc + 1.0) * s * (1.0 + 1.702 * gc * (1.0 - s)) * (g <= 7.0),
                gc * s * (u.abs() <= 7.0))
    if act == "gelu":
        c = 0.7978845608028654
        t = torch.tanh(c * (g + 0.044715 * g ** 3))
        d = 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)
        return 0.5 * g * (1.0 + t) * u, d * u, 0.5 * g * (1.0 + t)
    s = torch.sigmoid(g)
    return g * s * u, s * (1.0 + g * (1.0 - s)) * u, g * s


def _linear(st):
    x, w, g = st["x"].float(), st["weight"].float(), st["grad"].float()
    y = x @ w.t()
    y = y if st["bias"] is None else y + st["bias"]
    out = y.to(BF16), (g @ w).to(BF16), (g.t() @ _eight_bits(st["x"])).to(BF16)
    return out if st["bias"] is None else (*out, g.sum(0))


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    T, train = case["T"], case.get("train", True)
    if case["op"] == "balance":
        E, k, size = case["E"], case["k"], 2 if case["logits"] == "bf16" else 4
        by = T * (E * size + k * 8) + E * 4
        return dict(bytes=by + (T * (E * size + k * 4) if train else 0), flops=T * E * (30 if train else 20))
    if case["op"] == "residual":
        H, size = case["H"], 2 if case["res"] == "bf16" else 4
        full = 2 if case["gate"] == "full" else 0
        nxt = 2 if case["next"] else 0
        by = 2 + size + full + size + nxt  # y, residual, gate, h, z
        if train:
            by += size + nxt + 2 + size + full  # gradients of h and z in, of y, residual and gate out
        return dict(bytes=T * H * by, flops=T * H * (30 if train else 10))
    if case["op"] == "act":
        return dict(bytes=T * case["I"] * (4 + 2 + 2 + 4), flops=T * case["I"] * 40)
    K, N = case["K"], case["N"]
    return dict(bytes=4 * (T * K + N * K + T * N), flops=6 * T * K * N)


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    return {"balance": _exact_balance, "residual": _exact_residual, "act": _exact_act, "linear": _exact_linear}[
        case["op"]](st)


def _exact_balance(st):
    c, r = st["case"], st["routing"]
    T, E, k = c["T"], c["E"], c["k"]
    lg = st["logits"].double().requires_grad_(c["train"])
    s = torch.softmax(lg, -1) if r["scoring_func"] == "softmax" else torch.sigmoid(lg)
    # the choice compares scores as float32 holds them: k times the first of the largest
    choice = s.detach().float()
    if st["correction"] is not None:
        choice = choice + st["correction"]
    if r["num_expert_group"] > 1:
        size = E // r["num_expert_group"]
        best = torch.stack([choice[:, i: i + size].topk(2, -1)[0].sum(-1) for i in range(0, E, size)], -1)
        for _ in range(r["num_expert_group"] - r["topk_group"]):  # drop the last of the smallest
            worst = best.shape[1] - 1 - best.flip(-1).argmin(-1)
            best[torch.arange(T, device=DEV), worst] = math.inf
        choice = torch.where(best.isinf().repeat_interleave(size, -1), -math.inf, choice)
    ids = []
    for _ in range(k):
        ids.append(choice.argmax(-1))
        choice = choice.scatter(1, ids[-1][:, None], -math.inf)
    ids = torch.stack(ids, -1)
    live = torch.ones(T, dtype=torch.bool, device=DEV) if st["mask"] is None else st["mask"]
    top = torch.gather(s, 1, ids)
    w = top / top.sum(-1, keepdim=True) * r["routed_scaling_factor"] * live[:, None]
    counts = torch.bincount(ids[live].flatten(), minlength=E)
    n = int(live.sum())
    loss = E * ((counts.double() / (k * n)) @ (s / s.sum(-1, keepdim=True))[live].mean(0))
    if not c["train"]:
        return w, ids.int(), loss, counts.int()
    (d,) = torch.autograd.grad((w, loss), lg, (st["g_weights"].double(), st["g_loss"].double()))
    return w.detach(), ids.int(), loss.detach(), counts.int(), d


def _exact_residual(st):
    c = st["case"]
    names = [n for n in ("y", "residual", "gate", "norm_weight", "next_weight") if st[n] is not None]
    a = {n: st[n].double().requires_grad_(c["train"]) for n in names}

    def norm(v, w):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS) * w

    b = norm(a["y"], a["norm_weight"]) if c["post"] else a["y"]
    h = a["residual"] + st["scale"] * (a["gate"] * b if "gate" in a else b)
    h = h + (h.to(st["residual"].dtype).double() - h).detach()  # as it is stored; its gradient passes
    out = (h, norm(h, a["next_weight"])) if c["next"] else (h,)
    if not c["train"]:
        return [t.detach() for t in out]
    grads = torch.autograd.grad(out, list(a.values()), [st[n].double() for n in ("g_h", "g_z")[: len(out)]])
    return [*(t.detach() for t in out), *grads]


def _exact_eight(x):
    """x [T, n] rounded to 4 significant bits, 2^-9 at least, below each 32 columns' power of two."""
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    for c0 in range(0, x.shape[1], 32):
        v = x[:, c0: c0 + 32].double()
        top = v.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -119)
        unit = top / torch.frexp(top)[0] / 512.0  # top = f 2^n, f in [1/2, 1): 2^n / 512
        unit = torch.where(top > 448.0 * unit, 2.0 * unit, unit)
        q = (v / unit).abs()
        near = q.clamp_min(2.0 ** -6)
        step = near / torch.frexp(near)[0] / 16.0
        out[:, c0: c0 + 32] = torch.round(q / step) * step * unit * torch.sign(v)
    return out


def _exact_act(st):
    I, act = st["case"]["I"], st["case"]["act"]

    def value(g, u):
        if act == "swigluoai":
            g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
            return g / (1.0 + torch.exp(-1.702 * g)) * (1.0 + u)
        if act == "gelu":
            return g * u / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))
        return g / (1.0 + torch.exp(-g)) * u

    hs, ds = [], []
    for t0 in range(0, st["case"]["T"], 1024):  # (float64 autograd of whole tensors does not fit beside the rest)
        x = st["x"][t0: t0 + 1024]
        g = _exact_eight(x[:, :I]).requires_grad_()
        u = _exact_eight(x[:, I:]).requires_grad_()
        hs.append(value(x[:, :I].double(), x[:, I:].double()))
        ds.append(torch.cat(torch.autograd.grad(value(g, u), (g, u), st["grad"][t0: t0 + 1024].double()), -1))
    return torch.cat(hs), torch.cat(ds)


def _exact_linear(st):
    x, w, g = st["x"].double(), st["weight"].double(), st["grad"].double()
    y = torch.mm(x, w.T)
    if st["bias"] is not None:
        y += st["bias"].double()
    out = y, torch.mm(g, w), torch.mm(g.T, _exact_eight(st["x"]))
    return out if st["bias"] is None else (*out, g.sum(0))
