"""Measured operators: the two ends of the vocabulary table (row lookup with
scaling and its gradient, softmax cross entropy of a projection onto the table
with its gradients) and the whole MoE layer of a decode step, through the
framework's public entry points (``own``) and in plain torch operations.
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
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
IGNORE = -100


def listed():
    return [
        # the next tokens of 8 sequences, rows of an FP8 table (one scale per row): latency
        dict(name="lookup_fp8_8", op="lookup", table="fp8", N=8, V=131072, H=4096, scaled=False),
        # a batch of prompts, rows scaled by sqrt(H)
        dict(name="lookup_bf16_16384", op="lookup", table="bf16", N=16384, V=131072, H=7168, scaled=True),
        # a short fine-tuning batch (odd count, odd vocabulary, padding at its end): output and table gradient
        dict(name="lookup_train_777", op="lookup_train", table="bf16", N=777, V=50021, H=2880, scaled=True),
        # a training batch whose tokens follow a natural frequency law: output and table gradient
        dict(name="lookup_train_16384", op="lookup_train", table="bf16", N=16384, V=131072, H=4096, scaled=False),
        # log-probability of one sampled token: a decode step that reports it
        dict(name="score_bf16_1", op="score", table="bf16", T=1, V=131072, H=4096, ignored=0),
        # the same for a decode batch of 16, FP8 table
        dict(name="score_fp8_16", op="score", table="fp8", T=16, V=131072, H=7168, ignored=0),
        # log-probabilities of a prompt (odd length), INT8 table of an odd vocabulary
        dict(name="score_int8_613", op="score", table="int8", T=613, V=32003, H=2880, ignored=5),
        # a short fine-tuning batch with unscored prompt tokens: loss and both gradients
        dict(name="train_bf16_333", op="train", table="bf16", T=333, V=50021, H=2880, ignored=101),
        # a training batch: loss and both gradients
        dict(name="train_bf16_4096", op="train", table="bf16", T=4096, V=131072, H=4096, ignored=7),
        # MXFP4 experts with biases, one user's token: latency
        dict(name="moe_mxfp4_1", op="moe", fmt="mxfp4", T=1, E=128, k=4, H=2880, I=2880, act="swigluoai", bias=True,
             route="softmax"),
        # the same layer, a decode batch of 16
        dict(name="moe_mxfp4_16", op="moe", fmt="mxfp4", T=16, E=128, k=4, H=2880, I=2880, act="swigluoai", bias=True,
             route="softmax"),
        # NVFP4 experts, grouped sigmoid routing with a correction bias, a decode batch of 8
        dict(name="moe_nvfp4_8", op="moe", fmt="nvfp4", T=8, E=256, k=8, H=7168, I=2048, act="silu", bias=False,
             route="grouped"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_train", "score", "score", "train", "moe", "moe"])
    V, H = _log_int(rng, 1000, 131072), 8 * _log_int(rng, 64, 896)
    if op == "lookup":
        return dict(op=op, table=rng.choice(["bf16", "fp8", "int8"]), N=_log_int(rng, 1, 16384), V=V, H=H,
                    scaled=rng.random() < 0.5)
    if op == "lookup_train":
        return dict(op=op, table="bf16", N=_log_int(rng, 1, 16384), V=V, H=H, scaled=rng.random() < 0.5)
    if op == "score":
        T = _log_int(rng, 1, 4096)
        return dict(op=op, table=rng.choice(["bf16", "fp8", "int8"]), T=T, V=V, H=H, ignored=rng.randint(0, T // 2))
    if op == "train":
        T = _log_int(rng, 1, min(4096, 4096 * 131072 * 4096 // (V * H)))
        return dict(op=op, table="bf16", T=T, V=V, H=H, ignored=rng.randint(0, T // 2))
    route = rng.choice(["softmax", "sigmoid", "grouped"])
    E, k = rng.choice([16, 32, 60, 64, 128, 256]), rng.choice([1, 2, 4, 6, 8])
    if route == "grouped":
        E = 64 if E == 60 else E
    return dict(op=op, fmt=rng.choice(["mxfp4", "nvfp4", "int4", "fp8_w8a16", "bf16"]), T=rng.randint(1, 16), E=E, k=k,
                H=128 * _log_int(rng, 4, 56), I=128 * _log_int(rng, 2, 22),
                act=rng.choice(["silu", "swigluoai", "gelu"]), bias=rng.random() < 0.5, route=route)


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(shape, g, std=1.0, dtype=BF16):
    return torch.empty(shape, device=DEV, dtype=dtype).normal_(0.0, std, generator=g)


def _uniform(shape, g, lo, hi, dtype=torch.float32):
    return torch.empty(shape, device=DEV, dtype=dtype).uniform_(lo, hi, generator=g)


def _table(kind, V, H, g):
    """Gaussian table rows: bf16, or codes with one f32 scale per row."""
    w = _normal((V, H), g, 0.02)
    if kind == "bf16":
        return w, None
    top = w.abs().amax(-1).float()
    if kind == "fp8":
        s = top / 448.0
        return (w / s[:, None]).clamp(-448, 448).to(F8), s
    s = top / 127.0
    return (w / s[:, None]).round().clamp(-127, 127).to(torch.int8), s


def _natural_ids(n, V, g):
    """Token ids whose frequency falls with their rank, ranks in random order."""
    rank = (V ** _uniform((n,), g, 0.0, 1.0, torch.float64)).long().clamp(1, V) - 1
    return torch.randperm(V, generator=g, device=DEV)[rank]


def _expert_weights(fmt, E, N, K, g):
    """Expert matrices [E, N, K] of standard deviation about 0.02 and their scales."""
    if fmt == "bf16":
        return _normal((E, N, K), g, 0.02), None
    if fmt == "fp8_w8a16":
        return _normal((E, N, K), g, 100.0).clamp_(-448, 448).to(F8), _uniform((E, N, K // 128), g, 1e-4, 3e-4)
    q = torch.randint(0, 256, (E, N, K // 2), device=DEV, dtype=torch.uint8, generator=g)
    if fmt == "mxfp4":
        return q, torch.randint(119, 122, (E, N, K // 32), device=DEV, dtype=torch.uint8, generator=g)
    if fmt == "nvfp4":
        return q, _uniform((E, N, K // 16), g, 4e-3, 1e-2, BF16)
    return q.view(torch.int32), _uniform((E, N, K // 128), g, 2e-3, 6e-3, BF16)  # int4, groups of 128


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case=case)
    if case["op"] in ("lookup", "lookup_train"):
        N, V, H = case["N"], case["V"], case["H"]
        st["weight"], st["weight_scale"] = _table(case["table"], V, H, g)
        st["ids"] = _natural_ids(N, V, g)
        st["scale"] = math.sqrt(H) if case["scaled"] else 1.0
        if case["op"] == "lookup_train":
            st["padding_idx"] = V - 1
            st["ids"][N - N // 16:] = V - 1
            st["grad"] = _normal((N, H), g, 1e-3)
        return st
    if case["op"] in ("score", "train"):
        T, V, H = case["T"], case["V"], case["H"]
        st["weight"], st["weight_scale"] = _table(case["table"], V, H, g)
        st["x"] = _normal((T, H), g)
        st["targets"] = _natural_ids(T, V, g)
        st["targets"][: case["ignored"]] = IGNORE
        if case["op"] == "train":
            st["grad"] = torch.full((T,), 1.0 / max(1, T - case["ignored"]), device=DEV)
        return st
    T, E, H, I = case["T"], case["E"], case["H"], case["I"]
    st["w1"], st["w1_scale"] = _expert_weights(case["fmt"], E, 2 * I, H, g)
    st["w2"], st["w2_scale"] = _expert_weights(case["fmt"], E, H, I, g)
    st["b1"] = _normal((E, 2 * I), g, 0.1, torch.float32) if case["bias"] else None
    st["b2"] = _normal((E, H), g, 0.1, torch.float32) if case["bias"] else None
    st["x"] = _normal((T, H), g)
    st["logits"] = _normal((T, E), g)
    grouped = case["route"] == "grouped"
    st["correction"] = _normal((E,), g, 0.1, torch.float32) if grouped else None
    st["routing"] = dict(scoring_func="softmax" if case["route"] == "softmax" else "sigmoid", renormalize=True,
                         routed_scaling_factor=2.5 if grouped else 1.0, num_expert_group=8 if grouped else 1,
                         topk_group=4 if grouped else 1)
    return st


# ---------------------------------------------------------------- one pass


def run(st):
    op = st["case"]["op"]
    if op == "lookup":
        return _lookup_own(st) if own else _lookup(st)
    if op == "lookup_train":
        return _lookup_train_own(st) if own else _lookup_train(st)
    if op == "score":
        return _score_own(st) if own else _score(st)
    if op == "train":
        return _train_own(st) if own else _train(st)
    return _moe_own(st) if own else _moe(st)


def _lookup_own(st):
    from qmoe.layers.vocab import embedding

    return embedding(st["ids"], st["weight"], st["weight_scale"], scale=st["scale"])


def _lookup_train_own(st):
    from qmoe.layers.vocab import embedding

    w = st["weight"].detach().requires_grad_()
    out = embedding(st["ids"], w, scale=st["scale"], padding_idx=st["padding_idx"])
    return out.detach(), torch.autograd.grad(out, w, st["grad"])[0]


def _score_own(st):
    from qmoe.layers.vocab import vocab_cross_entropy

    return vocab_cross_entropy(st["x"], st["weight"], st["targets"], st["weight_scale"], ignore_index=IGNORE)


def _train_own(st):
    from qmoe.layers.vocab import vocab_cross_entropy

    x, w = st["x"].detach().requires_grad_(), st["weight"].detach().requires_grad_()
    loss, lse = vocab_cross_entropy(x, w, st["targets"], ignore_index=IGNORE)
    dx, dw = torch.autograd.grad(loss, (x, w), st["grad"])
    return loss.detach(), lse.detach(), dx, dw


def _moe_own(st):
    from qmoe.layers.fused_moe import few_token_moe

    c = st["case"]
    return few_token_moe(st["x"], st["logits"], st["w1"], st["w2"], st["w1_scale"], st["w2_scale"], st["b1"], st["b2"],
                         c["k"], c["act"], weight_format=c["fmt"], e_score_correction_bias=st["correction"],
                         **st["routing"])


# ---- plain forms (float32, rounded once at the end)


def _rows(st):
    rows = st["weight"][st["ids"]].float()
    if st["weight_scale"] is not None:  # the row's scale is held in the output's type
        rows = rows * st["weight_scale"][st["ids"]].to(BF16).float()[:, None]
    return rows * st["scale"]


def _lookup(st):
    return _rows(st).to(BF16)


def _lookup_train(st):
    kept = (st["ids"] != st["padding_idx"]).float()[:, None]
    dw = torch.zeros(st["weight"].shape, device=DEV)
    dw.index_add_(0, st["ids"], st["grad"].float() * (kept * st["scale"]))
    return _rows(st).to(BF16), dw.to(BF16)


def _logits(st):
    logits = st["x"].float() @ st["weight"].float().t()
    return logits if st["weight_scale"] is None else logits * st["weight_scale"]


def _loss(st, logits):
    top = logits.amax(-1)
    lse = top + (logits - top[:, None]).exp().sum(-1).log()
    kept = st["targets"] != IGNORE
    at = logits.gather(1, st["targets"].clamp_min(0)[:, None])[:, 0]
    return torch.where(kept, lse - at, torch.zeros_like(lse)), lse, kept


def _score(st):
    return _loss(st, _logits(st))[:2]


def _train(st):
    logits = _logits(st)
    loss, lse, kept = _loss(st, logits)
    g = (st["grad"] * kept)[:, None]
    d = (logits - lse[:, None]).exp() * g
    d.scatter_add_(1, st["targets"].clamp_min(0)[:, None], -g)
    return loss, lse, (d @ st["weight"].float()).to(BF16), (d.t() @ st["x"].float()).to(BF16)


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _experts(fmt, w, s, e):
    """The matrices of experts e [R] in float32 [R, N, K]."""
    w = w[e]
    if fmt == "bf16":
        return w.float()
    s = s[e]
    if fmt == "fp8_w8a16":
        return w.float() * s.repeat_interleave(128, -1)
    b = w.view(torch.uint8)
    codes = torch.stack((b & 15, b >> 4), -1).flatten(-2)
    if fmt == "int4":
        return (codes.float() - 8.0) * s.float().repeat_interleave(128, -1)
    v = torch.tensor(_E2M1, device=DEV).index_select(0, codes.flatten().int()).view(codes.shape)
    if fmt == "mxfp4":
        return v * torch.exp2(s.float() - 127.0).repeat_interleave(32, -1)
    return v * s.float().repeat_interleave(16, -1)


def _activate(act, h):
    gate, up = h.chunk(2, -1)
    if act == "swigluoai":
        gate, up = gate.clamp(max=7.0), up.clamp(-7.0, 7.0)
        return (up + 1.0) * gate * torch.sigmoid(1.702 * gate)
    if act == "gelu":
        return 0.5 * gate * (1.0 + torch.tanh(0.7978845608028654 * (gate + 0.044715 * gate ** 3))) * up
    return gate * torch.sigmoid(gate) * up


def _routes(st):
    """Routing weights [T, k] and experts [T, k]; ties go to the lowest expert."""
    c, r = st["case"], st["routing"]
    x = st["logits"].double()  # scores next to each other decide the choice
    score = (torch.softmax(x, -1) if r["scoring_func"] == "softmax" else 1.0 / (1.0 + (-x).exp())).float()
    choice = score if st["correction"] is None else score + st["correction"]
    if r["num_expert_group"] > 1:
        per = choice.view(c["T"], r["num_expert_group"], -1)
        rank = per.sort(dim=-1, descending=True)[0][..., :2].sum(-1).sort(dim=-1, descending=True, stable=True)[1]
        kept = torch.zeros(per.shape[:2], dtype=torch.bool, device=DEV).scatter_(1, rank[:, : r["topk_group"]], True)
        choice = torch.where(kept[..., None], per, torch.full_like(per, -math.inf)).view(c["T"], -1)
    e = choice.sort(dim=-1, descending=True, stable=True)[1][:, : c["k"]]
    w = score.gather(1, e)
    return w / w.sum(-1, keepdim=True) * r["routed_scaling_factor"], e


def _moe(st):
    c = st["case"]
    w, e = _routes(st)
    flat = e.flatten()
    x = st["x"].float().repeat_interleave(c["k"], 0)
    h = torch.bmm(_experts(c["fmt"], st["w1"], st["w1_scale"], flat), x[..., None])[..., 0]
    h = _activate(c["act"], h if st["b1"] is None else h + st["b1"][flat])
    y = torch.bmm(_experts(c["fmt"], st["w2"], st["w2_scale"], flat), h[..., None])[..., 0]
    y = y if st["b2"] is None else y + st["b2"][flat]
    return (y.view(c["T"], c["k"], -1) * w[..., None]).sum(1).to(BF16)


# ---------------------------------------------------------------- what a pass cannot do without


_TABLE_BYTES = {"bf16": 2, "fp8": 1, "int8": 1}
_EXPERT_BITS = {"mxfp4": 4 + 8 / 32, "nvfp4": 4 + 16 / 16, "int4": 4 + 16 / 128, "fp8_w8a16": 8 + 32 / 128, "bf16": 16}


def work(case):
    H = case["H"]
    if case["op"] in ("lookup", "lookup_train"):
        N, V = case["N"], case["V"]
        by = N * (8 + H * (2 + _TABLE_BYTES[case["table"]]))
        return dict(bytes=by + ((N + V) * H * 2 if case["op"] == "lookup_train" else 0), flops=N * H)
    if case["op"] in ("score", "train"):
        T, V = case["T"], case["V"]
        by = V * H * _TABLE_BYTES[case["table"]] + T * (H * 2 + 16)
        if case["op"] == "score":
            return dict(bytes=by, flops=2 * T * V * H)
        return dict(bytes=by + (T + V) * H * 2, flops=6 * T * V * H)
    T, E, k, I = case["T"], case["E"], case["k"], case["I"]
    touched = E * (1.0 - (1.0 - k / E) ** T)  # experts that a batch of evenly spread tokens reaches
    return dict(bytes=int(touched * 3 * H * I * _EXPERT_BITS[case["fmt"]] / 8 + T * (4 * H + 2 * E)),
                flops=T * k * 6 * H * I)


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    return {"lookup": _exact_lookup, "lookup_train": _exact_lookup, "score": _exact_loss, "train": _exact_loss,
            "moe": _exact_moe}[case["op"]](st)


def _exact_lookup(st):
    out = st["weight"].index_select(0, st["ids"]) if st["weight_scale"] is None else st["weight"].view(
        torch.uint8).index_select(0, st["ids"]).view(st["weight"].dtype)
    out = out.double().mul_(st["scale"])
    if st["weight_scale"] is not None:
        out.mul_(st["weight_scale"].to(BF16).double().index_select(0, st["ids"]).unsqueeze(1))
    if st["case"]["op"] == "lookup":
        return out
    V, ids = st["weight"].shape[0], st["ids"]
    order = ids.argsort(stable=True)
    dw = torch.zeros(st["weight"].shape, dtype=torch.float64, device=DEV)
    uniq, count = torch.unique_consecutive(ids[order], return_counts=True)
    sums = torch.segment_reduce(st["grad"].double()[order], "sum", lengths=count, axis=0)
    keep = uniq != st["padding_idx"]
    dw[uniq[keep]] = sums[keep] * st["scale"]
    return out, dw


def _exact_loss(st):
    x = st["x"].double()
    w = st["weight"].double()
    if st["weight_scale"] is not None:
        w *= st["weight_scale"].double().unsqueeze(1)
    lg = torch.mm(x, w.T)
    lse = torch.logsumexp(lg, 1)
    rows = torch.arange(x.shape[0], device=DEV)
    scored = st["targets"].ne(IGNORE)
    loss = torch.zeros_like(lse)
    loss[scored] = lse[scored] - lg[rows[scored], st["targets"][scored]]
    if st["case"]["op"] == "score":
        return loss, lse
    lg.sub_(lse.unsqueeze(1)).exp_()
    lg[rows[scored], st["targets"][scored]] -= 1.0
    lg.mul_((st["grad"].double() * scored).unsqueeze(1))
    return loss, lse, torch.mm(lg, w), torch.mm(lg.T, x)


def _exact_matrix(fmt, w, s, e):
    """Expert e's matrix in float64, decoded field by field."""
    w = w[e]
    if fmt == "bf16":
        return w.double()
    s = s[e]
    if fmt == "fp8_w8a16":
        return (w.double().view(w.shape[0], -1, 128) * s.double().unsqueeze(-1)).flatten(1)
    b = w.view(torch.uint8)
    n = torch.empty(b.shape[0], b.shape[1] * 2, dtype=torch.float64, device=DEV)
    n[:, 0::2], n[:, 1::2] = (b % 16).double(), (b // 16).double()
    if fmt == "int4":
        return ((n - 8.0).view(n.shape[0], -1, 128) * s.double().unsqueeze(-1)).flatten(1)
    mag = n % 8.0
    ex, m = (mag / 2.0).floor(), mag % 2.0
    v = torch.where(ex == 0, 0.5 * m, (1.0 + 0.5 * m) * 2.0 ** (ex - 1.0))
    v = torch.where(n >= 8.0, -v, v)
    if fmt == "mxfp4":
        return (v.view(n.shape[0], -1, 32) * (2.0 ** (s.double() - 127.0)).unsqueeze(-1)).flatten(1)
    return (v.view(n.shape[0], -1, 16) * s.double().unsqueeze(-1)).flatten(1)


def _exact_moe(st):
    c, r = st["case"], st["routing"]
    out = torch.zeros((c["T"], c["H"]), dtype=torch.float64, device=DEV)
    logits = st["logits"].double().cpu()
    correction = None if st["correction"] is None else st["correction"].cpu()
    chosen = {}
    for t in range(c["T"]):
        x = logits[t]
        p = ((x - x.max()).exp() / (x - x.max()).exp().sum() if r["scoring_func"] == "softmax"
             else torch.sigmoid(x)).float()
        choice = (p if correction is None else p + correction).tolist()
        if r["num_expert_group"] > 1:
            size = c["E"] // r["num_expert_group"]
            best = [sum(sorted(choice[i * size:(i + 1) * size])[-2:]) for i in range(r["num_expert_group"])]
            kept = sorted(range(len(best)), key=lambda i: (-best[i], i))[: r["topk_group"]]
            choice = [v if i // size in kept else -math.inf for i, v in enumerate(choice)]
        top = sorted(range(c["E"]), key=lambda i: (-choice[i], i))[: c["k"]]
        total = sum(float(p[i]) for i in top)
        for i in top:
            chosen.setdefault(i, []).append((t, float(p[i]) / total * r["routed_scaling_factor"]))
    for e, users in chosen.items():
        t = torch.tensor([u[0] for u in users], device=DEV)
        h = st["x"][t].double() @ _exact_matrix(c["fmt"], st["w1"], st["w1_scale"], e).T
        h = h if st["b1"] is None else h + st["b1"][e].double()
        a, u = h[:, : c["I"]], h[:, c["I"]:]
        if c["act"] == "swigluoai":
            a, u = a.clamp(max=7.0), u.clamp(-7.0, 7.0)
            h = a / (1.0 + torch.exp(-1.702 * a)) * (1.0 + u)
        elif c["act"] == "gelu":
            h = a * u / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (a + 0.044715 * a * a * a)))
        else:
            h = a / (1.0 + torch.exp(-a)) * u
        y = h @ _exact_matrix(c["fmt"], st["w2"], st["w2_scale"], e).T
        y = y if st["b2"] is None else y + st["b2"][e].double()
        out[t] += y * torch.tensor([u[1] for u in users], dtype=torch.float64, device=DEV).unsqueeze(1)
    return out
