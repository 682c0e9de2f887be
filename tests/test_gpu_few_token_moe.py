"""The two-launch MoE layer on the GPU against float64.

Bounds. A gate or up value is a float32 sum of H products of bf16 values (the
weights are the decoded codes times their scales, rounded once to bf16): off by
(H + 8) 2^-24 times the sum of the magnitudes. The activation carries that
through its partial derivatives (its clamps do not widen it), computes in
float32 with hardware exponentials (32 2^-24 of the magnitudes of its factors)
and is rounded to bf16 (half a step). The down sums add (I + 8) 2^-24 of their
magnitudes, the weighted sum one rounding each, the output half a bf16 step.
The routing weights are the router's float32 ones."""

from types import SimpleNamespace

import pytest
import torch

from qmoe import ops
from qmoe.layers.fused_moe import few_token_moe, moe_forward
from qmoe.layers.vocab import embedding, vocab_cross_entropy

pytestmark = pytest.mark.gpu

BF16, E4 = torch.bfloat16, torch.float8_e4m3fn
EPS, HALF = 2.0 ** -24, torch.finfo(BF16).eps / 2
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
FORMATS = ("mxfp4", "nvfp4", "int4", "fp8_w8a16", "bf16")


def _weights(dev, fmt, E, N, K, gen, group=64):
    """(stored weights, scales, the bf16 values the kernels multiply by, as float64)."""
    if fmt == "bf16":
        w = (torch.randn((E, N, K), generator=gen, device=dev) * 0.05).to(BF16)
        return w, None, w.double()
    if fmt == "fp8_w8a16":
        q = (torch.randn((E, N, K), generator=gen, device=dev) * 60).clamp(-448, 448).to(E4)
        s = torch.rand((E, N, K // 128), generator=gen, device=dev) * 1e-3 + 1e-4
        return q, s, (q.float() * s.repeat_interleave(128, -1)).to(BF16).double()
    b = torch.randint(0, 256, (E, N, K // 2), generator=gen, device=dev, dtype=torch.uint8)
    c = torch.stack((b & 15, b >> 4), -1).flatten(-2).int()
    if fmt == "int4":
        s = (torch.rand((E, N, K // group), generator=gen, device=dev) * 0.01 + 1e-3).to(BF16)
        return b.view(torch.int32), s, ((c - 8).float() * s.float().repeat_interleave(group, -1)).to(BF16).double()
    v = torch.tensor(E2M1 + [-x for x in E2M1], device=dev).index_select(0, c.flatten()).view(c.shape)
    if fmt == "mxfp4":
        s = torch.randint(118, 123, (E, N, K // 32), generator=gen, device=dev, dtype=torch.uint8)
        return b, s, (v * torch.exp2(s.float() - 127).repeat_interleave(32, -1)).double()
    s = (torch.rand((E, N, K // 16), generator=gen, device=dev) * 0.02 + 1e-3).to(BF16)
    return b, s, (v * s.float().repeat_interleave(16, -1)).to(BF16).double()


def _act(act, g, u):
    """(h, |dh/dg|, |dh/du|, the magnitude of its factors) at the clamped values."""
    lo, hi = (-7.0, 7.0) if act == "swigluoai" else (-10.0, 10.0)
    if act in ("swigluoai", "silu_and_mul_with_clamp"):
        g, u = g.clamp(max=hi), u.clamp(lo, hi)
    g, u = g.clone().requires_grad_(), u.clone().requires_grad_()
    if act == "swigluoai":
        h = (u + 1) * (g * torch.sigmoid(1.702 * g))
    elif act == "gelu":
        h = 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3))) * u
    elif act == "situ:4.0:none":
        h = 4.0 * torch.tanh(g / 4.0) * torch.sigmoid(g) * u
    else:
        h = g * torch.sigmoid(g) * u
    dg, du = torch.autograd.grad(h.sum(), (g, u))
    return h.detach(), dg.abs(), du.abs(), (g.abs() * (1 + u.abs())).detach()


def _layer(dev, fmt, T, E, k, H, I, seed=0, bias=True, group=64):
    gen = torch.Generator(device=dev).manual_seed(seed)
    c = SimpleNamespace(fmt=fmt, T=T, E=E, k=k, H=H, I=I)
    c.w1, c.s1, c.v1 = _weights(dev, fmt, E, 2 * I, H, gen, group)
    c.w2, c.s2, c.v2 = _weights(dev, fmt, E, H, I, gen, group)
    c.b1 = torch.randn((E, 2 * I), generator=gen, device=dev) * 0.2 if bias else None
    c.b2 = torch.randn((E, H), generator=gen, device=dev) * 0.2 if bias else None
    c.x = torch.randn((T, H), generator=gen, device=dev).to(BF16)
    c.logits = torch.randn((T, E), generator=gen, device=dev).to(BF16)
    return c


def _run(c, act="silu", **routing):
    return few_token_moe(c.x, c.logits, c.w1, c.w2, c.s1, c.s2, c.b1, c.b2, c.k, act, weight_format=c.fmt, **routing)


def _check(c, out, tw, ids, act, skip=False):
    """out against float64 for routing weights tw [T, k] and experts ids."""
    T, k, H, I = c.T, c.k, c.H, c.I
    e, x = ids.long().flatten(), c.x.double().repeat_interleave(k, 0)
    ref, bound = torch.zeros((T, H), dtype=torch.float64, device=x.device), torch.zeros((T, H), dtype=torch.float64, device=x.device)
    for r in range(T * k):
        w = float(tw.flatten()[r])
        if skip and w == 0:
            continue
        W1, W2 = c.v1[e[r]], c.v2[e[r]]
        gu, gue = W1 @ x[r], (H + 8) * EPS * (W1.abs() @ x[r].abs())
        if c.b1 is not None:
            gu = gu + c.b1[e[r]].double()
            gue = gue + EPS * gu.abs()
        h, dg, du, fac = _act(act, gu[:I], gu[I:])
        he = 1.01 * (dg * gue[:I] + du * gue[I:]) + 32 * EPS * fac
        he = he + HALF * (h.abs() + he)
        y, ye = W2 @ h, W2.abs() @ he + (I + 8) * EPS * (W2.abs() @ (h.abs() + he))
        if c.b2 is not None:
            y = y + c.b2[e[r]].double()
        ref[r // k] += w * y
        bound[r // k] += abs(w) * (ye + (2 * k + 16) * EPS * (y.abs() + ye + (W2.abs() @ h.abs())))
    bound = bound + HALF * (ref.abs() + bound)
    assert out.shape == (T, H) and out.dtype == BF16
    off = (out.double() - ref).abs()
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 256, 128), (2, 16, 1, 128, 128), (3, 60, 6, 384, 256), (7, 130, 4, 640, 384),
                                       (16, 16, 8, 512, 256), (16, 256, 8, 256, 128), (5, 512, 4, 128, 128),
                                       (1, 4, 4, 2944, 128), (4, 32, 4, 128, 1408)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_values(dev, fmt, T, E, k, H, I):
    print(f"few-token moe {fmt} T={T} E={E} k={k} H={H} I={I}", flush=True)
    c = _layer(dev, fmt, T, E, k, H, I, bias=T % 2 == 1, group=128 if T == 7 else 64)
    out = _run(c)
    tw, ids = ops.moe_route(c.logits, k, weights_f32=True)
    _check(c, out, tw, ids, "silu")
    assert torch.equal(out, _run(c))  # the same bits on every call


@pytest.mark.parametrize("H,I", [(32, 32), (96, 160), (736, 352), (2880, 2880)])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "int4", "bf16"])
def test_widths_that_end_inside_a_granule(dev, fmt, H, I):
    c = _layer(dev, fmt, 3, 6, 2, H, I, seed=H, group=32)
    tw, ids = ops.moe_route(c.logits, 2, weights_f32=True)
    _check(c, _run(c), tw, ids, "silu")


@pytest.mark.parametrize("act", ["silu", "swigluoai", "gelu", "silu_and_mul_with_clamp", "situ:4.0:none"])
def test_activations(dev, act):
    c = _layer(dev, "bf16", 4, 8, 2, 256, 128, seed=2)
    c.x *= 8  # into the clamps
    tw, ids = ops.moe_route(c.logits, 2, weights_f32=True)
    _check(c, _run(c, act), tw, ids, act)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_routing_rules(dev, scoring, grouped, f32):
    c = _layer(dev, "mxfp4", 9, 64, 4, 256, 128, seed=4)
    c.logits = c.logits.float() * 1.37 if f32 else c.logits
    bias = torch.randn(64, device=dev) * 0.1 if grouped else None
    ng, tg = (8, 3) if grouped else (1, 1)
    tw, ids = ops.moe_route(c.logits, 4, scoring, not grouped, bias, 2.5, ng, tg, weights_f32=True)
    out = _run(c, "swigluoai", scoring_func=scoring, renormalize=not grouped, routed_scaling_factor=2.5,
               e_score_correction_bias=bias, num_expert_group=ng, topk_group=tg)
    _check(c, out, tw, ids, "swigluoai")


def test_uneven_experts(dev):
    """All tokens on the same experts, and equal logits (ties go to the lowest)."""
    c = _layer(dev, "nvfp4", 16, 32, 4, 256, 128, seed=5)
    c.logits[:] = c.logits[:1]
    tw, ids = ops.moe_route(c.logits, 4, weights_f32=True)
    assert (ids == ids[:1]).all()
    _check(c, _run(c), tw, ids, "silu")
    c.logits[:] = 0
    tw, ids = ops.moe_route(c.logits, 4, weights_f32=True)
    assert torch.equal(ids[0].cpu(), torch.arange(4, dtype=torch.int32))
    _check(c, _run(c), tw, ids, "silu")


def test_odd_rows_stay_in_their_row(dev):
    """A token of NaN, a row of NaN logits, weights of NaN in an expert that no
    finite token takes: the other tokens are what they were."""
    c = _layer(dev, "bf16", 6, 16, 2, 256, 128, seed=6)
    clean = _run(c)
    c.x[1] = float("nan")
    c.logits[4] = float("nan")
    out = _run(c)
    assert out[1].isnan().all() and out[4].isnan().all()
    keep = [0, 2, 3, 5]
    assert torch.equal(out[keep], clean[keep])
    _, ids = ops.moe_route(c.logits, 2)
    only = [e for e in ids[0].tolist() if e not in ids[[2, 3, 5]].flatten().tolist()]
    if only:
        c.w1[only[0]] = float("nan")
        c.w2[only[0]] = float("nan")
        out = _run(c)
        assert out[0].isnan().any() and torch.equal(out[[2, 3, 5]], clean[[2, 3, 5]])


def test_skip_padded_routes(dev):
    """Routes of weight 0 are padding: their experts' values, not even NaN, count."""
    c = _layer(dev, "bf16", 3, 8, 2, 128, 128, seed=7)
    c.logits = torch.full((3, 8), -200.0, device=dev)  # sigmoid scores that are 0
    c.logits[0, 5], c.logits[1, 2], c.logits[1, 3] = 2.0, 1.0, 0.5
    tw, ids = ops.moe_route(c.logits, 2, "sigmoid", False, weights_f32=True)
    assert (tw == 0).sum() == 3
    unused = sorted(set(range(8)) - {5, 2, 3})
    c.w1[unused], c.w2[unused] = float("nan"), float("nan")
    out = _run(c, scoring_func="sigmoid", renormalize=False, skip_padded_tokens=True)
    _check(c, out, tw, ids, "silu", skip=True)
    assert not out[2].any()


def test_strided_tokens_and_offsets_past_4_gib(dev):
    """Rows further apart, unaligned rows, and the last of experts whose
    weights lie beyond 4 GiB."""
    E, H, I = 80, 4096, 2048  # bf16: w1 1.3e9 values, 2.7 GB; w2 1.3 GB
    c = _layer(dev, "int4", 2, 4, 2, 256, 128, seed=8)
    ref = _run(c)
    wide = torch.zeros((2, 264), dtype=BF16, device=dev)
    wide[:, :256] = c.x
    c.x = wide[:, :256]
    assert torch.equal(_run(c), ref)
    odd = torch.zeros((2, 257), dtype=BF16, device=dev)
    odd[:, 1:] = c.x
    c.x = odd[:, 1:]
    assert torch.equal(_run(c), ref)
    w1 = torch.zeros((E * 2, 2 * I, H), dtype=BF16, device=dev)  # 5.4 GB
    w2 = torch.zeros((E * 2, H, I), dtype=BF16, device=dev)
    w1[-1, :4], w1[-1, I:I + 4], w2[-1, :, :4] = 0.25, 0.5, 1.0
    x = torch.zeros((1, H), dtype=BF16, device=dev)
    x[0, -1] = 4.0
    logits = torch.zeros((1, E * 2), device=dev)
    logits[0, -1] = 9.0
    out = few_token_moe(x, logits, w1, w2, None, None, None, None, 1, "silu", weight_format="bf16")
    h = torch.tensor(1.0 / (1.0 + 2.718281828459045 ** -1.0) * 2.0).to(BF16).double()
    assert ((out.double() - 4 * h.to(dev)).abs() <= HALF * 4 * h.to(dev) * 2).all()


def test_streams_and_graph(dev):
    c = _layer(dev, "mxfp4", 8, 64, 4, 512, 256, seed=9)
    ref = _run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = _run(c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(c)
        again = _run(c)
    for _ in range(3):
        c.x.copy_(torch.randn_like(c.x))
        c.logits.copy_(torch.randn_like(c.logits))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _run(c)) and torch.equal(again, out)


def test_compiles(dev):
    c = _layer(dev, "nvfp4", 2, 8, 2, 256, 128)
    fn = torch.compile(lambda x, lg: few_token_moe(x, lg, c.w1, c.w2, c.s1, c.s2, c.b1, c.b2, 2, "silu",
                                                   weight_format="nvfp4"), fullgraph=True, backend="eager")
    assert torch.equal(fn(c.x, c.logits), _run(c))


@pytest.mark.parametrize("fmt", FORMATS)
def test_methods_take_it_on_request(dev, fmt, monkeypatch):
    """`moe_forward` keeps its results without the switch and takes the
    two-launch layer with it, up to its token count."""
    c = _layer(dev, fmt, 6, 32, 4, 256, 128, seed=11)
    layer = SimpleNamespace(moe_config=SimpleNamespace(experts_per_token=4), _qmoe_activation="silu",
                            scoring_func="softmax", renormalize=True)
    fwd = lambda: moe_forward(layer, c.x, c.logits, c.w1, c.w2, c.s1, c.s2, c.b1, c.b2, fmt)  # noqa: E731
    with ops.record_plans() as plans:
        before = fwd()
    assert len(plans) == 2  # its two grouped products
    monkeypatch.setenv("QMOE_FEW_TOKEN_MOE", "5")
    assert torch.equal(fwd(), before)
    monkeypatch.setenv("QMOE_FEW_TOKEN_MOE", "6")
    with ops.record_plans() as plans:
        after = fwd()
    assert not plans and torch.equal(after, _run(c))
    tw, ids = ops.moe_route(c.logits, 4, weights_f32=True)
    _check(c, after, tw, ids, "silu")


def test_a_step_from_tokens_to_their_scores(dev):
    """Lookup, MoE layer and vocabulary loss in a row, as a decode step that
    scores its tokens runs them, captured and replayed, against float64."""
    V = 997
    c = _layer(dev, "mxfp4", 5, 32, 4, 256, 128, seed=12)
    table = (torch.randn((V, 256), device=dev) * 0.1).to(BF16)
    gate = (torch.randn((32, 256), device=dev) * 0.1).to(BF16)
    ids, nxt = torch.randint(0, V, (5,), device=dev), torch.randint(0, V, (5,), device=dev)

    def step():
        x = embedding(ids, table, scale=16.0)
        logits = (x.float() @ gate.float().t())
        y = few_token_moe(x, logits, c.w1, c.w2, c.s1, c.s2, c.b1, c.b2, 4, "swigluoai", weight_format="mxfp4")
        return (x, logits, y) + vocab_cross_entropy(y, table, nxt)

    graph = torch.cuda.CUDAGraph()
    step()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        ids.copy_(torch.randint(0, V, (5,), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)
    c.x, c.logits, y, loss, lse = captured
    assert torch.equal(c.x, (table[ids].float() * 16).to(BF16))
    tw, e = ops.moe_route(c.logits, 4, weights_f32=True)
    _check(c, y, tw, e, "swigluoai")
    lg = y.double() @ table.double().t()
    ref = torch.logsumexp(lg, 1) - lg[torch.arange(5, device=dev), nxt]
    # logits' float32 sums, and the roundings of the loss
    lim = 264 * EPS * (y.double().abs() @ table.double().t().abs()).amax(1) + 300 * EPS * (1 + lg.abs().amax(1))
    assert ((loss.double() - ref).abs() <= 2 * lim).all()


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4", "int4"])
def test_a_scale_that_is_no_number_stays_in_its_row(dev, fmt, T):
    """Rows that end inside a pair of 16-byte chunks: the scale behind their end
    is the next row's first."""
    c = _layer(dev, fmt, T, 8, 2, 96, 96, seed=14, group=32)
    clean = _run(c)
    if fmt == "mxfp4":
        c.s2[:, 5, 0] = 255
    else:
        c.s2[:, 5, 0] = float("nan")
        c.s2[:, 40, 0] = float("inf")
    out, bad = _run(c), [5] if fmt == "mxfp4" else [5, 40]
    assert not out[:, bad].isfinite().any()
    kept = [n for n in range(96) if n not in bad]
    assert torch.equal(out[:, kept], clean[:, kept])


def _by_definition(c):
    """The experts' values as the weight formats define them, in float64: fp8's
    scales, too, are rounded to bf16 before they multiply the codes."""
    if c.fmt != "fp8_w8a16":
        return c.v1, c.v2
    return tuple((q.float() * s.to(BF16).float().repeat_interleave(128, -1)).to(BF16).double()
                 for q, s in ((c.w1, c.s1), (c.w2, c.s2)))


def _check_both(c, after, before, tw, ids):
    """Both paths' outputs against the layer with its bf16 intermediate values in
    float64. A value of h that float32 sums may round either way moves by its
    step (`flip`); the four-launch path (`before`) also rounds the routing
    weights and the route outputs to bf16, half a step each."""
    v1, v2 = _by_definition(c)
    T, k, H, I = c.T, c.k, c.H, c.I
    e, x = ids.long().flatten(), c.x.double().repeat_interleave(k, 0)
    ref, bound, mag = (torch.zeros((T, H), dtype=torch.float64, device=x.device) for _ in range(3))
    for r in range(T * k):
        w, W1, W2 = float(tw.flatten()[r]), v1[e[r]], v2[e[r]]
        gu, gue = W1 @ x[r], (H + 8) * EPS * (W1.abs() @ x[r].abs())
        if c.b1 is not None:
            gu = gu + c.b1[e[r]].double()
            gue = gue + EPS * gu.abs()
        h, dg, du, fac = _act("silu", gu[:I], gu[I:])
        he = 1.01 * (dg * gue[:I] + du * gue[I:]) + 32 * EPS * fac
        hr, lo, hi = (v.to(BF16).double() for v in (h, h - he, h + he))
        flip = torch.maximum((lo - hr).abs(), (hi - hr).abs())
        y, size = W2 @ hr, W2.abs() @ (hr.abs() + flip)
        ye = W2.abs() @ flip + (I + 8) * EPS * size
        if c.b2 is not None:
            y = y + c.b2[e[r]].double()
        ref[r // k] += w * y
        bound[r // k] += abs(w) * (ye + (2 * k + 16) * EPS * (y.abs() + ye + size))
        mag[r // k] += abs(w) * (y.abs() + ye)
    for out, more in ((after, 0.0), (before, (2 * HALF + HALF * HALF) * mag)):
        lim = bound + more
        lim = lim + HALF * (ref.abs() + lim)
        off = (out.double() - ref).abs()
        assert out.shape == (T, H) and (off <= lim).all(), float((off / lim).max())


def _method_outputs(c, monkeypatch, limit):
    """The layer through `moe_forward`: by the two-launch layer, and without it."""
    layer = SimpleNamespace(moe_config=SimpleNamespace(experts_per_token=c.k), _qmoe_activation="silu",
                            scoring_func="softmax", renormalize=True)
    outs = []
    for switch in (limit, "0"):
        monkeypatch.setenv("QMOE_FEW_TOKEN_MOE", switch)
        outs.append(moe_forward(layer, c.x, c.logits, c.w1, c.w2, c.s1, c.s2, c.b1, c.b2, c.fmt))
    return outs


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T", [1, 6])
def test_the_switch_keeps_the_weights(dev, fmt, T, monkeypatch):
    """With and without the switch a layer multiplies by the same weights: the
    results differ by the routing weights' and route outputs' roundings alone."""
    c = _layer(dev, fmt, T, 32, 4, 256, 128, seed=16)
    after, before = _method_outputs(c, monkeypatch, "16")
    tw, ids = ops.moe_route(c.logits, 4, weights_f32=True)
    _check_both(c, after, before, tw, ids)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,k", [(9, 8), (16, 8), (11, 10)])
def test_methods_take_steps_of_up_to_128_routes(dev, fmt, T, k, monkeypatch):
    """More routes than the other path's route + dispatch launch holds."""
    c = _layer(dev, fmt, T, 32, k, 256, 128, seed=17)
    after, before = _method_outputs(c, monkeypatch, "16")
    assert torch.equal(after, _run(c))
    tw, ids = ops.moe_route(c.logits, k, weights_f32=True)
    _check_both(c, after, before, tw, ids)
