"""Routing with its balance loss, counts and gradient on the GPU against float64.

Experts and weights are those of the router (`ops.moe_route`, float32), bit for
bit. Bounds, in units of EPS = 2^-24, a float32 rounding. Loss: every p is a
quotient (3 roundings) and no sum of positive terms is longer than 64 additions
deep (a wavefront's tokens, 16 wavefronts, 16 x 16 workgroups). Gradient: a score
is off by the rounding of its exponential's argument (|x - max|), the exponential
itself, sums of E terms in 64 lanes and a quotient (24 in all); `mag` adds the
magnitudes of what a gradient is the sum of; a bf16 result is rounded by half a step."""

import pytest
import torch

from qmoe import ops
from qmoe.layers.moe_routing import balanced_experts, select_experts

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
EPS = 2.0 ** -24


def _scores(lg, scoring):
    if scoring == "softmax":
        return torch.softmax(lg, -1)
    return torch.sigmoid(lg) if scoring == "sigmoid" else torch.nn.functional.softplus(lg).sqrt()


def _case(dev, T, E, dtype=F32, seed=0, pad=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    lg = (torch.randn((T, E), generator=g, device=dev) + 0.5 * torch.randn(E, generator=g, device=dev)).to(dtype)
    mask = torch.rand(T, generator=g, device=dev) < 0.7 if pad else None
    return lg, mask, g


def _check(lg, k, scoring, renorm, rsf, mask, ids, w, loss, counts, gw, gl, d):
    T, E = lg.shape
    live = torch.ones(T, dtype=torch.bool, device=lg.device) if mask is None else mask
    x = lg.double().requires_grad_()
    s = _scores(x, scoring)
    top = s.gather(1, ids.long())
    den = top.sum(-1, keepdim=True) if renorm else 1.0
    ref_w = rsf * top / den * live[:, None]
    assert ((w.double() - ref_w).abs() <= (k + 8) * EPS * ref_w).all()
    ref_c = torch.bincount(ids[live].flatten().long(), minlength=E)
    assert torch.equal(counts.long(), ref_c)
    n = int(live.sum())
    p = s / s.sum(-1, keepdim=True)
    coef = ref_c.double() * E / (k * n * n) if n else torch.zeros(E, device=lg.device, dtype=torch.float64)
    ref_loss = (coef * p[live].sum(0)).sum()
    assert (loss.double() - ref_loss).abs() <= (64 + 8) * EPS * ref_loss
    if gw is None and gl is None:
        return
    total = 0.0
    if gw is not None:
        total = total + (ref_w * gw.double()).sum()
    if gl is not None:
        total = total + ref_loss * gl.double()
    (ref,) = torch.autograd.grad(total, x)
    with torch.no_grad():
        c = coef * (gl.double().abs() if gl is not None else 0.0)
        if scoring == "softmax":
            gs = c.expand(T, E).clone()
        else:
            gs = (c + (c * p).sum(-1, keepdim=True)) / s.sum(-1, keepdim=True)
        if gw is not None:
            a = gw.double().abs()
            part = rsf * (a + (a * top).sum(-1, keepdim=True) / den) / den if renorm else rsf * a
            gs = gs.scatter_add(1, ids.long(), part)
        if scoring == "softmax":
            mag = s * (gs + (gs * s).sum(-1, keepdim=True))
        elif scoring == "sigmoid":
            mag = gs * s * (1 - s)
        else:
            mag = gs * torch.sigmoid(x) / (2 * s)
        mag = mag * live[:, None]
        depth = 48 + 4 * (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True))
        half = torch.finfo(d.dtype).eps / 2
        assert d.dtype == lg.dtype
        assert ((d.double() - ref).abs() <= half * ref.abs() + depth * EPS * mag).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("T,E,k,dtype", [(1, 1, 1, F32), (1, 8, 2, BF16), (2, 3, 3, F32), (16, 64, 6, F32),
                                         (17, 65, 4, BF16), (32, 128, 4, F32), (33, 60, 4, BF16), (257, 256, 8, F32),
                                         (777, 129, 5, BF16), (1025, 384, 8, F32), (4097, 512, 64, BF16),
                                         (9001, 40, 1, F32)])
@pytest.mark.parametrize("pad", [0, 1])
def test_values_and_gradient(dev, T, E, k, dtype, scoring, pad):
    print(f"balance T={T} E={E} k={k} {dtype} {scoring} pad={pad}", flush=True)
    lg, mask, g = _case(dev, T, E, dtype, T + E, pad)
    renorm, rsf = T % 2 == 1, 2.5 if E % 2 else 1.0
    gw, gl = torch.randn((T, k), generator=g, device=dev), torch.tensor(0.7, device=dev)
    a = lg.clone().requires_grad_()
    w, ids, loss, counts = balanced_experts(a, k, scoring, renorm, routed_scaling_factor=rsf, token_mask=mask)
    rw, rids = ops.moe_route(lg, k, scoring, renorm, routed_scaling_factor=rsf, weights_f32=True)
    assert torch.equal(ids, rids)
    assert torch.equal(w, rw if mask is None else rw * mask[:, None])
    (d,) = torch.autograd.grad((w, loss), a, (gw, gl))
    _check(lg, k, scoring, renorm, rsf, mask, ids, w, loss, counts, gw, gl, d)
    again = balanced_experts(lg, k, scoring, renorm, routed_scaling_factor=rsf, token_mask=mask)
    for x, y in zip(again, (w, ids, loss, counts)):
        assert torch.equal(x, y)
    if mask is not None:
        assert (d[~mask] == 0).all() and (w[~mask] == 0).all()


@pytest.mark.parametrize("E,groups,keep", [(64, 8, 4), (256, 8, 4), (60, 4, 2), (96, 2, 1)])
@pytest.mark.parametrize("bias", [False, True])
def test_grouped_choice_is_the_routers(dev, E, groups, keep, bias):
    lg, _, g = _case(dev, 50, E, BF16, E)
    b = torch.randn(E, generator=g, device=dev) * 0.1 if bias else None
    layer = torch.nn.Module()
    layer.use_grouped_topk, layer.num_expert_group, layer.topk_group = True, groups, keep
    layer.e_score_correction_bias, layer.routed_scaling_factor = b, 2.5
    a = lg.clone().requires_grad_()
    w, ids, loss, counts = balanced_experts(a, 6, "sigmoid", True, b, 2.5, groups, keep)
    sw, sids = select_experts(lg, lg, topk=6, renormalize=True, scoring_fn="sigmoid", layer=layer)
    assert torch.equal(ids, sids) and torch.equal(w.to(BF16), sw)
    gw = torch.randn(w.shape, generator=g, device=dev)
    (d,) = torch.autograd.grad((w, loss), a, (gw, torch.ones((), device=dev)))
    _check(lg, 6, "sigmoid", True, 2.5, None, ids, w, loss, counts, gw, torch.ones((), device=dev), d)


def test_one_gradient_alone(dev):
    lg, mask, g = _case(dev, 70, 48, seed=5, pad=1)
    gw, gl = torch.randn((70, 4), generator=g, device=dev), torch.tensor(-2.0, device=dev)
    for part in ("weights", "loss"):
        a = lg.clone().requires_grad_()
        w, ids, loss, counts = balanced_experts(a, 4, "sigmoid", token_mask=mask)
        (d,) = torch.autograd.grad(w, a, gw) if part == "weights" else torch.autograd.grad(loss, a, gl)
        _check(lg, 4, "sigmoid", True, 1.0, mask, ids, w, loss, counts, gw if part == "weights" else None,
               gl if part == "loss" else None, d)


def test_gradient_against_differences(dev):
    """Central differences of step h of the float64 operator's float32 values: off by
    the third derivative (below 1 here) times h^2, and by the values' rounding / h.
    A step across which the choice changes is left out: weights and counts jump by a
    fixed amount there, which no difference of the smooth parts bounds."""
    lg, mask, g = _case(dev, 5, 8, seed=9, pad=1)
    gw = torch.randn((5, 2), generator=g, device=dev)
    a = lg.clone().requires_grad_()
    w, ids, loss, _ = balanced_experts(a, 2, "softmax", token_mask=mask)
    (d,) = torch.autograd.grad((w * gw).sum() + loss, a)
    h, compared = 2.0 ** -7, 0
    for t in range(5):
        for e in range(8):
            v = []
            for sign in (1, -1):
                x = lg.clone()
                x[t, e] += sign * h
                xw, xids, xl, _ = balanced_experts(x, 2, "softmax", token_mask=mask)
                v.append(((xw * gw).sum() + xl).double() if torch.equal(xids, ids) else None)
            if None in v:
                continue
            compared += 1
            assert abs((v[0] - v[1]) / (2 * h) - d[t, e].double()) <= 16 * h * h + 64 * EPS / h
    assert compared >= 30


def test_masked_tokens_may_hold_anything(dev):
    lg, _, _ = _case(dev, 40, 32, seed=2)
    mask = torch.arange(40, device=dev) < 29
    dirty = lg.clone()
    dirty[29:33], dirty[33:36], dirty[36:] = float("nan"), float("inf"), -float("inf")
    out, grads = [], []
    for x in (lg, dirty):
        a = x.clone().requires_grad_()
        w, ids, loss, counts = balanced_experts(a, 3, token_mask=mask)
        (d,) = torch.autograd.grad(w.sum() * 2 + loss, a)
        out.append((w, ids[:29], loss, counts))
        grads.append(d)
    for x, y in zip(*out):
        assert torch.equal(x, y)
    assert torch.equal(*grads) and (grads[0][29:] == 0).all()


@pytest.mark.parametrize("T", [1, 20, 300])
def test_no_counted_token(dev, T):
    lg, _, _ = _case(dev, T, 16)
    a = lg.clone().requires_grad_()
    w, ids, loss, counts = balanced_experts(a, 2, token_mask=torch.zeros(T, dtype=torch.bool, device=dev))
    (d,) = torch.autograd.grad(loss + w.sum(), a)
    assert loss == 0 and (counts == 0).all() and (w == 0).all() and (d == 0).all()


def test_infinite_and_nan_logits(dev):
    """An expert at -inf is never preferred and has no share; a NaN row is a NaN loss
    and gradient of its own row."""
    lg, _, _ = _case(dev, 6, 16, seed=3)
    lg[:, 5] = -float("inf")
    for scoring in ("softmax", "sigmoid", "sqrtsoftplus"):
        a = lg.clone().requires_grad_()
        w, ids, loss, counts = balanced_experts(a, 4, scoring)
        (d,) = torch.autograd.grad(w.square().sum() + loss, a)
        assert torch.isfinite(d).all() and torch.isfinite(loss) and (d[:, 5] == 0).all() and counts[5] == 0
    lg[2, 3] = float("nan")
    a = lg.clone().requires_grad_()
    w, ids, loss, counts = balanced_experts(a, 4, "softmax")
    (d,) = torch.autograd.grad(w.square().sum() + loss, a)
    assert torch.isnan(loss) and torch.isnan(w[2]).all() and torch.isnan(d[2]).all()
    rest = torch.arange(6, device=dev) != 2
    assert torch.isfinite(w[rest]).all() and torch.isfinite(d[rest]).all()


def test_half_precision_strided_and_empty(dev):
    lg, _, g = _case(dev, 30, 16, seed=4)
    want = balanced_experts(lg.half().float(), 2)
    a = lg.half().requires_grad_()
    got = balanced_experts(a, 2)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    assert torch.autograd.grad(got[0].sum() * 0.5 + got[2], a)[0].dtype == torch.float16
    wide = torch.randn((30, 64), generator=g, device=dev)
    for v in (wide[:, 8:24], wide.t()[:30], wide[:1, :16].expand(9, 16)):
        for x, y in zip(balanced_experts(v, 2), balanced_experts(v.contiguous(), 2)):
            assert torch.equal(x, y)
    a = lg[:0].clone().requires_grad_()
    w, ids, loss, counts = balanced_experts(a, 2)
    assert w.shape == ids.shape == (0, 2) and loss == 0 and (counts == 0).all()
    assert torch.autograd.grad(loss + w.sum(), a)[0].shape == (0, 16)


def test_captured_and_on_two_streams(dev):
    """Replays of a captured step, with other work between them, and calls on two
    streams at once equal the plain calls."""
    lgs = [_case(dev, 700, 96, seed=s)[0] for s in (1, 2, 3)]

    def step(x):
        a = x.detach().requires_grad_()
        w, ids, loss, counts = balanced_experts(a, 4, "sigmoid")
        return w.detach(), ids, loss.detach(), counts, torch.autograd.grad((w, loss), a, (gw, gl))[0]

    gw, gl = torch.randn((700, 4), device=dev), torch.tensor(0.3, device=dev)
    want = [step(x) for x in lgs]
    static = lgs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in (1, 2, 0, 1):
        static.copy_(lgs[i])
        graph.replay()
        step(lgs[2 - i])
        torch.cuda.synchronize()
        for x, y in zip(out, want[i]):
            assert torch.equal(x, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(lgs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            for x, y in zip(res, want[i]):
                assert torch.equal(x, y)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_renormalized_weight_has_no_gradient(dev, dtype, scoring):
    """It is the scaling factor whatever the logits are."""
    lg, mask, g = _case(dev, 70, 64, dtype, pad=1)
    gw = torch.randn((70, 1), generator=g, device=dev)
    a = lg.clone().requires_grad_()
    w, _, loss, _ = balanced_experts(a, 1, scoring, routed_scaling_factor=2.5, token_mask=mask)
    (alone,) = torch.autograd.grad(loss, a, retain_graph=True)
    (both,) = torch.autograd.grad((w, loss), a, (gw, torch.ones_like(loss)), retain_graph=True)
    (none,) = torch.autograd.grad(w, a, gw)
    assert alone.any() and torch.equal(both, alone) and not none.any()


@pytest.mark.parametrize("scoring,low", [("softmax", -7.0), ("sigmoid", -14.0)])
def test_a_weight_that_is_nearly_all(dev, scoring, low):
    """The gradient is of the size of the other weight, e^-14, and as exact relative to
    itself: the scores are off by the rounding of their argument (up to 14 EPS), 24 EPS
    more, and no sum cancels but those of the two weights' own terms (twice as many)."""
    E = 16
    x = torch.full((1, E), -40.0, device=dev)
    x[0, 3], x[0, 5] = (7.0, low) if scoring == "softmax" else (8.0, low)
    gw = torch.tensor([[3.0, 1.0]], device=dev)
    a = x.clone().requires_grad_()
    w, ids, _, _ = balanced_experts(a, 2, scoring)
    assert ids.tolist() == [[3, 5]]
    (got,) = torch.autograd.grad(w, a, gw)
    b = x.double().requires_grad_()
    top = _scores(b, scoring)[:, [3, 5]]
    (ref,) = torch.autograd.grad(top / top.sum(-1, keepdim=True), b, gw.double())
    assert ((got.double() - ref).abs() <= 2 * (14 + 24) * EPS * ref.abs() + 2.0 ** -60).all()
