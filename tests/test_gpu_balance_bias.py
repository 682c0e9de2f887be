"""Gradient of balanced routing where a correction bias, or the groups, put an expert
of a small score first, against float64 with the bounds of the balance's other tests."""

import pytest
import torch

from qmoe.layers.moe_routing import balanced_experts
from test_gpu_balance import EPS, F32, _case, _check, _scores

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("first", [-20.0, -13.0, -9.0, -2.0])
@pytest.mark.parametrize("k", [2, 3, 8])
def test_a_small_score_first(dev, first, scoring, k):
    """The other weights' gradients come from their own gw and the first's share of the
    sum, which is as small as its score: no rounding error of the first's gw."""
    E, T = 24, 9
    g = torch.Generator(device=dev).manual_seed(k)
    lg = torch.randn((T, E), generator=g, device=dev)
    lg[:, 5] = first
    bias = torch.zeros(E, device=dev)
    bias[5] = 8.0
    gw = 1e-6 * torch.randn((T, k), generator=g, device=dev)
    gw[:, 0] = 1.0 + torch.rand(T, generator=g, device=dev)
    a = lg.clone().requires_grad_()
    w, ids, loss, counts = balanced_experts(a, k, scoring, e_score_correction_bias=bias)
    assert (ids[:, 0] == 5).all() and (w[:, 0] < w[:, 1]).all()
    (d,) = torch.autograd.grad(w, a, gw)
    _check(lg, k, scoring, True, 1.0, None, ids, w, loss, counts, gw, None, d)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "sqrtsoftplus"])
def test_biased_choices(dev, scoring):
    """Random biases: the largest score is anywhere among the choices, masks and groups
    beside them; the loss's gradient with them."""
    lg, mask, g = _case(dev, 300, 96, F32, 11, 1)
    bias = 3.0 * torch.randn(96, generator=g, device=dev)
    gw, gl = torch.randn((300, 6), generator=g, device=dev), torch.tensor(0.7, device=dev)
    for groups, keep in ((1, 1), (8, 3)):
        a = lg.clone().requires_grad_()
        w, ids, loss, counts = balanced_experts(a, 6, scoring, True, bias, 2.5, groups, keep, mask)
        assert (w.argmax(-1)[mask] != 0).any()
        (d,) = torch.autograd.grad((w, loss), a, (gw, gl))
        _check(lg, 6, scoring, True, 2.5, mask, ids, w, loss, counts, gw, gl, d)


def test_the_largest_score_last(dev):
    """One weight that is nearly all, chosen last: the gradient has the size of the other
    score, e^-14, relative to which it is exact (14 EPS of the scores' argument, 24 more,
    twice)."""
    x = torch.full((1, 16), -40.0, device=dev)
    x[0, 3], x[0, 5] = 8.0, -14.0
    bias = torch.zeros(16, device=dev)
    bias[5] = 4.0
    gw = torch.tensor([[3.0, 1.0]], device=dev)
    a = x.clone().requires_grad_()
    w, ids, _, _ = balanced_experts(a, 2, "sigmoid", e_score_correction_bias=bias)
    assert ids.tolist() == [[5, 3]]
    (got,) = torch.autograd.grad(w, a, gw)
    b = x.double().requires_grad_()
    top = _scores(b, "sigmoid")[:, [5, 3]]
    (ref,) = torch.autograd.grad(top / top.sum(-1, keepdim=True), b, gw.double())
    assert ((got.double() - ref).abs() <= 2 * (14 + 24) * EPS * ref.abs() + 2.0 ** -60).all()
