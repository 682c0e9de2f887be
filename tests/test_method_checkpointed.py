"""`apply_checkpointed` on layers that the unquantized method has made and loaded:
frozen and trainable weights, every bias and output size that `apply` takes.

Bounds: an output is off by half a bf16 step and by its float32 sum, `n + 8` roundings
(EPS = 2^-24) of its terms' magnitudes, n at most 128 here; a gradient the same."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from qmoe.layers.quantization.unquantized import UnquantizedLinearMethod

BF16, F16, F32, D = torch.bfloat16, torch.float16, torch.float32, torch.float64
EPS = 2.0 ** -24
METHOD = UnquantizedLinearMethod()


@pytest.mark.parametrize("n", [1, 7, 20, 24])
@pytest.mark.parametrize("bias", [None, BF16, F16, F32, D])
def test_shapes_of_every_size_and_bias(n, bias):
    with FakeTensorMode():
        layer = torch.nn.Module()
        layer.weight = torch.nn.Parameter(torch.empty((n, 64), dtype=BF16))
        x = torch.empty((3, 5, 64), dtype=F32, requires_grad=True)
        b = None if bias is None else torch.empty(n, dtype=bias, requires_grad=True)
        y = METHOD.apply_checkpointed(layer, x, b)
        assert y.shape == (3, 5, n) and y.dtype == BF16
        leaves = [t for t in (x, layer.weight, b) if t is not None]
        for g, t in zip(torch.autograd.grad(y.sum(), leaves), leaves):
            assert g.shape == t.shape and g.dtype == t.dtype


def _layer(n, k, dev, seed):
    layer = torch.nn.Module()
    METHOD.create_weights(layer, k, [n], k, n, BF16)
    g = torch.Generator().manual_seed(seed)
    layer.weight.data.copy_(0.1 * torch.randn((n, k), generator=g))
    return layer, (lambda *s: torch.randn(s, generator=g).to(dev))


def _near(got, ref, mag, n):
    lim = torch.finfo(got.dtype).eps / 2 * ref.abs() + (n + 8) * EPS * mag
    assert ((got.to(D) - ref).abs() <= lim).all()


def _eight(x):
    """the 8-bit values of rows [T, 32 m] of integers up to 8 in size: themselves"""
    assert torch.equal(x, x.round()) and x.abs().max() <= 8
    return x.to(D)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 13, 72])
@pytest.mark.parametrize("bias", [None, F16, F32])
def test_a_loaded_layer_made_trainable(dev, n, bias):
    T, K = 37, 96
    layer, rand = _layer(n, K, dev, n)
    METHOD.process_weights_after_loading(layer)
    layer.weight.requires_grad_()
    assert layer.weight.requires_grad and layer.weight.is_leaf and layer.weight.is_cuda
    x = (2 * rand(T, K)).round().clamp(-8, 8).to(BF16).requires_grad_()
    b = None if bias is None else rand(n).to(bias).requires_grad_()
    dy = rand(T, n).to(BF16)
    y = METHOD.apply_checkpointed(layer, x, b)
    leaves = [t for t in (x, layer.weight, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    xd, wd, gd = _eight(x.detach()), layer.weight.detach().to(D), dy.to(D)
    plus = 0.0 if b is None else b.detach().to(D)
    assert y.shape == (T, n) and y.dtype == BF16
    _near(y.detach(), xd @ wd.t() + plus, xd.abs() @ wd.abs().t() + abs(plus), K)
    _near(grads[0], gd @ wd, gd.abs() @ wd.abs(), n)
    _near(grads[1], gd.t() @ xd, gd.abs().t() @ xd.abs(), T)
    if b is not None:
        assert grads[2].dtype == bias
        _near(grads[2], gd.sum(0), gd.abs().sum(0), T)
    with torch.no_grad():
        assert torch.equal(METHOD.apply_checkpointed(layer, x, b), y)


@pytest.mark.gpu
def test_a_loaded_layer_is_frozen(dev):
    """... as it comes, also where the weight was trainable before: the input's gradient
    alone, and nothing of the input kept."""
    layer, rand = _layer(72, 96, dev, 1)
    layer.weight.requires_grad_()
    METHOD.process_weights_after_loading(layer)
    assert not layer.weight.requires_grad
    x = rand(20, 96).to(BF16).requires_grad_()
    y = METHOD.apply_checkpointed(layer, x)
    assert [t is None for t in y.grad_fn.saved_tensors] == [False, True, True]
    y.sum().backward()
    assert x.grad is not None and layer.weight.grad is None
