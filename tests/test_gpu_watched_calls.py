"""The vocabulary operators and the few-token MoE layer under traces and
transforms on the GPU: the same bits as the plain calls, for inputs that the
trace has not seen."""

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from qmoe.layers.fused_moe import few_token_moe
from qmoe.layers.quantization.fp8 import Fp8LinearMethod
from qmoe.layers.vocab import embedding, vocab_cross_entropy

pytestmark = pytest.mark.gpu

BF16, E4, E5, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e5m2, torch.int8


def _traces(fn, *args):
    return (make_fx(fn)(*args), make_fx(fn, pre_dispatch=True)(*args),
            torch.jit.trace(fn, args, check_trace=False))


def test_traced_and_batched_calls(dev):
    gen = torch.Generator(device=dev).manual_seed(1)
    w = torch.randn((300, 64), generator=gen, device=dev).to(BF16)
    x, up = (torch.randn((2, 9, 64), generator=gen, device=dev).to(BF16) for _ in range(2))
    ids = torch.randint(0, 300, (2, 9), generator=gen, device=dev)
    w1, w2 = (torch.randn(s, generator=gen, device=dev).to(BF16) for s in ((8, 128, 64), (8, 64, 64)))
    lg = torch.randn((9, 8), generator=gen, device=dev)

    def scores(h, t):
        return torch.stack(vocab_cross_entropy(h, w, t))

    def gradients(h, t):
        a, b = h.detach().requires_grad_(), w.detach().requires_grad_()
        return torch.autograd.grad(vocab_cross_entropy(a, b, t)[0].sum() + embedding(t, b).float().sum(), (a, b))

    def lookup(i):
        return embedding(i, w, scale=3.0)

    def layer(h):
        return few_token_moe(h, lg, w1, w2, None, None, None, None, 2, "silu")

    for fn, args in ((lookup, (ids,)), (scores, (x, ids)), (layer, (x,))):
        one, two = ([a[k] for a in args] for k in (0, 1))
        want = torch.stack((fn(*one), fn(*two)))
        for traced in _traces(fn, *one):
            assert torch.equal(traced(*two), want[1]) and torch.equal(traced(*one), want[0])
        assert torch.equal(torch.vmap(fn)(*args), want)
    for got, want in zip(make_fx(gradients)(x[0], ids[0])(x[1], ids[1]), gradients(x[1], ids[1])):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [E4, E5, I8])
def test_traced_and_batched_method_embedding(dev, dtype):
    """As the gather, cast and product of torch operations would be."""
    layer = torch.nn.Module()
    layer.weight = (torch.randn((70, 40), device=dev) * 20).to(dtype)
    layer.weight_scale, layer.params_dtype = torch.rand(70, device=dev) + 0.5, BF16
    ids = torch.randint(0, 70, (2, 5), device=dev)
    fn = lambda i: Fp8LinearMethod.embedding(None, layer, i)  # noqa: E731
    want = layer.weight.view(torch.uint8)[ids].view(dtype).to(BF16) * layer.weight_scale.to(BF16)[ids, None]
    for traced in _traces(fn, ids[0]):
        assert torch.equal(traced(ids[1]), want[1])
    assert torch.equal(torch.vmap(fn)(ids), want)
    with fw.dual_level():
        layer.weight_scale = fw.make_dual(layer.weight_scale, torch.ones(70, device=dev))
        out, tangent = fw.unpack_dual(fn(ids))
        assert torch.equal(out, want) and torch.equal(tangent, layer.weight.view(torch.uint8)[ids].view(dtype).to(BF16))
