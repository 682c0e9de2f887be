"""The vocabulary operators and the few-token MoE layer under traces, dispatch
modes and transforms, without a GPU: in the place of the launches stand simple
functions that, like them, write their results where torch cannot see it."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from qmoe import ops
from qmoe.layers.fused_moe import few_token_moe
from qmoe.layers.quantization.fp8 import Fp8LinearMethod
from qmoe.layers.vocab import embedding, vocab_cross_entropy

BF16 = torch.bfloat16


def _read(t):
    return list((ctypes.c_int64 * t.numel()).from_address(t.data_ptr()))


def _lookup(ids, weight, weight_scale=None, scale=1.0, out_dtype=BF16):
    row = weight.shape[1] * weight.element_size()
    out = torch.empty((*ids.shape, weight.shape[1]), dtype=weight.dtype)
    for i, k in enumerate(_read(ids.contiguous())):
        ctypes.memmove(out.data_ptr() + i * row, weight.data_ptr() + k * row, row)
    return out


def _lookup_grad(grad, ids, vocab, scale=1.0, padding_idx=None, dtype=BF16, into=None):
    out = torch.zeros((vocab, grad.shape[-1]), dtype=dtype)
    size = grad.shape[-1] * grad.element_size()
    for i, k in enumerate(_read(ids.contiguous())):  # (the ids of the tests that use it differ)
        ctypes.memmove(out.data_ptr() + k * size, grad.data_ptr() + i * size, size)
    return out


def _loss(x, weight, targets, weight_scale=None, ignore_index=-100):
    loss, lse = torch.empty(targets.shape), torch.empty(targets.shape)
    for out, sign in ((loss, 1.0), (lse, -1.0)):
        for i, k in enumerate(_read(targets.contiguous())):
            ctypes.c_float.from_address(out.data_ptr() + 4 * i).value = sign * k
    return loss, lse


def _few(x, *args):
    out, x = torch.empty(x.shape, dtype=BF16), x.contiguous()
    ctypes.memmove(out.data_ptr(), x.data_ptr(), 2 * x.numel())
    return out


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    calls = []
    for name, fn in (("vocab_lookup", _lookup), ("vocab_lookup_grad", _lookup_grad), ("vocab_loss", _loss),
                     ("moe_few_tokens", _few)):
        monkeypatch.setattr(ops, name, lambda *a, _fn=fn, _name=name: (calls.append(_name), _fn(*a))[1])
    return calls


TABLE = torch.arange(80.0).view(10, 8)
IDS, OTHER = torch.tensor([1, 3, 1]), torch.tensor([9, 0, 4])
X = torch.arange(24.0).view(3, 8).to(BF16)


def _experts():
    return (torch.zeros(3, 4, dtype=BF16), torch.zeros(4, 64, 32, dtype=BF16), torch.zeros(4, 32, 32, dtype=BF16))


def _calls():
    """(function of one operand, an operand, another, the answers to both)"""
    w = TABLE.to(BF16)
    lg, w1, w2 = _experts()
    x = torch.arange(96.0).view(3, 32).to(BF16)
    few = lambda v: few_token_moe(v, lg, w1, w2, None, None, None, None, 2, "silu")  # noqa: E731
    return {"lookup": (lambda i: embedding(i, w), IDS, OTHER, w[IDS], w[OTHER]),
            "loss": (lambda t: torch.stack(vocab_cross_entropy(X, w, t)), IDS, OTHER,
                     torch.stack((IDS.float(), -IDS.float())), torch.stack((OTHER.float(), -OTHER.float()))),
            "few": (few, x, x + 1, x, x + 1)}


@pytest.mark.parametrize("which", ["lookup", "loss", "few"])
def test_traces_record_the_call(which, launches):
    fn, a, b, at_a, at_b = _calls()[which]
    assert torch.equal(fn(a), at_a) and len(launches) == 1
    for traced in (make_fx(fn)(a), make_fx(fn, pre_dispatch=True)(a), make_fx(fn, tracing_mode="fake", _allow_non_fake_inputs=True)(a),
                   torch.jit.trace(fn, (a,)), torch.compile(fn, backend="eager", fullgraph=True)):
        assert torch.equal(traced(b), at_b) and torch.equal(traced(a), at_a)


@pytest.mark.parametrize("which", ["lookup", "loss", "few"])
def test_a_dispatch_mode_sees_the_call(which, launches):
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    fn, a, _, at_a, _ = _calls()[which]
    with Mode():
        assert torch.equal(fn(a), at_a)
    assert len([s for s in seen if s.startswith("qmoe.")]) == 1
    del seen[:]
    assert torch.equal(fn(a), at_a) and not seen


@pytest.mark.parametrize("which", ["lookup", "loss", "few"])
def test_vmap(which, launches):
    fn, a, b, at_a, at_b = _calls()[which]
    assert torch.equal(torch.vmap(fn)(torch.stack((a, b))), torch.stack((at_a, at_b)))


def test_vmap_over_tables():
    w = torch.stack((TABLE, TABLE + 100))
    assert torch.equal(torch.vmap(lambda t: embedding(IDS, t, out_dtype=torch.float32))(w), w[:, IDS])


def test_tangents_are_refused():
    """Forward mode, by dual numbers and by torch.func.jvp: an error, not a
    result without a tangent. Operands without one pass."""
    w, lg = TABLE.to(BF16), _experts()
    scales = torch.ones(10)
    few = lambda v, **kw: few_token_moe(v, lg[0], lg[1], lg[2], None, None, None, None, 2, "silu", **kw)  # noqa: E731
    x = torch.zeros(3, 32, dtype=BF16)
    for fn, t in ((lambda t: embedding(IDS, t), w), (lambda t: vocab_cross_entropy(X, t, IDS)[0], w),
                  (lambda t: vocab_cross_entropy(t, w, IDS)[0], X), (lambda t: embedding(IDS, w.to(torch.int8), t), scales),
                  (few, x), (lambda t: few(x, e_score_correction_bias=t), torch.zeros(4))):
        with fw.dual_level():
            fn(t)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(fw.make_dual(t, torch.ones_like(t)))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(fn, (t,), (torch.ones_like(t),))


def test_traces_of_a_gradient_record_the_call():
    def grad(i, up):
        w = TABLE.to(BF16).requires_grad_()
        return torch.autograd.grad(embedding(i, w), w, up)[0]

    ids, other = torch.tensor([1, 3, 5]), torch.tensor([9, 0, 4])
    want = torch.zeros(10, 8, dtype=BF16)
    want[other] = X
    assert torch.equal(make_fx(grad)(ids, X)(other, X), want)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_method_embedding_traces_and_batches(dtype):
    layer = torch.nn.Module()
    layer.weight, layer.params_dtype = TABLE.to(dtype), BF16
    layer.weight_scale = torch.arange(1.0, 11.0) / 8
    fn = lambda i: Fp8LinearMethod.embedding(None, layer, i)  # noqa: E731
    want = lambda i: TABLE.to(dtype).to(BF16)[i] * layer.weight_scale.to(BF16)[i, None]  # noqa: E731
    for traced in (make_fx(fn)(IDS), torch.jit.trace(fn, (IDS,))):
        assert torch.equal(traced(OTHER), want(OTHER))
    if dtype == torch.int8:  # (torch has no batched gather of float8 on the CPU)
        assert torch.equal(torch.vmap(fn)(torch.stack((IDS, OTHER))), torch.stack((want(IDS), want(OTHER))))
    with fw.dual_level():
        layer.weight_scale = fw.make_dual(layer.weight_scale, torch.ones(10))
        tangent = fw.unpack_dual(fn(IDS)).tangent
        assert torch.equal(tangent, TABLE.to(dtype).to(BF16)[IDS])


@pytest.mark.parametrize("which", ["x", "logits", "w1", "w2", "bias"])
def test_a_gradient_asked_of_the_layer_is_an_error(which):
    """Of any operand, the correction bias among them: the output says so when
    the gradient is asked for."""
    x, (lg, w1, w2), bias = torch.zeros(3, 32, dtype=BF16), _experts(), torch.zeros(4)
    {"x": x, "logits": lg, "w1": w1, "w2": w2, "bias": bias}[which].requires_grad_()
    out = few_token_moe(x, lg, w1, w2, None, None, None, None, 2, "silu", e_score_correction_bias=bias)
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="autograd"):
        out.sum().backward()


def test_tangents_of_a_gradient_are_refused():
    """Forward over reverse: the operand has no tangent, what comes back has."""
    w, x = TABLE.to(BF16).requires_grad_(), X.clone().requires_grad_()
    for fn, leaf in ((lambda: embedding(IDS, w), w), (lambda: vocab_cross_entropy(x, w, IDS)[0], x)):
        with fw.dual_level():
            out = fn()
            scaled = out * fw.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(scaled.sum(), leaf)


def test_tangents_of_trainable_operands_are_refused():
    w, x = TABLE.to(BF16).requires_grad_(), X.clone().requires_grad_()
    for fn, t in ((lambda t: embedding(IDS, t), w), (lambda t: vocab_cross_entropy(x, t, IDS)[0], w),
                  (lambda t: vocab_cross_entropy(t, w, IDS)[0], x)):
        with fw.dual_level():
            with pytest.raises(NotImplementedError, match="forward"):
                fn(fw.make_dual(t, torch.ones_like(t)))
