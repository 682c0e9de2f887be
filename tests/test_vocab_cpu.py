"""The vocabulary operators without a GPU: shapes and types under fake
tensors, and the refusals of the wrappers and of the C entry points."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from qmoe import _capi, ops
from qmoe.layers.vocab import embedding, vocab_cross_entropy


def test_lookup_fake_shapes_and_gradient():
    with FakeTensorMode():
        w = torch.empty((1000, 96), dtype=torch.bfloat16, device="cuda", requires_grad=True)
        ids = torch.empty((3, 5), dtype=torch.int32, device="cuda")
        out = embedding(ids, w, scale=2.0, padding_idx=7)
        assert out.shape == (3, 5, 96) and out.dtype == torch.bfloat16
        assert out.requires_grad
        dw = torch.ops.qmoe.vocab_lookup_grad(torch.empty_like(out), ids, 1000, 2.0, 7, torch.bfloat16)
        assert dw.shape == w.shape and dw.dtype == w.dtype
        q = torch.empty((1000, 96), dtype=torch.float8_e4m3fn, device="cuda")
        out = embedding(ids, q, torch.empty((1000, 1), device="cuda"), out_dtype=torch.float32)
        assert out.shape == (3, 5, 96) and out.dtype == torch.float32


def test_lookup_refusals():
    w, ids = torch.zeros((8, 16), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="device tensors"):
        embedding(ids, w)
    with pytest.raises(ValueError, match="int32 or int64"):
        embedding(ids.to(torch.int16), w)
    with pytest.raises(ValueError, match="one scale per row"):
        embedding(ids, w.to(torch.float8_e4m3fn))
    with pytest.raises(ValueError, match="no row scales"):
        embedding(ids, w, torch.ones(8))
    with pytest.raises(ValueError, match="row scales must be"):
        embedding(ids, w.to(torch.int8), torch.ones(7))
    with pytest.raises(ValueError, match="contiguous"):
        embedding(ids, w.t())
    with pytest.raises(ValueError, match="bf16, f32"):
        embedding(ids, w.to(torch.float16))
    with pytest.raises(ValueError, match="padding_idx"):
        embedding(ids, w, padding_idx=8)
    with pytest.raises(ValueError, match="bf16, f16 or f32"):
        embedding(ids, w, out_dtype=torch.float64)
    with pytest.raises(NotImplementedError, match="no gradient"):
        q = w.float().requires_grad_()
        embedding(ids, q.to(torch.float8_e4m3fn), torch.ones(8))
    with pytest.raises(NotImplementedError, match="not f16"):
        embedding(ids, w.clone().requires_grad_(), out_dtype=torch.float16)


def test_lookup_grad_refusals():
    g, ids = torch.zeros((3, 16)), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="device tensors"):
        ops.vocab_lookup_grad(g, ids, 8)
    with pytest.raises(ValueError, match="for ids of"):
        ops.vocab_lookup_grad(g[:2], ids, 8)
    with pytest.raises(ValueError, match="bf16 or f32"):
        ops.vocab_lookup_grad(g.half(), ids, 8)
    with pytest.raises(ValueError, match="padding_idx"):
        ops.vocab_lookup_grad(g, ids, 8, padding_idx=-1)
    with pytest.raises(ValueError, match="`into`"):
        ops.vocab_lookup_grad(g, ids, 8, into=torch.zeros((7, 16)))
    with pytest.raises(ValueError, match="not torch.float16"):
        ops.vocab_lookup_grad(g, ids, 8, dtype=torch.float16)


def test_lookup_entry_points_check_their_arguments():
    lib, n = _capi.lib, ctypes.c_int64(0)
    a = ctypes.c_void_p(0x1000)
    call = lambda N=4, wt=0, ldw=64, rs=None, V=8, H=64, ot=0: lib.qmoe_vocab_lookup(  # noqa: E731
        a, 1, N, a, wt, ldw, rs, V, H, 1.0, a, ot, 64, None)
    assert call(N=-1) == 1 and call(N=1 << 24) == 1 and call(V=0) == 1 and call(ldw=63) == 1 and call(ot=3) == 1
    assert call(wt=2) == 1 and call(wt=6) == 1
    assert call(wt=3) == 1 and call(rs=a) == 1  # row scales exactly for 1-byte codes
    assert call(N=0) == 0
    assert lib.qmoe_vocab_lookup_grad_workspace_size(100, 50, 64, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.qmoe_vocab_lookup_grad_workspace_size(100, 0, 64, ctypes.byref(n)) == 1
    grad = lambda gt=0, wt=0, ws=a, size=1 << 20, ldg=64: lib.qmoe_vocab_lookup_grad(  # noqa: E731
        a, 1, 100, a, gt, ldg, 50, 64, 1.0, -1, a, wt, 64, 0, ws, size, None)
    assert grad(gt=2) == 1 and grad(wt=3) == 1 and grad(ldg=63) == 1
    assert grad(ws=None) == 2 and grad(size=n.value - 1) == 2


def test_loss_fake_shapes():
    with FakeTensorMode():
        x = torch.empty((3, 5, 96), dtype=torch.bfloat16, device="cuda", requires_grad=True)
        t = torch.empty((3, 5), dtype=torch.int64, device="cuda")
        w = torch.empty((1000, 96), dtype=torch.bfloat16, device="cuda", requires_grad=True)
        loss, lse = vocab_cross_entropy(x, w, t)
        assert loss.shape == lse.shape == (3, 5) and loss.dtype == lse.dtype == torch.float32 and loss.requires_grad
        dx, dw = torch.ops.qmoe.vocab_loss_grad(x, w, t, lse, lse, None, None, -100, True, True)
        assert dx.shape == x.shape and dw.shape == w.shape and dx.dtype == dw.dtype == torch.bfloat16
        q = torch.empty((1000, 96), dtype=torch.int8, device="cuda")
        assert vocab_cross_entropy(x.detach(), q, t, torch.empty(1000, device="cuda"))[0].shape == (3, 5)
        with pytest.raises(ValueError, match="multiples of 8"):
            vocab_cross_entropy(x.detach()[..., :95], w.detach()[:, :95], t)


def test_loss_refusals():
    x, w = torch.zeros((3, 16), dtype=torch.bfloat16), torch.zeros((8, 16), dtype=torch.bfloat16)
    t = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="device tensors"):
        vocab_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="hidden states must be bf16"):
        vocab_cross_entropy(x.float(), w, t)
    with pytest.raises(ValueError, match="hidden states must be bf16"):
        vocab_cross_entropy(x[:, :8], w, t)
    with pytest.raises(ValueError, match="targets of"):
        vocab_cross_entropy(x, w, t[:2])
    with pytest.raises(ValueError, match="int32 or int64"):
        vocab_cross_entropy(x, w, t.float())
    with pytest.raises(ValueError, match="must be bf16, e4m3"):
        vocab_cross_entropy(x, w.float(), t)
    with pytest.raises(ValueError, match="multiples of 8"):
        vocab_cross_entropy(x[:, :12], w[:, :12], t)
    with pytest.raises(ValueError, match="multiples of 8"):
        vocab_cross_entropy(x, torch.zeros((8, 20), dtype=torch.bfloat16)[:, :16], t)
    with pytest.raises(ValueError, match="16-byte aligned"):
        vocab_cross_entropy(x, torch.zeros(8 * 16 + 1, dtype=torch.bfloat16)[1:].view(8, 16), t)
    with pytest.raises(ValueError, match="one scale per row"):
        vocab_cross_entropy(x, w.to(torch.int8), t)
    with pytest.raises(NotImplementedError, match="no gradient"):
        ops.vocab_loss_grad(x, w.to(torch.int8), t, torch.zeros(3), torch.zeros(3), weight_scale=torch.ones(8))
    with pytest.raises(ValueError, match="g_loss must be"):
        ops.vocab_loss_grad(x, w, t, torch.zeros(3), torch.zeros(2))


def test_loss_entry_points_check_their_arguments():
    lib, n, a = _capi.lib, ctypes.c_int64(0), ctypes.c_void_p(0x1000)
    size = lambda T=100, V=500, H=64, wt=0: lib.qmoe_vocab_loss_workspace_size(T, V, H, wt, ctypes.byref(n))  # noqa: E731
    assert size() == 0 and n.value > 0
    assert size(H=60) == size(V=0) == size(T=-1) == size(wt=1) == size(T=1 << 20, V=1 << 24) == 1
    assert lib.qmoe_vocab_loss_grad_workspace_size(100, 500, 64, 0, 1, 1, ctypes.byref(n)) == 0
    need = n.value
    loss = lambda x=a, ldx=64, wt=0, rs=None, ws=a, size=1 << 24, T=100: lib.qmoe_vocab_loss(  # noqa: E731
        x, ldx, T, a, wt, 64, rs, 500, 64, a, 1, -100, a, a, ws, size, None)
    assert loss(ldx=60) == loss(ldx=68) == loss(wt=1) == loss(wt=3) == loss(rs=a) == loss(x=ctypes.c_void_p(0x1008)) == 1
    assert loss(ws=None) == loss(size=100) == 2 and loss(T=0) == 0
    grad = lambda dx=a, dw=a, wt=0, rs=None, lddx=64, size=1 << 24, T=100: lib.qmoe_vocab_loss_grad(  # noqa: E731
        a, 64, T, a, wt, 64, rs, 500, 64, a, 1, -100, a, a, None, dx, lddx, dw, 64, a, size, None)
    assert grad(dx=None, dw=None) == grad(wt=4, rs=a) == grad(lddx=62) == grad(T=0) == 1
    assert grad(size=need - 1) == 2


def test_no_gradient_through_row_scales():
    q, s = torch.zeros((8, 16), dtype=torch.int8), torch.ones(8, requires_grad=True)
    ids, x = torch.zeros(3, dtype=torch.int64), torch.zeros((3, 16), dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="or its scales"):
        embedding(ids, q, s)
    with pytest.raises(NotImplementedError, match="or its scales"):
        vocab_cross_entropy(x, q, ids, s)
    with torch.no_grad(), pytest.raises(ValueError, match="device tensors"):
        embedding(ids, q, s)


def test_which_tables_of_a_method_the_lookup_takes():
    """The others keep the method's torch operations, and with them their results,
    errors and gradients."""
    z = lambda *s, dtype=torch.int8: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    w, s, ids = z(50, 64), z(50, 1, dtype=torch.float32), z(3, 4, dtype=torch.int64)
    takes = lambda i=ids, t=w, r=s, o=torch.bfloat16: ops.vocab_lookup_takes(i, t, r, o)  # noqa: E731
    assert takes() and takes(t=z(50, 64, dtype=torch.float8_e4m3fn)) and takes(t=z(50, 96)[:, :64]) and takes(i=ids[:0])
    assert takes(i=z((1 << 24) - 1, dtype=torch.int32)) and not takes(i=z(1 << 24, dtype=torch.int32))
    assert takes(t=z(1 << 27, 8), r=z(1 << 27, dtype=torch.float32))
    assert not takes(t=z((1 << 27) + 1, 8), r=z((1 << 27) + 1, dtype=torch.float32))
    assert takes(t=z(50, 1 << 20)) and not takes(t=z(50, (1 << 20) + 8))
    assert not takes(t=z(0, 64), r=z(0, dtype=torch.float32)) and not takes(t=z(64, 50).t()) and not takes(r=s[:49])
    assert not takes(t=z(50, 64, dtype=torch.uint8)) and not takes(r=s.double()) and not takes(o=torch.float64)
    assert not takes(t=z(50, 64, dtype=torch.bfloat16))
    assert not takes(r=s.clone().requires_grad_())
    trainable = z(50, 64, dtype=torch.float8_e4m3fn).requires_grad_()
    assert not takes(t=trainable)  # (its output asks for a gradient, which torch then refuses)
    with torch.no_grad():
        assert takes(t=trainable) and takes(r=s.clone().requires_grad_())


def test_method_embedding_of_a_trainable_code_table_asks_for_its_gradient():
    from qmoe.layers.quantization.fp8 import Fp8LinearMethod

    with FakeTensorMode():
        layer = torch.nn.Module()
        layer.weight = torch.empty((9, 16), dtype=torch.float8_e4m3fn, device="cuda").requires_grad_()
        layer.weight_scale, layer.params_dtype = torch.empty(9, device="cuda"), torch.bfloat16
        assert Fp8LinearMethod.embedding(None, layer, torch.empty(3, dtype=torch.int64, device="cuda")).requires_grad


def test_methods_leave_the_padding_of_a_table_out():
    from qmoe.layers.quantization.unquantized import UnquantizedLinearMethod
    from qmoe.layers.vocab import unpadded_rows

    w, s = torch.arange(24.0).view(8, 3), torch.arange(8.0)[:, None]
    assert unpadded_rows(w, s, None) == (w, s)
    rows, scales = unpadded_rows(w, s, 5)
    assert torch.equal(rows, w[:5]) and torch.equal(scales, torch.arange(5.0))
    assert unpadded_rows(w, None, 8)[1] is None
    for bad in (0, -1, 9):
        with pytest.raises(ValueError, match="vocab_size"):
            unpadded_rows(w, s, bad)
    with FakeTensorMode():
        layer = torch.nn.Module()
        layer.weight = torch.empty((64, 16), dtype=torch.bfloat16, device="cuda", requires_grad=True)
        x, t = torch.empty((3, 16), dtype=torch.bfloat16, device="cuda"), torch.empty(3, dtype=torch.int64, device="cuda")
        assert UnquantizedLinearMethod().cross_entropy(layer, x, t, vocab_size=50)[0].requires_grad
