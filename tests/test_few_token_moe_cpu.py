"""The two-launch MoE layer without a GPU: shapes under fake tensors, the
descriptor's layout, refusals of the wrapper and of the C entry points."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from qmoe import _capi, ops
from qmoe.layers.fused_moe import few_token_moe


def _operands(fmt="mxfp4", T=3, E=8, H=256, I=128, device="cpu"):
    per, dt = {"mxfp4": (2, torch.uint8), "bf16": (1, torch.bfloat16), "int4": (8, torch.int32)}[fmt]
    sc = {"mxfp4": (32, torch.uint8), "int4": (64, torch.bfloat16), "bf16": None}[fmt]
    z = lambda *s, dtype: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    s1 = z(E, 2 * I, H // sc[0], dtype=sc[1]) if sc else None
    s2 = z(E, H, I // sc[0], dtype=sc[1]) if sc else None
    return [z(T, H, dtype=torch.bfloat16), z(T, E, dtype=torch.bfloat16), z(E, 2 * I, H // per, dtype=dt),
            z(E, H, I // per, dtype=dt), s1, s2, None, None]


@pytest.mark.parametrize("fmt", ["mxfp4", "int4", "bf16"])
def test_fake_shapes(fmt):
    with FakeTensorMode():
        out = few_token_moe(*_operands(fmt, device="cuda"), 2, "silu")
        assert out.shape == (3, 256) and out.dtype == torch.bfloat16
        with pytest.raises(ValueError, match="router logits"):
            a = _operands(fmt, device="cuda")
            few_token_moe(a[0], a[1][:2], *a[2:], 2, "silu")


def test_refusals():
    call = lambda a, k=2, act="silu", **kw: few_token_moe(*a, k, act, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="device tensors"):
        call(_operands())
    with pytest.raises(NotImplementedError, match="weight format"):
        call(_operands(), weight_format="fp8_block")
    with pytest.raises(NotImplementedError, match="scoring function"):
        call(_operands(), scoring_func="tanh")
    with pytest.raises(NotImplementedError, match="activation"):
        call(_operands(), act="relu")
    with pytest.raises(ValueError, match="activation is required"):
        call(_operands(), act=None)
    with pytest.raises(ValueError, match="tokens"):
        call(_operands(T=17))
    with pytest.raises(ValueError, match="tokens"):
        call(_operands(T=16, E=16), k=9)
    with pytest.raises(ValueError, match="tokens"):
        call(_operands(), k=9)
    a = _operands()
    with pytest.raises(ValueError, match="bf16"):
        call([a[0].float()] + a[1:])
    with pytest.raises(ValueError, match="inconsistent"):
        call(a[:3] + [a[3][:, :-1]] + a[4:])
    with pytest.raises(ValueError, match="contiguous"):
        call(a[:2] + [a[2].transpose(0, 1).contiguous().transpose(0, 1)] + a[3:], weight_format="mxfp4")
    with pytest.raises(ValueError, match="w2_scale"):
        call(a[:5] + [a[5][..., :-1]] + a[6:], weight_format="mxfp4")
    with pytest.raises(ValueError, match="w1_scale"):
        call(a[:4] + [None] + a[5:], weight_format="mxfp4")
    with pytest.raises(ValueError, match="no scales"):
        b = _operands("bf16")
        call(b[:4] + [torch.zeros(1), None] + b[6:], weight_format="bf16")
    with pytest.raises(ValueError, match="w1_bias"):
        call(a[:6] + [torch.zeros(8, 3), None])
    with pytest.raises(ValueError, match="multiples of 32"):
        call(_operands("bf16", H=40))
    with pytest.raises(ValueError, match="group"):
        b = _operands("int4")
        call(b[:4] + [b[4][..., :3]] + b[5:], weight_format="int4")
    with pytest.raises(ValueError, match="correction bias"):
        call(a, e_score_correction_bias=torch.zeros(7))


def _desc(**kw):
    d = _capi.FewDesc()
    for name in ("x", "router_logits", "w1", "w2", "w1_scale", "w2_scale", "out"):
        setattr(d, name, 0x1000)
    d.T, d.H, d.I, d.E, d.topk, d.ldx, d.ldo = 4, 256, 128, 16, 2, 256, 256
    d.num_group = d.topk_group = 1
    d.act = _capi.ACT_SILU
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_entry_points_check_the_descriptor():
    lib, n, a = _capi.lib, ctypes.c_int64(0), ctypes.c_void_p(0x1000)
    size = lambda **kw: lib.qmoe_moe_few_workspace_size(ctypes.byref(_desc(**kw)), ctypes.byref(n))  # noqa: E731
    assert size() == 0 and n.value >= 4 * 2 * 128 * 2
    for bad in (dict(format=5), dict(format=-1), dict(T=0), dict(T=17), dict(E=513), dict(topk=0), dict(topk=17), dict(H=48),
                dict(I=40), dict(ldx=255), dict(ldx=252), dict(ldo=255), dict(ldo=258), dict(act=0), dict(act=6), dict(scoring=4),
                dict(T=16, topk=9), dict(num_group=3, topk_group=1), dict(format=2, group=0), dict(format=2, group=128, H=192),
                dict(format=3, H=160)):
        assert size(**bad) == 1, bad
    assert lib.qmoe_moe_few_workspace_size(None, ctypes.byref(n)) == 1
    call = lambda ws=a, nbytes=1 << 20, **kw: lib.qmoe_moe_few(ctypes.byref(_desc(**kw)), ws, nbytes, None)  # noqa: E731
    assert call(ws=None) == 2 and call(nbytes=16) == 2
    for bad in (dict(x=None), dict(router_logits=None), dict(out=None), dict(w1_scale=None), dict(x=0x1008), dict(w2=0x1008),
                dict(out=0x1004), dict(w1_scale=0x1002), dict(format=4)):
        assert call(**bad) == 1, bad


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_descriptor_layout_matches_c(tmp_path):
    fields = [f[0] for f in _capi.FewDesc._fields_]
    lines = ['printf("size %zu\\n", sizeof(qmoe_moe_few_desc));']
    lines += [f'printf("{f} %zu\\n", offsetof(qmoe_moe_few_desc, {f}));' for f in fields]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "qmoe.h"\nint main(void) {\n' + "\n".join(lines) +
                   "\nreturn 0;\n}\n")
    include = os.path.join(os.path.dirname(__file__), os.pardir, "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "layout")], check=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True,
                                                       text=True).stdout.splitlines())
    assert int(out["size"]) == ctypes.sizeof(_capi.FewDesc)
    assert all(int(out[f]) == getattr(_capi.FewDesc, f).offset for f in fields)


def test_which_steps_it_takes():
    assert ops.few_token_moe_takes(16, 8, "mxfp4") and ops.few_token_moe_takes(1, 64, "bf16")
    assert not ops.few_token_moe_takes(17, 1, "mxfp4") and not ops.few_token_moe_takes(16, 9, "mxfp4")
    assert not ops.few_token_moe_takes(1, 1, "fp8")


def test_takes_only_sizes_that_it_has():
    """What `moe_forward` asks before it leaves its other paths."""
    z = lambda *s: torch.empty(s, dtype=torch.uint8, device="meta")  # noqa: E731
    takes = ops.few_token_moe_takes
    assert takes(4, 2, "mxfp4", z(8, 256, 64)) and takes(4, 2, "nvfp4", z(8, 96, 16))
    assert not takes(4, 2, "mxfp4", z(8, 256, 24)) and not takes(4, 2, "bf16", z(8, 80, 64))
    assert not takes(4, 2, "mxfp4", z(513, 256, 64)) and not takes(4, 2, "bf16", z(1, 65568, 32))
    assert takes(4, 2, "fp8_w8a16", z(8, 256, 128)) and not takes(4, 2, "fp8_w8a16", z(8, 256, 64))
    assert takes(4, 2, "int4", z(8, 128, 32), z(8, 128, 4)) and not takes(4, 2, "int4", z(8, 128, 18), z(8, 128, 3))
    assert takes(4, 2, "int4", z(8, 128, 32), z(8, 128, 2)) and not takes(4, 2, "int4", z(8, 96, 32), z(8, 96, 2))
    assert not takes(4, 2, "int4", z(8, 128, 32), z(8, 128, 16))


def test_a_gradient_asked_of_it_is_an_error():
    """It has no backward pass: the output says so instead of dropping the path."""
    with FakeTensorMode():
        a = _operands(device="cuda")
        a[0].requires_grad_()
        out = few_token_moe(*a, 2, "silu")
        assert out.requires_grad
        with torch.no_grad():
            assert not few_token_moe(*a, 2, "silu").requires_grad


@pytest.mark.parametrize("T,topk,switch,takes", [(1, 4, 16, True), (8, 8, 16, True), (9, 8, 16, True), (16, 8, 16, True),
                                                 (16, 9, 16, False), (9, 8, 8, False), (9, 8, 0, False), (17, 1, 64, False)])
def test_which_steps_of_a_method_take_it(monkeypatch, T, topk, switch, takes):
    """Every step that the layer has a form for, up to the switch's tokens,
    whatever the route + dispatch launch of the other path holds."""
    from types import SimpleNamespace

    from qmoe.layers import fused_moe, moe_routing

    called = []
    monkeypatch.setenv("QMOE_FEW_TOKEN_MOE", str(switch))
    monkeypatch.setattr(fused_moe, "few_token_moe", lambda *a, **k: called.append("few"))
    monkeypatch.setattr(fused_moe, "fused_moe_gmm", lambda *a, **k: called.append("other"))
    monkeypatch.setattr(moe_routing, "route", lambda *a, **k: (None, None))
    layer = SimpleNamespace(moe_config=SimpleNamespace(experts_per_token=topk), _qmoe_activation="silu",
                            scoring_func="softmax", renormalize=True)
    a = _operands("bf16", T=T, E=16)
    run = lambda ly, x: fused_moe.moe_forward(ly, x, *a[1:], "bf16")  # noqa: E731
    with FakeTensorMode(allow_non_fake_inputs=True):
        run(layer, a[0])
        assert (called == ["few"]) == takes
        del called[:]
        # a model's own routing function, other activations: never
        layer.custom_routing_function = lambda *x, **k: None
        run(layer, a[0])
        del layer.custom_routing_function
        run(layer, a[0].float())
        assert called == ["other", "other"]
