"""Refusals, fake shapes and the C ABI's argument checks of the block operators and
the balanced router, without a GPU: nothing here launches a kernel."""

import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode

from qmoe import _capi, ops
from qmoe.layers.block import block_norm, block_residual, checkpointed_activation, checkpointed_linear
from qmoe.layers.moe_routing import balanced_experts

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_structures_match_the_header():
    src = open(os.path.join(ROOT, "include", "qmoe.h")).read()
    for name, cls in (("qmoe_block_desc", _capi.BlockDesc), ("qmoe_block_grads", _capi.BlockGrads)):
        body = src[src.index("typedef struct " + name):src.index("} " + name + ";")].split("{", 1)[1]
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [part.replace("*", " ").split()[-1] for decl in body.split(";") if decl.strip()
                  for part in decl.split(",")]
        assert [f for f, _ in cls._fields_] == fields


def test_cpu_tensors_are_refused():
    x, w = torch.zeros((4, 32), dtype=BF16), torch.ones(32, dtype=BF16)
    for call in (lambda: block_norm(x, w), lambda: block_residual(x, x), lambda: checkpointed_activation(x),
                 lambda: checkpointed_linear(x, torch.zeros((8, 32), dtype=BF16)), lambda: balanced_experts(x, 2)):
        with pytest.raises(ValueError, match="device tensors"):
            call()
        with torch.enable_grad():
            x.requires_grad_()
            with pytest.raises(ValueError, match="device tensors"):
                call()
            x = x.detach()


@pytest.mark.parametrize("call,match", [
    (lambda: block_residual(torch.zeros(2, 8), torch.zeros(2, 9)), "a residual of"),
    (lambda: block_residual(torch.zeros(2, 8), torch.zeros(2, 8, dtype=BF16)), "a residual of"),
    (lambda: block_residual(torch.zeros(2, 8).double(), torch.zeros(2, 8)), "a residual of"),
    (lambda: block_residual(torch.zeros(2, 8), torch.zeros(2, 8), gate=torch.zeros(2)), "the gate"),
    (lambda: block_residual(torch.zeros(2, 8), torch.zeros(2, 8), gate=torch.zeros(2, 8, dtype=BF16)), "a gate per element"),
    (lambda: block_residual(torch.zeros(2, 8), torch.zeros(2, 8), gate=torch.zeros(1, 8)), "the gate"),
    (lambda: block_residual(torch.zeros(2, 8), torch.zeros(2, 8), norm_weight=torch.zeros(7)), "norm_weight"),
    (lambda: block_residual(torch.zeros(2, 8), torch.zeros(2, 8), norm_weight=torch.zeros(8),
                            next_weight=torch.zeros(8, dtype=BF16)), "one type"),
    (lambda: block_residual(None, torch.zeros(2, 8)), "the block's output"),
    (lambda: block_residual(torch.zeros(2, 16385), torch.zeros(2, 16385)), "rows of 1 to"),
    (lambda: block_residual(torch.zeros(()), torch.zeros(())), "rows must be"),
    (lambda: block_norm(torch.zeros(2, 0), torch.zeros(0)), "rows of 1 to"),
    (lambda: block_norm(torch.zeros(2, 8), None), "a weight"),
    (lambda: block_norm(torch.zeros(2, 8, dtype=BF16), torch.zeros(8), out_dtype=F16), "a residual of"),
    (lambda: block_norm(torch.zeros(2, 8, dtype=torch.int32), torch.zeros(8)), "rows must be"),
    (lambda: checkpointed_activation(torch.zeros(2, 8)), "bf16 or f16"),
    (lambda: checkpointed_activation(torch.zeros(2, 7, dtype=BF16)), "takes"),
    (lambda: checkpointed_activation(torch.zeros((), dtype=BF16)), "takes"),
    (lambda: checkpointed_activation(torch.zeros(2, 8, dtype=BF16), None), "a gate / up activation"),
    (lambda: checkpointed_linear(torch.zeros(2, 32), torch.zeros(8, 32)), "bf16"),
    (lambda: checkpointed_linear(torch.zeros(2, 32, dtype=BF16), torch.zeros(8, 64, dtype=BF16)), "bf16"),
    (lambda: checkpointed_linear(torch.zeros(2, 40, dtype=BF16), torch.zeros(8, 40, dtype=BF16)), "multiples of 32"),
    (lambda: checkpointed_linear(torch.zeros(2, 32, dtype=BF16), torch.zeros(9, 32, dtype=BF16)), "multiples of 8"),
    (lambda: checkpointed_linear(torch.zeros(2, 32, dtype=BF16), torch.zeros(32, 8, dtype=BF16).t()), "rows must be"),
    (lambda: checkpointed_linear(torch.zeros(2, 32, dtype=BF16), torch.zeros(8, 32, dtype=BF16), torch.zeros(7)), "bias"),
    (lambda: checkpointed_linear(torch.zeros(2, 32, dtype=BF16), torch.zeros(8, 32, dtype=BF16),
                                 torch.zeros(8, dtype=F16)), "bias"),
    (lambda: balanced_experts(torch.zeros(2, 3, 4), 2), "router logits"),
    (lambda: balanced_experts(torch.zeros(2, 4, dtype=torch.int32), 2), "router logits"),
    (lambda: balanced_experts(torch.zeros(2, 4), 5), "topk"),
    (lambda: balanced_experts(torch.zeros(2, 4), 0), "topk"),
    (lambda: balanced_experts(torch.zeros(2, 513), 2), "experts"),
    (lambda: balanced_experts(torch.zeros(2, 10), 2, num_expert_group=4, topk_group=2), "groups"),
    (lambda: balanced_experts(torch.zeros(2, 8), 5, num_expert_group=4, topk_group=2), "groups"),
    (lambda: balanced_experts(torch.zeros(2, 8), 2, token_mask=torch.zeros(3, dtype=torch.bool)), "token mask"),
    (lambda: balanced_experts(torch.zeros(2, 8), 2, token_mask=torch.zeros(2)), "token mask"),
    (lambda: balanced_experts(torch.zeros(2, 8), 2, e_score_correction_bias=torch.zeros(7)), "correction bias"),
])
def test_bad_arguments(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_what_is_not_there():
    with pytest.raises(NotImplementedError, match="scores"):
        balanced_experts(torch.zeros(2, 8), 2, "none")
    with pytest.raises(NotImplementedError, match="activation"):
        checkpointed_activation(torch.zeros(2, 8, dtype=BF16), "relu")
    b = torch.zeros(8, requires_grad=True)
    with pytest.raises(NotImplementedError, match="only chooses"):
        balanced_experts(torch.zeros(2, 8), 2, e_score_correction_bias=b)
    with fw.dual_level():
        x = fw.make_dual(torch.zeros(2, 32), torch.ones(2, 32))
        for call in (lambda: block_norm(x, torch.ones(32)), lambda: block_residual(x, x), lambda: balanced_experts(x, 2),
                     lambda: checkpointed_activation(fw.make_dual(torch.zeros(2, 32, dtype=BF16),
                                                                  torch.zeros(2, 32, dtype=BF16))),
                     lambda: checkpointed_linear(fw.make_dual(torch.zeros(2, 32, dtype=BF16),
                                                              torch.zeros(2, 32, dtype=BF16)),
                                                 torch.zeros(8, 32, dtype=BF16))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_fake_shapes():
    with FakeTensorMode():
        dev = "cpu"
        y, r = torch.empty((3, 5, 64), dtype=BF16, device=dev), torch.empty((3, 5, 64), device=dev)
        w = torch.empty(64, device=dev)
        h, z = block_residual(y, r, gate=w, norm_weight=w, next_weight=w)
        assert h.shape == z.shape == r.shape and h.dtype == F32 and z.dtype == BF16
        assert block_residual(y, y).dtype == BF16
        assert block_norm(r, w, out_dtype=F16).dtype == F16
        assert checkpointed_activation(y).shape == (3, 5, 32)
        lin = torch.empty((24, 64), dtype=BF16, device=dev)
        assert checkpointed_linear(y, lin).shape == (3, 5, 24)
        tw, ids, loss, counts = balanced_experts(r[0], 4)
        assert tw.shape == ids.shape == (5, 4) and loss.shape == () and counts.shape == (64,) and ids.dtype == torch.int32
        leaves = [t.detach().requires_grad_() for t in (y, r, w, lin)]
        h, z = block_residual(leaves[0], leaves[1], leaves[2], leaves[2], leaves[2])
        out = checkpointed_activation(checkpointed_linear(z, leaves[3]))
        tw, _, loss, _ = balanced_experts(h[0], 4)
        grads = torch.autograd.grad((out.sum(), tw.sum() + loss), leaves)
        for g, t in zip(grads, leaves):
            assert g.shape == t.shape and g.dtype == t.dtype


def test_c_arguments():
    lib, n = _capi.lib, ctypes.c_int64(0)
    at = 0x1000
    assert lib.qmoe_moe_balance_workspace_size(4, 513, ctypes.byref(n)) == 1
    assert lib.qmoe_moe_balance_workspace_size(5000, 64, ctypes.byref(n)) == 0 and n.value > 0
    args = [at, 1, 5000, 64, 4, 0, None, 1, 1.0, 1, 1, None, at, at, at, at]
    assert lib.qmoe_moe_balance(*args, at, n.value - 1, None) == 2
    assert lib.qmoe_moe_balance(*args, None, n.value, None) == 2
    for i, v in ((0, None), (2, 0), (4, 65), (5, 3), (12, None), (14, None)):
        bad = list(args)
        bad[i] = v
        assert lib.qmoe_moe_balance(*bad, at, n.value, None) == 1
    assert lib.qmoe_moe_balance_grad(at, 1, 8, 64, 4, 0, 1, 1.0, None, None, at, at, at, at, None) == 1

    def desc(**kw):
        d = _capi.BlockDesc()
        for k, v in dict(T=4, H=64, y=at, ldy=64, residual=at, ldr=64, h=at, ldh=64, z=at, ldz=64, next_weight=at,
                         residual_scale=1.0, scale=1.0, eps=1e-6, **kw).items():
            setattr(d, k, v)
        return ctypes.byref(d)

    for bad in (dict(residual_type=2), dict(y_type=1, residual_type=0), dict(gate_kind=1), dict(gate_kind=4),
                dict(gate_kind=3, gate=at, ldg=64, gate_type=1), dict(weight_type=3)):
        assert lib.qmoe_block_residual(desc(**bad), None) == 1
    for k, v in (("T", 0), ("H", 16385), ("ldy", 63), ("ldh", 63), ("ldr", 63), ("ldz", 63), ("h", None), ("z", None),
                 ("residual", None)):
        d = desc()._obj
        setattr(d, k, v)
        assert lib.qmoe_block_residual(ctypes.byref(d), None) == 1, k
    g = _capi.BlockGrads()
    assert lib.qmoe_block_residual_grad(desc(), ctypes.byref(g), None, 0, None) == 1
    g.g_h, g.ldgh, g.g_z, g.ldgz, g.d_next_weight = at, 64, at, 64, at
    assert lib.qmoe_block_residual_grad(desc(), ctypes.byref(g), None, 0, None) == 1  # no row factors
    assert lib.qmoe_block_residual_grad(desc(rstd_h=at), ctypes.byref(g), None, 0, None) == 2
    act = [at, 64, 0, 4, 32, 1, 0.0, 0.0, at, 32, at, at]
    for i, v in ((0, None), (1, 63), (2, 1), (3, 0), (4, 0), (5, 0), (5, 6), (9, 31), (11, None)):
        bad = list(act)
        bad[i] = v
        assert lib.qmoe_act_checkpoint(*bad, None) == 1
    assert lib.qmoe_act_checkpoint_grad(at, at, 4, 32, 1, 0.0, 0.0, at, 31, 0, at, None) == 1
    assert lib.qmoe_pack_8bit(at, 64, 4, 36, at, at, None) == 1
    assert lib.qmoe_pack_8bit(at + 2, 64, 4, 64, at, at, None) == 1
    assert lib.qmoe_linear_grad_workspace_size(4, 20, 64, 1, 1, 1, ctypes.byref(n)) == 1
    assert lib.qmoe_linear_grad_workspace_size(100, 256, 64, 1, 1, 1, ctypes.byref(n)) == 0
    lin = [at, 256, 100, 256, 64, at, 64, at, at, at, at, at, 0]
    assert lib.qmoe_linear_grad(*lin, at, n.value - 1, None) == 2
    for i, v in ((0, None), (0, at + 8), (1, 255), (1, 260), (5, None), (6, 60), (7, None), (9, at + 4), (10, at + 8)):
        bad = list(lin)
        bad[i] = v
        assert lib.qmoe_linear_grad(*bad, at, n.value, None) == 1, i


def test_c_outputs_without_operands_and_workspaces():
    """outputs whose operand the call has not, and workspaces that the kernels' 16-byte
    accesses do not take"""
    lib, n = _capi.lib, ctypes.c_int64(0)
    at = 0x1000

    def grads(desc, **kw):
        d, g = _capi.BlockDesc(), _capi.BlockGrads()
        for k, v in dict(T=4, H=64, y=at, ldy=64, h=at, ldh=64, rstd_y=at, rstd_h=at, residual_scale=1.0, scale=1.0,
                         eps=1e-6, **desc).items():
            setattr(d, k, v)
        for k, v in dict(g_h=at, ldgh=64, **kw).items():
            setattr(g, k, v)
        return ctypes.byref(d), ctypes.byref(g)

    for desc, out in ((dict(next_weight=at, post_weight=at), dict(d_next_weight=at, d_post_weight=at)),
                      (dict(next_weight=at), dict(d_post_weight=at)), (dict(post_weight=at), dict(d_gate=at))):
        assert lib.qmoe_block_residual_grad(*grads(desc, **out), at, 1 << 20, None) == 1
    d, g = grads(dict(next_weight=at), g_z=at, ldgz=64, d_y=at)
    d._obj.y = None
    assert lib.qmoe_block_residual_grad(d, g, at, 1 << 20, None) == 1
    d, g = grads(dict(post_weight=at), d_post_weight=at)
    assert lib.qmoe_block_residual_grad(d, g, at + 8, 1 << 20, None) == 2
    assert lib.qmoe_moe_balance_workspace_size(5000, 64, ctypes.byref(n)) == 0
    assert lib.qmoe_moe_balance(at, 1, 5000, 64, 4, 0, None, 1, 1.0, 1, 1, None, at, at, at, at, at + 4, n.value, None) == 2
    assert lib.qmoe_linear_grad_workspace_size(1000, 256, 64, 1, 1, 1, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.qmoe_linear_grad(at, 256, 1000, 256, 64, at, 64, at, at, at, at, at, 0, at + 8, n.value, None) == 2


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("cname,cls", [("qmoe_block_desc", _capi.BlockDesc), ("qmoe_block_grads", _capi.BlockGrads)])
def test_structures_have_the_c_layout(tmp_path, cname, cls):
    names = [f for f, *_ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "qmoe.h"\nint main(void) {\n'
                   + f'printf("%zu", sizeof({cname}));\n'
                   + "".join(f'printf(" %zu", offsetof({cname}, {f}));\n' for f in names) + "return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in names]
