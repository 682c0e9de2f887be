"""Norms around a block of the longest rows whose two vectors lie in LDS (8192 values,
16 wavefronts a row in the gradient) and of their neighbours, with the float32 bounds
of the block's other tests: a row's mean terms are about 1 / sqrt(H) of a gradient, far
above them."""

import pytest
import torch

from qmoe.layers.block import block_norm
from test_gpu_block_norm import BF16, E, F16, F32, NAMES, _check, _operands, _rand, _run

pytestmark = pytest.mark.gpu

# (8190, 8191: rows that are not read 16 bytes at a time)
ROWS = [(3, 8184), (3, 8192), (2, 8190), (5, 8191), (2, 8200), (600, 8192)]


@pytest.mark.parametrize("T,H", ROWS)
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("yt,rt,wt", [(F32, F32, F32), (BF16, F32, F32), (F16, F16, F16)])
def test_gradients_of_the_longest_rows(dev, T, H, gate, yt, rt, wt):
    print(f"rows T={T} H={H} gate={gate} {yt} {rt} {wt}", flush=True)
    for post, nxt in ((True, True), (True, False), (False, True)):
        ts = _operands(dev, T, H, yt, rt, wt, gate, post, nxt, T + H)
        out, grads = _run(T, H, ts, 0.5, -1.25, 1.0, nxt)
        assert [n for n in NAMES if grads[n] is not None] == [n for n, t in zip(NAMES, ts) if t is not None]
        _check(*ts, 0.5, -1.25, 1.0, out[0].detach(), out[1].detach() if nxt else None, grads)


@pytest.mark.parametrize("T,H", ROWS)
@pytest.mark.parametrize("xt,zt", [(F32, F32), (F32, BF16), (F16, F16)])
def test_norm_alone_of_the_longest_rows(dev, T, H, xt, zt):
    g = torch.Generator(device=dev).manual_seed(H)
    x, w, gz = _rand(g, (T, H), xt, 3.0), _rand(g, (H,), F32, 0.1), _rand(g, (T, H), zt)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    z = block_norm(a, b, E, 1.0, zt)
    dx, dw = torch.autograd.grad(z, (a, b), gz)
    _check(torch.zeros_like(x).to(zt), x, None, None, w, None, gz, 1.0, 1.0, 1.0, x, z.detach(),
           {"residual": dx, "next": dw})
