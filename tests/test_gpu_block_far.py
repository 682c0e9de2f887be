"""Block operators on tensors of more than 2^31 values: places beyond 32 bits. The last
rows of a long call equal those of a call of their own, bit for bit where a row does
not depend on how many there are."""

import pytest
import torch

from qmoe import ops
from qmoe.layers.block import block_residual, checkpointed_activation, checkpointed_linear
from qmoe.layers.moe_routing import balanced_experts

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
LAST = 61


@pytest.fixture(autouse=True)
def dev():
    yield torch.device("cuda:0")
    torch.cuda.empty_cache()


def _rows(T, n, dev, std=1.0):
    return torch.empty((T, n), dtype=BF16, device=dev).normal_(0, std)


def test_block(dev):
    T, H = (1 << 19) + LAST, 4104
    assert T * H > 1 << 31
    y, gh = _rows(T, H, dev), _rows(T, H, dev)
    w = torch.ones(H, dtype=BF16, device=dev)

    def run(y, gh):
        leaf = y.detach().requires_grad_()
        h, z = block_residual(leaf, y, norm_weight=w, next_weight=w)
        return h.detach(), z.detach(), *torch.autograd.grad((h, z), leaf, (gh, gh))

    far, near = run(y, gh), run(y[-LAST:].clone(), gh[-LAST:].clone())
    for a, b in zip(far, near):
        assert torch.equal(a[-LAST:], b)


def test_activation(dev):
    T, I = (1 << 19) + LAST, 2056
    assert T * 2 * I > 1 << 31
    x, dh = _rows(T, 2 * I, dev), _rows(T, I, dev)

    def run(x, dh):
        leaf = x.detach().requires_grad_()
        h = checkpointed_activation(leaf)
        return h.detach(), *torch.autograd.grad(h, leaf, dh)

    far, near = run(x, dh), run(x[-LAST:].clone(), dh[-LAST:].clone())
    for a, b in zip(far, near):
        assert torch.equal(a[-LAST:], b)


def test_linear(dev):
    """dy is zero but for the last rows, so that dw is theirs; sums of up to 2080 products
    in float32, one rounding to bf16"""
    T, K, N = 1 << 20, 2080, 2072
    assert T * N > 1 << 31
    x, w = _rows(T, K, dev), _rows(N, K, dev, 0.02)
    dy = torch.zeros((T, N), dtype=BF16, device=dev)
    dy[-LAST:].normal_()
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = checkpointed_linear(a, b)
    dx, dw = torch.autograd.grad(y, (a, b), dy)
    _, codes, scales = ops.linear_checkpoint(x[-LAST:].clone(), w)
    x8 = codes.view(torch.float8_e4m3fn).to(F64).view(LAST, K // 32, 32) * torch.exp2(scales.to(F64) - 127)[..., None]
    g, xl, x8, w = dy[-LAST:].to(F64), x[-LAST:].to(F64), x8.view(LAST, K), w.to(F64)
    for got, p, q in ((y[-LAST:], xl, w.t()), (dx[-LAST:], g, w), (dw, g.t(), x8)):
        ref, mag = p @ q, p.abs() @ q.abs()
        assert ((got.to(F64) - ref).abs() <= 2.0 ** -8 * ref.abs() + 2080 * 2.0 ** -24 * mag).all()
    assert not dx[:-LAST].any()


# more tiles than CUs, with ragged ends: of 256 and of 192 rows along K, across it in the
# input's gradient, and in the weight's; then each tile where K is short or long for it
@pytest.mark.parametrize("T,K,N,bias", [(4072, 512, 4104, True), (3000, 512, 8200, False), (3000, 512, 8200, True),
                                        (4072, 4128, 512, False), (3000, 8224, 512, True), (2048, 5152, 5128, False),
                                        (250, 96, 28680, True), (4070, 28672, 72, True), (777, 96, 14344, True),
                                        (777, 14368, 72, False), (3000, 28640, 72, False), (3000, 96, 28680, False),
                                        (4070, 96, 28680, True), (4070, 64, 28672, False)])
def test_linear_of_many_tiles(dev, T, K, N, bias):
    """sums of K, N and T products in float32, one rounding to bf16; what is read behind
    each matrix is its own, so that a wrong place shows"""
    g = torch.Generator(device=dev).manual_seed(T + K + N)
    x, dy = (torch.randn((T, n), generator=g, device=dev).to(BF16) for n in (K, N))
    w = (0.05 * torch.randn((N, K), generator=g, device=dev)).to(BF16)
    b = torch.randn(N, generator=g, device=dev) if bias else None
    leaves = [t.detach().requires_grad_() for t in ((x, w, b) if bias else (x, w))]
    y = checkpointed_linear(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    _, codes, scales = ops.linear_checkpoint(x, w)
    x8 = (codes.view(torch.float8_e4m3fn).to(F64).view(T, K // 32, 32) * torch.exp2(scales.to(F64) - 127)[..., None]).view(T, K)
    gd, xd, wd = dy.to(F64), x.to(F64), w.to(F64)
    for got, p, q, n, plus in ((y.detach(), xd, wd.t(), K, b), (grads[0], gd, wd, N, None), (grads[1], gd.t(), x8, T, None)):
        ref, mag = p @ q, p.abs() @ q.abs()
        if plus is not None:
            ref, mag = ref + plus, mag + plus.abs()
        assert ((got.to(F64) - ref).abs() <= 2.0 ** -8 * ref.abs() + (n + 8) * 2.0 ** -24 * mag).all()
    for g1, g2 in zip(grads, torch.autograd.grad(checkpointed_linear(*leaves), leaves, dy)):
        assert torch.equal(g1, g2)


def test_balance(dev):
    T, E, k = (1 << 23) + LAST, 264, 4
    assert T * E > 1 << 31
    x = _rows(T, E, dev)
    gw = torch.empty((T, k), device=dev).normal_()

    def run(x, gw):
        leaf = x.detach().requires_grad_()
        w, ids, _, counts = balanced_experts(leaf, k, "sigmoid")
        return w.detach(), ids, *torch.autograd.grad(w, leaf, gw), counts

    far, near = run(x, gw), run(x[-LAST:].clone(), gw[-LAST:].clone())
    for a, b in zip(far[:3], near[:3]):
        assert torch.equal(a[-LAST:], b)
    assert torch.equal(far[3], torch.bincount(far[1].flatten(), minlength=E).int())
