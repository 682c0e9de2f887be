"""Block operators at the ends of their ranges: more rows than a launch's first axis
takes, the longest rows whose vectors lie in LDS, gates without a workspace. Rows do
not depend on one another, so the last rows of a long call equal those of a call of
their own, bit for bit."""

import pytest
import torch

from qmoe import ops
from qmoe.layers.block import block_norm, block_residual, checkpointed_activation, checkpointed_linear

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
MANY = (1 << 17) + 5  # workgroups of one row: three times the launch's first axis


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _pieces(T):
    """rows around the seams of the launch"""
    return [slice(0, 3), slice((1 << 16) - 2, (1 << 16) + 2), slice((1 << 17) - 2, T)]


def test_norms_of_many_rows(dev):
    H = 520  # two wavefronts: four rows of a workgroup
    T = MANY * 4
    x = torch.randn((T, H), device=dev).to(BF16)
    w = torch.randn(H, device=dev)
    z = block_norm(x, w)
    h, n = block_residual(x, x, norm_weight=w, next_weight=w, scale=0.5)
    for s in [slice(4 * s.start, 4 * s.stop if s.stop != MANY else T) for s in _pieces(MANY)]:
        assert torch.equal(z[s], block_norm(x[s], w))
        h1, n1 = block_residual(x[s], x[s], norm_weight=w, next_weight=w, scale=0.5)
        assert torch.equal(h[s], h1) and torch.equal(n[s], n1)


def test_activation_of_many_rows(dev):
    x = (2 * torch.randn((MANY, 40), device=dev)).to(BF16)
    dh = torch.randn((MANY, 20), device=dev).to(BF16)
    leaf = x.clone().requires_grad_()
    h = checkpointed_activation(leaf)
    (dx,) = torch.autograd.grad(h, leaf, dh)
    _, codes, scales = ops.act_checkpoint(x, "silu")
    for s in _pieces(MANY):
        part = x[s].clone().requires_grad_()
        h1 = checkpointed_activation(part)
        (dx1,) = torch.autograd.grad(h1, part, dh[s])
        assert torch.equal(h[s], h1) and torch.equal(dx[s], dx1)
        _, c1, s1 = ops.act_checkpoint(x[s], "silu")
        assert torch.equal(codes[s], c1) and torch.equal(scales[s], s1)


def test_eight_bits_of_many_rows(dev):
    x = torch.randn((MANY, 32), device=dev).to(BF16)
    w = torch.randn((8, 32), device=dev).to(BF16)
    y, codes, scales = ops.linear_checkpoint(x, w)
    for s in _pieces(MANY):
        _, c1, s1 = ops.linear_checkpoint(x[s], w)
        assert torch.equal(codes[s], c1) and torch.equal(scales[s], s1)
    assert torch.equal(y, checkpointed_linear(x, w))


@pytest.mark.parametrize("H", [8184, 8192, 8200])
def test_longest_rows_in_shared_memory(dev, H):
    """gradients of rows whose two vectors fill 64 KB, and of the first that do not lie
    there, against float64"""
    T = 3
    g = torch.Generator(device=dev).manual_seed(H)
    y, r = (torch.randn((T, H), generator=g, device=dev).to(BF16) for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, generator=g, device=dev)).to(BF16)
    gh, gz = (torch.randn((T, H), generator=g, device=dev).to(BF16) for _ in range(2))

    def run(h, z, leaves):
        return torch.autograd.grad((h, z), leaves, (gh, gz))

    a = [t.clone().requires_grad_() for t in (y, r, w)]
    got = run(*block_residual(a[0], a[1], norm_weight=a[2], next_weight=a[2]), a)
    b = [t.double().requires_grad_() for t in (y, r, w)]
    n = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    h = b[1] + n(b[0]) * b[2]
    want = torch.autograd.grad((h, n(h) * b[2]), b, (gh.double(), gz.double()))
    for name, p, q in zip(("y", "residual", "weights"), got, want):
        # h is rounded to bf16 before its norm (half a step, 2^-9 of it: n(h) and with it the
        # gradient move by as much of the row's largest terms), and the result once more; the
        # weights' two parts are rounded and added in bf16
        lim = 2.0 ** -7 * (q.abs() + q.abs().amax())
        assert ((p.double() - q).abs() <= lim).all(), name


def test_gates_of_rows_alone(dev):
    """their gradient comes from the rows' own launch, without a workspace"""
    T, H = 6, 64
    y, r = torch.randn((T, H), device=dev), torch.randn((T, H), device=dev)
    for gate in (torch.randn((T, 1), device=dev), torch.randn((T, H), device=dev)):
        leaf = gate.clone().requires_grad_()
        h = block_residual(y, r, gate=leaf)
        (dg,) = torch.autograd.grad(h, leaf, r)
        want = (r * y).double()
        want = want.sum(-1, keepdim=True) if gate.shape[-1] == 1 else want
        # 64 products and their sum in float32
        lim = 2.0 ** -24 * 70 * (r * y).abs().double().sum(-1, keepdim=True)
        assert ((dg.double() - want).abs() <= lim).all()
