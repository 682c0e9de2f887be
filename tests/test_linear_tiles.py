"""The tiles of the linear layer and its gradients, each by sizes that take it (the
plans are checked without a GPU).

Exact cases: x, w, dy and the bias are small whole numbers, x's so small that 8 bits
hold them, so that every sum of products is a whole number below 2^24, which float32
holds in any order, and so are the sums of the slices. The results have to be the
correctly rounded ones, bit for bit: a k, row, column, stage or slice that is lost or
taken twice changes them, however long the sum is."""

import math
import random

import pytest
import torch

from qmoe import ops
from qmoe.layers.block import checkpointed_linear

BF16, F32, D = torch.bfloat16, torch.float32, torch.float64

# (T, K, N), each for what it adds to `_forms` of those before it; long sums last
CASES = [(73, 6016, 1072), (320, 736, 11184), (512, 4096, 4096), (777, 4096, 4096), (7015, 704, 18728), (1, 32, 8),
         (65, 64, 64), (64, 96, 72), (134, 128, 144), (576, 896, 128), (1, 5088, 784), (17273, 288, 8), (18304, 32, 272),
         (16, 672, 704), (5177, 32, 4864), (395, 64, 16600), (6365, 1824, 8), (17091, 288, 296), (6550, 2112, 536),
         (17183, 384, 320), (16448, 64, 2712), (391, 288, 23344), (64, 32, 17600), (832, 320, 13232), (19099, 1728, 64),
         (1472, 96, 20288), (16453, 2080, 64), (5642, 640, 5632), (640, 416, 24328), (17166, 288, 72), (16511, 96, 272),
         (12629, 800, 72), (17268, 544, 128), (17616, 128, 560), (16962, 544, 168), (13658, 1088, 128), (7182, 1568, 256),
         (7612, 3232, 256), (1792, 608, 11560), (79, 12608, 22024), (9344, 544, 3624), (219, 3744, 21128), (1920, 7776, 3376),
         (610, 3392, 24448), (300, 28672, 264), (300, 256, 28680), (70000, 64, 72), (4070, 28672, 72)]


def _cdiv(a, b):
    return -(-a // b)


def _forms(T, K, N):
    """(product, tile, in slices, the axis ends inside a stage, codes, tiles go on in one
    workgroup, whole stages of a slice: 0, 1 or more) of the three products"""
    p, forms = ops.linear_plan(T, N, K), set()
    for name, na, nb, k in (("y", N, T, K), ("dx", K, T, N), ("dw", K, N, T)):
        tile, slices = p[name], p[name + "_slices"]
        tiles = _cdiv(na, 256) * _cdiv(nb, 128 if tile == 1 else tile)
        on = tile >= 192 and slices == 1 and k % 64 == 0 and k > 64 and tiles > 256
        per = _cdiv(_cdiv(k, 64), slices) * 64 if slices > 1 else k
        forms.add((name, tile, slices > 1, k % 64 != 0, name == "dw" and bool(p["dw_codes"]), on, min(per // 64, 2)))
    return forms


def test_the_cases_take_every_form():
    """... that any of 100000 random sizes takes."""
    rng, seen = random.Random(1), set()
    size = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    for _ in range(100000):
        K, N, T = 32 * size(1, 480), 8 * size(1, 4000), size(1, 20000)
        if T * N * K + 300 * (T * N + N * K + T * K) < 118 * 10 ** 9:
            seen |= _forms(T, K, N)
    covered = set().union(*(_forms(*c) for c in CASES))
    assert len(seen) > 80 and not seen - covered
    # codes multiplied as they are: from part of a stage to many of them
    assert {min(T // 64, 5) for T, K, N in CASES if ops.linear_plan(T, N, K)["dw_codes"]} >= {0, 1, 5}


@pytest.mark.parametrize("T,N,K,want", [
    (4096, 28672, 4096, dict(y=256, y_slices=1, dx=256, dx_slices=1, dw=256, dw_slices=1, dw_codes=0)),
    (777, 4096, 4096, dict(y=64, y_slices=1, dx=64, dx_slices=1, dw=1, dw_slices=1, dw_codes=0)),
    (512, 4096, 4096, dict(dw=1, dw_slices=1, dw_codes=1)),
    (513, 4096, 4096, dict(dw=1, dw_codes=0)),  # codes up to 512 tokens only
    (19, 2048, 2048, dict(dw_codes=0)),         # ... and in the tiles without a ring only
])
def test_plans(T, N, K, want):
    plan = ops.linear_plan(T, N, K)
    assert {name: plan[name] for name in want} == want


def test_plans_of_wrong_sizes():
    for bad in ((0, 8, 32), (1, 0, 32), (1, 12, 32), (1, 8, 40), (1, 8, 1 << 17)):
        with pytest.raises(RuntimeError, match="invalid argument"):
            ops.linear_plan(*bad)


def _rounded(v, dtype=BF16):
    assert v.abs().max() < 1 << 24 and torch.equal(v, v.round())
    return v.to(F32).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N", CASES)
def test_exact_sums(dev, T, K, N):
    print(f"exact T={T} K={K} N={N}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(T + K + N)
    ints = lambda hi, *s: torch.randint(-hi, hi + 1, s, generator=gen, device=dev).to(BF16)  # noqa: E731
    x, w, dy, b = ints(3, T, K), ints(3, N, K), ints(3, T, N), ints(100, N).to(F32)
    leaves = [t.requires_grad_() for t in ((x, w, b) if (T + N // 8) % 2 else (x, w))]
    y = checkpointed_linear(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    xd, wd, gd = (t.detach().to(D) for t in (x, w, dy))
    ref = xd @ wd.t()
    assert torch.equal(y.detach(), _rounded(ref + b.detach().to(D) if len(leaves) == 3 else ref))
    assert torch.equal(grads[0], _rounded(gd @ wd))
    assert torch.equal(grads[1], _rounded(gd.t() @ xd))
    if len(leaves) == 3:
        assert torch.equal(grads[2], _rounded(gd.sum(0), F32))
