"""The tiles of the vocabulary loss, each by sizes that take it (the plans are
checked without a GPU), and pieces of the vocabulary.

Exact cases. x = [y, y] and w = [u, -u] in small integers: every logit of an
"on" row is 0, by products of every K stage that only cancel over all of them;
an "off" row's is -128 or less (one value more), so that its exponential is 0
in float32. With 1024 on rows the probabilities are exactly 2^-10, and with
gradients that are powers of two every product and sum of dx and dw is a whole
number of units that float32 holds: the results have to be the correctly rounded
ones, bit for bit. A row, token, stage or piece that is lost or taken twice
changes them.

Ordinary cases are compared in float64 with the bounds of the loss's other
tests, their table scaled by 1 / sqrt(H)."""

import math

import pytest
import torch

from qmoe import ops

BF16, E4, E5, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e5m2, torch.int8
EPS = 2.0 ** -24

# (T, V, H, table) -> (logits, probs, dx, dw, pieces of the gradients); 1: 128 rows without a ring
CASES = [
    (60, 3100, 1032, BF16, (64, 64, 64, 1, 1)),
    (100, 3001, 1088, BF16, (128, 128, 192, 1, 1)),
    (150, 33100, 264, BF16, (1, 1, 192, 1, 1)),
    (150, 33100, 1088, BF16, (192, 192, 192, 1, 1)),
    (150, 33100, 1032, BF16, (192, 192, 192, 1, 1)),  # (1032, 72, 80, 528: K ends inside a stage)
    (250, 33100, 1088, BF16, (256, 256, 256, 1, 1)),
    (250, 33100, 1032, BF16, (256, 256, 256, 1, 1)),
    (1100, 13000, 1032, BF16, (256, 256, 192, 256, 1)),
    (1100, 60001, 72, BF16, (1, 1, 192, 256, 2)),  # the second piece: 1889 rows
    (1100, 13000, 640, BF16, (1, 1, 192, 256, 1)),
]
CASES += [(T, 33100, H, dtype, (rows, 1, rows, 1, 1))
          for T, rows in ((150, 192), (250, 256)) for H in (64, 80, 528) for dtype in (E4, I8, E5)]
CASES += [(150, 33100, 72, I8, (1, 1, 192, 1, 1)), (150, 33100, 1040, I8, (192, 192, 192, 1, 1)),
          (250, 65000, 1040, E4, (256, 256, 256, 1, 2))]


def _id(c):
    return f"{c[0]}x{c[1]}x{c[2]}-{str(c[3])[6:]}"


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_plans(case):
    T, V, H, dtype, want = case
    p = ops.vocab_loss_plan(T, V, H, dtype)
    assert (p["logits"], p["probs"], p["dx"], p["dw"], p["grad_pieces"]) == want


def test_plans_of_wrong_sizes():
    for bad in ((0, 10, 8), (1, 0, 8), (1, 10, 12)):
        with pytest.raises(RuntimeError, match="invalid argument"):
            ops.vocab_loss_plan(*bad)


def _exact_case(dev, T, V, H, dtype, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    ints = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=gen, device=dev).float()  # noqa: E731
    u, y = ints(-3, 3, V, H // 2), ints(-3, 3, T, H // 2)
    y[:, 0] = 8
    on = torch.zeros(V, dtype=torch.bool, device=dev)
    on[torch.randperm(V, generator=gen, device=dev)[:1024]] = True
    w, x = torch.cat((u, -u), 1), torch.cat((y, y), 1)
    w[~on, 0], w[~on, H // 2] = 0, -32  # logit -256 times the row's scale
    s = None if dtype == BF16 else 2.0 ** ints(-1, 1, V)
    t = torch.randint(0, V, (T,), generator=gen, device=dev)
    rows = torch.nonzero(on).flatten()
    half = torch.rand(T, generator=gen, device=dev) < 0.5
    t[half] = rows[torch.randint(0, 1024, (T,), generator=gen, device=dev)][half]
    t[torch.rand(T, generator=gen, device=dev) < 0.2] = -100
    # gradients of loss, lse or both; their sum of a scored token is g, g / 2 or h
    g, h = (2.0 ** ints(-1, 1, T) * (2 * ints(0, 1, T) - 1) for _ in range(2))
    kind = torch.randint(0, 4, (T,), generator=gen, device=dev)
    g[kind == 1] = 0
    h = torch.where(kind == 2, -g / 2, torch.where(kind == 0, 0.0, h))
    h[(kind == 3) & (t != -100)] = 0
    return x.to(BF16), w.to(dtype), s, t, on, g, h


def _rounded(v):
    assert torch.equal(v.float().double(), v)  # (the sums are exact in float32)
    return v.float().to(BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_exact_sums(dev, case):
    T, V, H, dtype, _ = case
    print("exact", _id(case), flush=True)
    x, w, s, t, on, g, h = _exact_case(dev, T, V, H, dtype)
    sw = w.double() if s is None else w.double() * s.double()[:, None]
    logits = x.double() @ sw.t()
    assert (logits[:, on] == 0).all() and (logits[:, ~on] <= -128).all()
    loss, lse = ops.vocab_loss(x, w, t, s)
    # 1024 ones and nothing else are summed: the logarithm's rounding is left (and the loss's)
    assert ((lse.double() - math.log(1024)).abs() <= 4 * EPS * 7).all()
    scored = t != -100
    at = logits.gather(1, t.clamp_min(0)[:, None])[:, 0]
    off = (loss.double() - torch.where(scored, math.log(1024) - at, 0.0)).abs()
    assert (off <= 4 * EPS * 7 + EPS * (7 - at)).all()
    dx, dw = ops.vocab_loss_grad(x, w, t, lse, g, h, s, need_weight=dtype == BF16)
    gl = torch.where(scored, g, 0.0).double()
    P = torch.where(on, (gl + h.double())[:, None] / 1024, torch.zeros((), dtype=torch.float64, device=dev))
    P.scatter_add_(1, t.clamp_min(0)[:, None], -gl[:, None])
    P = P.float().to(BF16).double()
    assert torch.equal(dx, _rounded(P @ sw))
    if dtype == BF16:
        assert torch.equal(dw, _rounded(P.t() @ x.double()))
    else:
        assert dw is None


@pytest.mark.gpu
@pytest.mark.parametrize("case", [c for c in CASES if c[2] != 528], ids=_id)
def test_values(dev, case):
    from test_gpu_vocab_loss import _case, _check_grads, _reference

    T, V, H, dtype, _ = case
    print("values", _id(case), flush=True)
    x, w, s, t = _case(dev, T, V, H, dtype, seed=5, ignored=T // 5)
    if s is None:
        w = (w.float() * (20 / math.sqrt(H))).to(BF16)
    else:
        s = s * (20 / math.sqrt(H))
    t[-1] = V - 1
    loss, lse = ops.vocab_loss(x, w, t, s)
    _, _, _, _, rlse, rloss, lim, _ = _reference(x, w, s, t)
    assert ((lse.double() - rlse).abs() <= lim).all() and ((loss.double() - rloss).abs() <= 2 * lim).all()
    gen = torch.Generator(device=dev).manual_seed(2)
    g, h = torch.randn(T, generator=gen, device=dev), torch.randn(T, generator=gen, device=dev)
    dx, dw = ops.vocab_loss_grad(x, w, t, lse, g, h, s, need_weight=dtype == BF16)
    _check_grads(dx, dw, x, w, s, t, g, h)
