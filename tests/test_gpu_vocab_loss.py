"""The vocabulary loss and its gradients on the GPU against float64 (products
in float64 on the GPU).

Bounds. A logit is a float32 sum of H products of bf16 values: off by at most H
2^-24 times the sum of the products' magnitudes (`mag`), and its scaling and
exponentials by a few roundings. lse moves by at most the largest error of its
logits, plus the roundings of V terms' sum (the tiles sum 256 terms, then tiles)
and of the result. P is rounded to bf16 (half a step, eps / 2) and multiplied
with float32 sums; the gradients are rounded to bf16 once more."""

import pytest
import torch

from qmoe import ops
from qmoe.layers.quantization.fp8 import Fp8LinearMethod
from qmoe.layers.quantization.unquantized import UnquantizedLinearMethod
from qmoe.layers.vocab import embedding, vocab_cross_entropy

pytestmark = pytest.mark.gpu

BF16, E4, E5, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e5m2, torch.int8
EPS = 2.0 ** -24
HALF = torch.finfo(BF16).eps / 2


def _table(dev, V, H, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn((V, H), generator=g, device=dev) * 0.05
    if dtype == BF16:
        return w.to(BF16), None
    s = w.abs().amax(-1) / {E4: 448.0, E5: 57344.0, I8: 127.0}[dtype]
    q = w / s[:, None]
    return (q.round().clamp(-127, 127).to(I8) if dtype == I8 else q.to(dtype)), s


def _case(dev, T, V, H, dtype=BF16, seed=3, ignored=0):
    w, s = _table(dev, V, H, dtype, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    x = torch.randn((T, H), generator=g, device=dev).to(BF16)
    t = torch.randint(0, V, (T,), generator=g, device=dev)
    t[:ignored] = -100
    return x, w, s, t


def _reference(x, w, s, t):
    xd, wd = x.double(), w.double()
    if s is not None:
        wd = wd * s.double()[:, None]
    lg = xd @ wd.t()
    err = (x.shape[1] + 4) * EPS * (xd.abs() @ wd.abs().t())  # of each logit
    lse = torch.logsumexp(lg, 1)
    rows = torch.arange(x.shape[0], device=x.device)
    keep = (t >= 0) & (t < w.shape[0])
    at = torch.where(keep, lg[rows, t.clamp(0, w.shape[0] - 1)], torch.zeros_like(lse))
    loss = torch.where(keep, lse - at, torch.zeros_like(lse))
    # 16 roundings: the exponentials' arguments and values, the joins, the logarithm
    lim = err.amax(1) + (256 + 16) * EPS * (1 + lg.abs().amax(1)) + 16 * EPS * lse.abs()
    return xd, wd, lg, err, lse, loss, lim, keep


@pytest.mark.parametrize("T,V,H", [(1, 1, 8), (1, 2, 64), (1, 1000, 4096), (2, 257, 72), (3, 255, 2880), (16, 5003, 512),
                                   (17, 300, 136), (64, 1031, 256), (65, 4096, 520), (128, 777, 64), (129, 3001, 1024),
                                   (257, 2049, 328), (613, 1003, 2880), (1000, 50, 128)])
@pytest.mark.parametrize("dtype", [BF16, E4, I8, E5])
def test_loss_values(dev, T, V, H, dtype):
    print(f"loss T={T} V={V} H={H} {dtype}", flush=True)
    x, w, s, t = _case(dev, T, V, H, dtype, ignored=T // 3)
    loss, lse = vocab_cross_entropy(x, w, t, s)
    assert loss.dtype == lse.dtype == torch.float32 and loss.shape == lse.shape == (T,)
    _, _, _, _, rlse, rloss, lim, keep = _reference(x, w, s, t)
    assert ((lse.double() - rlse).abs() <= lim).all()
    assert ((loss.double() - rloss).abs() <= 2 * lim).all()
    assert (loss[~keep] == 0).all()
    again = vocab_cross_entropy(x, w, t.to(torch.int32), s)
    assert torch.equal(loss, again[0]) and torch.equal(lse, again[1])


def test_loss_far_apart_logits(dev):
    """Logits from about -600 to 600: the running maximum carries."""
    x, w, s, t = _case(dev, 40, 2000, 256)
    w = (w.float() * 150).to(BF16)
    loss, lse = vocab_cross_entropy(x, w, t)
    _, _, _, _, rlse, rloss, lim, _ = _reference(x, w, s, t)
    assert ((lse.double() - rlse).abs() <= lim).all() and ((loss.double() - rloss).abs() <= 2 * lim).all()


@pytest.mark.parametrize("T", [5, 300])
def test_loss_odd_values(dev, T):
    """Targets outside the table, infinite and NaN logits, an ignored row of NaN:
    each stays in its own row."""
    x, w, _, t = _case(dev, T, 700, 64)
    clean, clean_lse = vocab_cross_entropy(x, w, t)
    t[0], t[1] = 700, -5
    x[2] = float("nan")
    x[3, 0] = float("inf")
    t[4], x[4] = -100, float("nan")
    loss, lse = vocab_cross_entropy(x, w, t)
    assert loss[:2].isnan().all() and torch.equal(lse[:2], clean_lse[:2])
    assert loss[2].isnan() and lse[2].isnan()
    assert lse[3].isinf() or lse[3].isnan()
    assert loss[4] == 0 and lse[4].isnan()
    assert torch.equal(loss[5:], clean[5:])
    # an ignore index inside the table
    loss, _ = vocab_cross_entropy(x[5:], w, t[5:], ignore_index=int(t[5]) if T > 5 else 0)
    assert T == 5 or loss[0] == 0


def test_loss_shapes_strides_empty(dev):
    x, w, _, t = _case(dev, 12, 500, 128)
    ref = vocab_cross_entropy(x, w, t)
    loss, lse = vocab_cross_entropy(x.view(3, 4, 128), w, t.view(3, 4))
    assert loss.shape == (3, 4) and torch.equal(loss.flatten(), ref[0]) and torch.equal(lse.flatten(), ref[1])
    wide = torch.full((500, 136), float("nan"), dtype=BF16, device=dev)
    wide[:, :128] = w
    xs = torch.full((12, 131), float("nan"), dtype=BF16, device=dev)
    xs[:, 3:] = x
    loss, lse = vocab_cross_entropy(xs[:, 3:], wide[:, :128], torch.stack((t, t), 1)[:, 0])
    assert torch.equal(loss, ref[0]) and torch.equal(lse, ref[1])
    assert vocab_cross_entropy(x[:0], w, t[:0])[0].shape == (0,)
    xg, wg = x[:0].clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(vocab_cross_entropy(xg, wg, t[:0])[0].sum(), (xg, wg))
    assert dx.shape == (0, 128) and not dw.any()


def _grad_bounds(x, w, s, t, g, h):
    """((dx, bound), (dw, bound)) in float64."""
    xd, wd, lg, err, lse, _, lim, keep = _reference(x, w, s, t)
    g = torch.where(keep, g.double(), torch.zeros_like(lse))
    c = g + (0 if h is None else h.double())
    p = (lg - lse[:, None]).exp()
    hot = torch.zeros_like(p).scatter_(1, t.clamp(0, w.shape[0] - 1)[:, None], g[:, None])
    P = p * c[:, None] - hot
    # P's own error: of its logit and lse, the float32 roundings of the
    # exponential (its argument up to the spread of the logits) and of the
    # subtraction, half a bf16 step
    spread = (lg - lse[:, None]).abs()
    perr = p * c.abs()[:, None] * (err + lim[:, None] + (8 + 2 * spread) * EPS) + 2 * EPS * hot.abs()
    perr = perr + HALF * (P.abs() + perr)
    out = []
    for ref, b, m, n in ((P @ wd, perr @ wd.abs(), P.abs() @ wd.abs(), w.shape[0]),
                         (P.t() @ xd, perr.t() @ xd.abs(), P.t().abs() @ xd.abs(), x.shape[0])):
        b = b + (n + 8) * EPS * m
        out.append((ref, b + HALF * (ref.abs() + b) + 1e-38))
    return out


def _check_grads(dx, dw, x, w, s, t, g, h):
    for got, (ref, bound) in zip((dx, dw), _grad_bounds(x, w, s, t, g, h)):
        if got is not None:
            assert got.dtype == BF16 and got.shape == ref.shape
            off = (got.double() - ref).abs()
            assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("T,V,H", [(1, 1, 8), (1, 1000, 512), (5, 257, 72), (63, 300, 264), (64, 1031, 64), (130, 777, 136),
                                   (200, 3001, 520), (333, 5021, 2880), (700, 513, 256)])
def test_gradients(dev, T, V, H):
    print(f"gradients T={T} V={V} H={H}", flush=True)
    x, w, _, t = _case(dev, T, V, H, ignored=T // 4)
    gen = torch.Generator(device=dev).manual_seed(8)
    g, h = torch.randn(T, generator=gen, device=dev), torch.randn(T, generator=gen, device=dev)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss, lse = vocab_cross_entropy(xg, wg, t)
    dx, dw = torch.autograd.grad((loss, lse), (xg, wg), (g, h), retain_graph=True)
    _check_grads(dx, dw, x, w, None, t, g, h)
    dx, dw = torch.autograd.grad(loss, (xg, wg), g)
    _check_grads(dx, dw, x, w, None, t, g, None)
    assert not dx[: T // 4].any()  # tokens that are not scored
    again = ops.vocab_loss_grad(x, w, t, lse.detach(), g)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    # one at a time
    only, none = ops.vocab_loss_grad(x, w, t, lse.detach(), g, need_weight=False)
    assert none is None and torch.equal(only, dx)
    none, only = ops.vocab_loss_grad(x, w, t, lse.detach(), g, need_x=False)
    assert none is None and torch.equal(only, dw)


@pytest.mark.parametrize("dtype", [E4, I8, E5])
@pytest.mark.parametrize("T,V,H", [(1, 500, 128), (77, 1003, 264), (300, 2000, 512)])
def test_gradient_through_a_coded_table(dev, dtype, T, V, H):
    x, w, s, t = _case(dev, T, V, H, dtype, ignored=T // 4)
    g = torch.randn(T, device=dev)
    xg = x.clone().requires_grad_()
    loss, _ = vocab_cross_entropy(xg, w, t, s)
    (dx,) = torch.autograd.grad(loss, xg, g)
    _check_grads(dx, None, x, w, s, t, g, None)
    with pytest.raises(NotImplementedError):
        ops.vocab_loss_grad(x, w, t, loss.detach(), g, weight_scale=s)


@pytest.mark.parametrize("T,V,H,dtype", [(70, 1500, 65536, BF16), (33, 3000, 32768, BF16), (33, 3000, 32768, I8),
                                         (150, 2500, 32776, E4)])
def test_gradients_over_several_pieces(dev, T, V, H, dtype):
    """More table rows than one piece (the wide rows make the pieces short),
    with and without a K split of dx."""
    x, w, s, t = _case(dev, T, V, H, dtype)
    g = torch.randn(T, device=dev)
    _, lse = vocab_cross_entropy(x, w, t, s)
    dx, dw = ops.vocab_loss_grad(x, w, t, lse, g, weight_scale=s, need_weight=dtype == BF16)
    _check_grads(dx, dw, x, w, s, t, g, None)


def test_gradients_by_differences(dev):
    """Central differences of the kernel's own loss, steps of four units of each
    value's last place (exact: the values' last two bits are cleared)."""
    T, V, H = 40, 600, 256
    x, w, _, t = _case(dev, T, V, H, ignored=6)
    x, w = ((v.view(torch.int16) & -4).view(BF16) for v in (x, w))
    g = torch.rand(T, device=dev)
    _, lse = vocab_cross_entropy(x, w, t)
    grads = ops.vocab_loss_grad(x, w, t, lse, g)
    bounds = _grad_bounds(x, w, None, t, g, None)
    lim, keep = _reference(x, w, None, t)[6:]
    for which in (0, 1):
        v = (x, w)[which].float()
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -60))) - 5) * torch.sign(torch.randn_like(v))
        ends = [(v + k * step).to(BF16) for k in (1, -1)]
        assert torch.equal((ends[0].double() + ends[1].double()) / 2, v.double())
        a, b = (vocab_cross_entropy(*((e, w) if which == 0 else (x, e)), t)[0].double() for e in ends)
        moved = float(((a - b) * g.double()).sum())
        linear = 2 * float((grads[which].double() * step.double()).sum())
        # the third derivative of a token's loss along the step is a third
        # cumulant of logit changes, at most (2 d)^3 for changes within +-d
        d = (step.double() @ w.double().t() if which == 0 else x.double() @ step.double().t()).abs().amax(1)
        third = float((g.double() * keep * (2 * d) ** 3).sum()) / 3
        rounding = 2 * float((bounds[which][1] * step.double().abs()).sum()) + 8 * float((g.double() * lim).sum())
        assert abs(moved - linear) <= third + rounding


def test_masked_rows_of_nan_leave_nothing(dev):
    """Unscored padding rows that hold NaN reach neither gradient."""
    x, w, _, t = _case(dev, 100, 900, 192)
    g = torch.rand(100, device=dev)
    t[::3] = -100
    _, lse = vocab_cross_entropy(x, w, t)
    dx, dw = ops.vocab_loss_grad(x, w, t, lse, g)
    x2 = x.clone()
    x2[::3] = float("nan")
    _, lse2 = vocab_cross_entropy(x2, w, t)
    dx2, dw2 = ops.vocab_loss_grad(x2, w, t, lse2, g)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and not dx2[::3].any()


def test_loss_streams_and_graph(dev):
    """On a side stream, and loss and gradients captured once and replayed with
    other inputs, eager work between the replays."""
    x, w, _, t = _case(dev, 90, 1500, 256)
    g = torch.rand(90, device=dev)
    ref = vocab_cross_entropy(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss, lse = vocab_cross_entropy(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(loss, ref[0]) and torch.equal(lse, ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lse = vocab_cross_entropy(x, w, t)
        dx, dw = ops.vocab_loss_grad(x, w, t, lse, g)
    for k in range(3):
        x.copy_(torch.randn_like(x))
        t.copy_(torch.randint(0, 1500, t.shape, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        e = vocab_cross_entropy(x, w, t)
        assert torch.equal(loss, e[0]) and torch.equal(lse, e[1])
        edx, edw = ops.vocab_loss_grad(x, w, t, e[1], g)
        assert torch.equal(dx, edx) and torch.equal(dw, edw)


def test_loss_compiles(dev):
    x, w, _, t = _case(dev, 20, 300, 64)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    fn = torch.compile(lambda a, b, c: vocab_cross_entropy(a, b, c)[0].mean(), fullgraph=True, backend="eager")
    a, b = fn(xg, wg, t), vocab_cross_entropy(xg, wg, t)[0].mean()
    assert torch.equal(a, b)
    for p, q in zip(torch.autograd.grad(a, (xg, wg)), torch.autograd.grad(b, (xg, wg))):
        assert torch.equal(p, q)


def test_methods_score_their_own_logits(dev):
    """The quant methods' cross_entropy against softmax over their apply: the
    logits there are rounded to bf16 (half a step of the largest)."""
    class VocabParallelEmbedding(torch.nn.Module):
        pass

    x, w, s, t = _case(dev, 33, 500, 256, E4)
    layer = VocabParallelEmbedding()
    layer.weight, layer.weight_scale = w, s
    m = Fp8LinearMethod.__new__(Fp8LinearMethod)
    bf = torch.nn.Module()
    bf.weight = (w.float() * s[:, None]).to(BF16)
    for method, ly in ((m, layer), (UnquantizedLinearMethod(), bf)):
        lg = method.apply(ly, x).double()
        ref = torch.logsumexp(lg, 1) - lg[torch.arange(33, device=dev), t]
        loss, _ = method.cross_entropy(ly, x, t)
        assert ((loss.double() - ref).abs() <= 2 * HALF * lg.abs().amax(1) + 1e-4).all()
    with pytest.raises(NotImplementedError):
        m.cross_entropy(bf, x, t)


def test_tied_table_step(dev):
    """Lookup, loss and both gradients of one tied table, the lookup's added into
    the loss's in place, against autograd's sum of the two."""
    V, H = 801, 128
    w = (torch.randn((V, H), device=dev) * 0.05).to(BF16).requires_grad_()
    ids = torch.randint(0, V, (4, 25), device=dev)
    x = embedding(ids, w, scale=H ** 0.5)
    loss, lse = vocab_cross_entropy(x[:, :-1], w, ids[:, 1:])
    (both,) = torch.autograd.grad(loss.mean(), w)
    g = torch.full(loss.shape, 1.0 / loss.numel(), device=dev)
    xd = x.detach()
    dx, dw = ops.vocab_loss_grad(xd[:, :-1], w.detach(), ids[:, 1:], lse.detach(), g)
    full = torch.zeros_like(xd)
    full[:, :-1] = dx
    alone = ops.vocab_lookup_grad(full, ids, V, H ** 0.5)
    assert torch.equal(both, dw + alone)
    ops.vocab_lookup_grad(full, ids, V, H ** 0.5, into=dw)
    # one rounding less than the sum of two rounded gradients
    assert ((dw.double() - both.double()).abs() <= 2 * HALF * (both.double().abs() + alone.double().abs())).all()


@pytest.mark.parametrize("T", [5, 300])
def test_a_loss_that_is_not_used_leaves_no_gradient(dev, T):
    """Targets outside the table whose loss is dropped by a `where`: zero
    gradient, as if the tokens were not there."""
    x, w, _, t = _case(dev, T, 700, 64)
    t[0], t[3] = 700, -5
    good = torch.ones(T, dtype=torch.bool, device=dev)
    good[0], good[3] = False, False
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss, _ = vocab_cross_entropy(xg, wg, t)
    dx, dw = torch.autograd.grad(torch.where(good, loss, 0.0).sum(), (xg, wg))
    assert not dx[~good].any()
    _check_grads(dx, dw, x, w, None, torch.where(good, t, -100), good.float(), None)


def test_a_tied_step_the_ways_autograd_runs_it(dev):
    """Lookup and loss on one table: traced without a break, on autograd's own
    thread and on the caller's, twice from one graph, under checkpointing, on a
    side stream and captured -- the same bits each time."""
    from torch.utils.checkpoint import checkpoint
    V, H = 1000, 128
    gen = torch.Generator(device=dev).manual_seed(15)
    table = (torch.randn((V, H), generator=gen, device=dev) * 0.1).to(BF16)
    ids, nxt = (torch.randint(0, V, (6, 7), generator=gen, device=dev) for _ in range(2))

    def step(w, ids, nxt):
        loss, lse = vocab_cross_entropy(embedding(ids, w, scale=8.0, padding_idx=3), w, nxt)
        return (loss + 1e-4 * lse * lse).sum()

    def grad(fn):
        w = table.clone().requires_grad_()
        fn(w, ids, nxt).backward()
        return w.grad

    ref = grad(step)
    torch._dynamo.reset()
    assert torch.equal(grad(torch.compile(step, backend="aot_eager", fullgraph=True)), ref)
    with torch.autograd.set_multithreading_enabled(False):
        assert torch.equal(grad(step), ref)
    for reentrant in (False, True):
        assert torch.equal(grad(lambda *a: checkpoint(step, *a, use_reentrant=reentrant)), ref)
    w = table.clone().requires_grad_()
    out = step(w, ids, nxt)
    once, again = (torch.autograd.grad(out, w, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(once, ref) and torch.equal(again, ref)
    del out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(torch.autograd.grad(step(w, ids, nxt), w)[0], ref)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (captured,) = torch.autograd.grad(step(w, ids, nxt), w)
    for _ in range(3):
        ids.copy_(torch.randint(0, V, (6, 7), generator=gen, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, torch.autograd.grad(step(w, ids, nxt), w)[0])


@pytest.mark.parametrize("T,V,H", [(1, 300, 64), (70, 1031, 264), (333, 777, 128), (2500, 513, 64)])
@pytest.mark.parametrize("kept", [0, 1, 0.1, 1.0])
def test_gradients_of_few_kept_tokens(dev, T, V, H, kept):
    """None, one, a tenth or all of the tokens scored, spread over the batch."""
    x, w, _, t = _case(dev, T, V, H)
    n = int(kept) if kept in (0, 1) and isinstance(kept, int) else max(1, int(T * kept))
    gen = torch.Generator(device=dev).manual_seed(21)
    keep = torch.zeros(T, dtype=torch.bool, device=dev)
    keep[torch.randperm(T, generator=gen, device=dev)[:n]] = True
    t = torch.where(keep, t, -100)
    g = torch.randn(T, generator=gen, device=dev)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    xg.data[~keep] = float("nan")
    loss, lse = vocab_cross_entropy(xg, wg, t)
    dx, dw = torch.autograd.grad(loss, (xg, wg), g)
    assert not dx[~keep].any()
    _check_grads(dx, dw, x, w, None, t, g, None)


def test_methods_score_without_the_padding(dev):
    """A table padded beyond its vocabulary: with the vocabulary's size the loss,
    its log-sum and the gradients are those of the rows that count."""
    class VocabParallelEmbedding(torch.nn.Module):
        pass

    V, rows = 450, 512
    x, w, s, t = _case(dev, 33, V, 256, E4)
    layer, bf = VocabParallelEmbedding(), torch.nn.Module()
    layer.weight = torch.zeros((rows, 256), device=dev).to(E4)
    layer.weight.view(torch.uint8)[:V] = w.view(torch.uint8)
    layer.weight_scale = torch.cat((s, torch.ones(rows - V, device=dev)))[:, None]
    m = Fp8LinearMethod.__new__(Fp8LinearMethod)
    for got, want in zip(m.cross_entropy(layer, x, t, vocab_size=V), vocab_cross_entropy(x, w, t, s)):
        assert torch.equal(got, want)
    assert not torch.equal(m.cross_entropy(layer, x, t)[1], vocab_cross_entropy(x, w, t, s)[1])
    bf.weight = torch.nn.Parameter(torch.zeros((rows, 256), dtype=BF16, device=dev))
    bf.weight.data[:V] = (w.float() * s[:, None]).to(BF16)
    loss, lse = UnquantizedLinearMethod().cross_entropy(bf, x, t, vocab_size=V)
    short = bf.weight.detach()[:V].clone().requires_grad_()
    want = vocab_cross_entropy(x, short, t)
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    dw, ref = torch.autograd.grad(loss.sum(), bf.weight)[0], torch.autograd.grad(want[0].sum(), short)[0]
    assert torch.equal(dw[:V], ref) and not dw[V:].any()
