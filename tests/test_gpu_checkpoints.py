"""8-bit checkpoints of a gated activation and a linear layer on the GPU.

The 8 bits themselves are compared exactly with an encoder in float64. Bounds, in
units of EPS = 2^-24, a float32 rounding: an exponential of x is off by 2 |x| + 2, a
sigmoid by 4 more, a derivative by a few products: `16 + 8 |x|` for all of them,
times the magnitudes that a value is the sum of. A product of K terms is off by K
times the sum of its terms' magnitudes. Results are rounded by half a step of their
type. The float32 exponential of gelu's argument is zero below 2^-126, so a sigmoid
there is off by up to 2^-125 whatever its size: `floor` multiplies that."""

import pytest
import torch

from qmoe import ops
from qmoe.layers.block import checkpointed_activation, checkpointed_linear
from qmoe.layers.quantization.unquantized import UnquantizedLinearMethod

pytestmark = pytest.mark.gpu

BF16, F16, F32, D = torch.bfloat16, torch.float16, torch.float32, torch.float64
EPS = 2.0 ** -24
ACTS = ["silu", "swigluoai", "gelu", "silu_and_mul_with_clamp", "situ:2.0:1.5", "situ:1.0:none"]


def _near(got, ref, mag, depth, what, floor=0.0):
    fi = torch.finfo(got.dtype)
    lim = fi.eps / 2 * ref.abs() + depth * EPS * mag + fi.smallest_normal * fi.eps / 2 + 2.0 ** -125 * floor
    bad = ~((got.to(D) - ref).abs() <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond, first {got[bad][:3].tolist()} ref {ref[bad][:3].tolist()}"


def _encode(x):
    """(codes' values, scale bytes) of rows [T, n], from the format's definition."""
    T, n = x.shape
    v = torch.nn.functional.pad(x.to(D), (0, -n % 32)).unflatten(1, (-1, 32))
    fin = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    top = fin.abs().amax(-1)
    e = torch.frexp(top)[1] - 9                        # top < 2^(e + 9)
    unit = torch.ldexp(torch.ones((), dtype=D), e.cpu()).to(x.device)
    e = torch.where(top > 448 * unit, e + 1, e)
    e = torch.where(top == 0, torch.full_like(e, -127), e.clamp_min(-127))
    unit = torch.ldexp(torch.ones((), dtype=D), e.cpu()).to(x.device)[..., None]
    q = fin / unit
    step = torch.ldexp(torch.ones((), dtype=D), (torch.frexp(q.abs().clamp_min(2.0 ** -6))[1] - 4).cpu()).to(x.device)
    out = torch.where(torch.isfinite(v), torch.round(q / step) * step * unit, torch.full_like(v, float("nan")))
    return out.flatten(1)[:, :n], (e + 127).to(torch.uint8)


def _decode(codes, scales):
    n = codes.shape[1]
    s = torch.ldexp(torch.ones((), dtype=D), scales.cpu().to(torch.int32) - 127).to(codes.device)
    return codes.view(torch.float8_e4m3fn).to(F32).to(D) * s.repeat_interleave(32, 1)[:, :n]


def _same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


def _hard_rows(dev, T, n, dtype, seed):
    """Rows of normal values with blocks of zeros, huge, tiny and tied values."""
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((T, n), generator=g, device=dev) * 2.0 ** torch.randint(-6, 3, (T, 1), generator=g, device=dev)
    x[::5, : n // 2] = 0.0
    x[1::5] = torch.randint(-480, 481, (x[1::5].shape), generator=g, device=dev).to(F32)  # ties, and 448 in reach
    x[2::5] *= 2.0 ** (-12 if dtype == F16 else -125)
    x[3::5] = (x[3::5] * (2.0 ** (8 if dtype == F16 else 118))).clamp(-6e4, 6e4) if dtype == F16 else x[3::5] * 2.0 ** 118
    return x.to(dtype)


@pytest.mark.parametrize("T,K", [(1, 32), (2, 64), (7, 2880), (64, 4096), (33, 14336), (300, 160)])
def test_eight_bits_of_rows(dev, T, K):
    print(f"pack T={T} K={K}", flush=True)
    x = _hard_rows(dev, T, K, BF16, K)
    x[0, 3], x[0, 31], x[-1, K - 1] = float("inf"), float("nan"), -float("inf")
    w = torch.zeros((8, K), dtype=BF16, device=dev)
    _, codes, scales = ops.linear_checkpoint(x, w)
    ref, byte = _encode(x)
    assert torch.equal(scales, byte)
    assert _same(_decode(codes, scales), ref)


def _act_parts(act, g, u):
    """(value, d/dg, d/du) in float64 and the magnitudes that they are sums of."""
    one = torch.ones_like(g)
    if act == "swigluoai":
        gc, uc = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        s = torch.sigmoid(1.702 * gc)
        dg, du = (uc + 1) * s * (1 + 1.702 * gc * (1 - s)) * (g <= 7), gc * s * (u.abs() <= 7)
        return (uc + 1) * gc * s, dg, du, ((uc.abs() + 1) * gc.abs() * s, (uc.abs() + 1) * s * (1 + 1.702 * gc.abs()), du.abs())
    if act == "gelu":
        c = (2.0 / torch.pi) ** 0.5
        a = c * (g + 0.044715 * g ** 3)
        s = torch.sigmoid(2 * a)
        q = 2 * c * g * s * torch.sigmoid(-2 * a) * (1 + 3 * 0.044715 * g * g)
        # an error of a is one of s: 2 a s' against s, largest where the exponential is
        return g * s * u, (s + q) * u, g * s, ((g * s * u).abs(), (s + q.abs()) * u.abs(), (g * s).abs())
    if act.startswith("situ"):
        _, b, lin = act.split(":")
        b = float(b)
        s, t = torch.sigmoid(g), torch.tanh(g / b)
        l = None if lin == "none" else float(lin)
        uc, ud = (u, one) if l is None else (l * torch.tanh(u / l), 1 - torch.tanh(u / l) ** 2)
        dg = ((1 - t * t) * s + b * t * s * (1 - s)) * uc
        return (b * t * s * uc, dg, b * t * s * ud,
                ((b * t * s * uc).abs(), (2 * s + b * t.abs() * s) * uc.abs(), 2 * (b * t * s).abs()))
    lim = 10.0 if act != "silu" else float("inf")
    gc, uc = g.clamp(max=lim), u.clamp(-lim, lim)
    s = torch.sigmoid(gc)
    dg, du = s * (1 + gc * (1 - s)) * uc * (g <= lim), gc * s * (u.abs() <= lim)
    return gc * s * uc, dg, du, ((gc * s * uc).abs(), s * (1 + gc.abs()) * uc.abs(), du.abs())


def _depth(act, g):
    x = g.abs() * (1.702 if act == "swigluoai" else 1.0)
    if act == "gelu":
        x = 1.6 * (g.abs() + 0.045 * g.abs() ** 3)
    return 24 + 8 * x.clamp(max=100.0)  # (beyond, an exponential is 0 or infinite)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,I,dtype", [(1, 1, BF16), (1, 8, F16), (3, 31, BF16), (2, 33, F16), (5, 64, BF16),
                                       (17, 2880, BF16), (4, 4099, BF16), (9, 2056, F16), (130, 520, BF16),
                                       (3, 14336, BF16), (700, 40, F16)])
def test_activation_values_and_gradient(dev, T, I, dtype, act):
    print(f"act T={T} I={I} {dtype} {act}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(T + I)
    x = (torch.randn((T, 2 * I), generator=gen, device=dev) * 4).to(dtype)
    x.view(-1)[::97] = 0.0
    dh = torch.randn((T, I), generator=gen, device=dev).to(dtype)
    a = x.clone().requires_grad_()
    h = checkpointed_activation(a, act)
    (dx,) = torch.autograd.grad(h, a, dh)
    assert h.dtype == dx.dtype == dtype and h.shape == (T, I) and dx.shape == x.shape
    g, u = x.to(D)[:, :I], x.to(D)[:, I:]
    val, _, _, (mag, _, _) = _act_parts(act, g, u)
    _near(h.detach(), val, mag, _depth(act, g), "h", (g * u).abs() if act == "gelu" else 0.0)
    g8, u8 = _encode(x[:, :I])[0], _encode(x[:, I:])[0]
    _, dg, du, (_, mg, mu) = _act_parts(act, g8, u8)
    dd = dh.to(D)
    fg = (dd * u8).abs() * (1 + 1.6 * g8.abs() * (1 + 0.135 * g8 * g8)) if act == "gelu" else 0.0
    _near(dx[:, :I], dd * dg, dd.abs() * mg, _depth(act, g8), "gradient of gate", fg)
    _near(dx[:, I:], dd * du, dd.abs() * mu, _depth(act, g8), "gradient of up", (dd * g8).abs() if act == "gelu" else 0.0)
    with torch.no_grad():
        assert torch.equal(checkpointed_activation(x, act), h)
    _, codes, scales = ops.act_checkpoint(x, act)
    for half, (lo, ref) in enumerate(((0, x[:, :I]), (I, x[:, I:]))):
        want, byte = _encode(ref)
        assert torch.equal(scales[:, half], byte)
        assert _same(_decode(codes[:, lo: lo + I].contiguous(), scales[:, half]), want)


@pytest.mark.parametrize("act", ACTS)
def test_activation_gradient_against_differences(dev, act):
    """At 8-bit values the checkpoint is exact: central differences of the float64
    activation, whose third derivative is below 8 here times the values' 4."""
    gen = torch.Generator(device=dev).manual_seed(7)
    x = _encode((torch.randn((4, 64), generator=gen, device=dev) * 2).to(BF16))[0].to(BF16)
    x = torch.cat((_encode(x[:, :32])[0], _encode(x[:, 32:])[0]), 1).to(BF16)
    a = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(checkpointed_activation(a, act).sum(), a)
    g, u = x.to(D)[:, :32], x.to(D)[:, 32:]
    s = 2.0 ** -12
    fg = (_act_parts(act, g + s, u)[0] - _act_parts(act, g - s, u)[0]) / (2 * s)
    fu = (_act_parts(act, g, u + s)[0] - _act_parts(act, g, u - s)[0]) / (2 * s)
    ref = torch.cat((fg, fu), 1)
    assert ((dx.to(D) - ref).abs() <= torch.finfo(BF16).eps / 2 * ref.abs() + 64 * s * s + 2.0 ** -16).all()


def test_activation_clamps_pass_their_limits(dev):
    """7 and -7 are 8-bit values; a NaN passes the clamps."""
    x = torch.tensor([[7.0, 7.5, -20.0, 1.0, 2.0, float("nan"), 3.0] + [7.0, -7.0, 7.5, -7.5, 0.0, 1.0, float("nan")]],
                     device=dev, dtype=BF16, requires_grad=True)
    h = checkpointed_activation(x, "swigluoai")
    (dx,) = torch.autograd.grad(h.sum(), x)
    assert (dx[0, [1]] == 0).all() and (dx[0, [9, 10]] == 0).all()
    assert (dx[0, [0, 7, 8, 11]] != 0).all()
    assert torch.isnan(h[0, 5:]).all() and torch.isfinite(h[0, :5]).all()
    assert torch.isnan(dx[0, [5, 6, 12]]).all() and torch.isfinite(dx[0, :5]).all() and torch.isfinite(dx[0, 7:12]).all()


def test_activation_far_values(dev):
    """Large and infinite values: what the formulas give in the limit, and nothing
    beside the columns that hold them."""
    for act in ACTS[:4]:
        x = torch.zeros((1, 128), device=dev, dtype=BF16)
        x[0, :4] = torch.tensor([3e38, -3e38, 1e4, -1e4])
        x[0, 64:68] = 1.0
        x[0, 40] = float("inf")
        a = x.clone().requires_grad_()
        h = checkpointed_activation(a, act)
        (dx,) = torch.autograd.grad(h.sum(), a)
        assert h[0, 1] == 0 and h[0, 3] == 0 and h[0, 0] > 0 and h[0, 2] > 0
        assert torch.isfinite(dx[0, :40]).all() and torch.isfinite(dx[0, 41:104]).all()
        assert torch.isnan(dx[0, 40])


def test_activation_layouts(dev):
    gen = torch.Generator(device=dev).manual_seed(3)
    wide = torch.randn((3, 5, 200), generator=gen, device=dev).to(BF16)
    for v in (wide[..., 8:136], wide[..., 3:131], wide.transpose(0, 1)[..., :96], wide[:1].expand(3, 5, 200), wide[0, 0],
              wide[:, :0]):
        a, b = v.detach().requires_grad_(), v.clone(memory_format=torch.contiguous_format).requires_grad_()
        h, w = checkpointed_activation(a), checkpointed_activation(b)
        assert h.shape == (*v.shape[:-1], v.shape[-1] // 2) and torch.equal(h, w)
        dh = torch.ones_like(h[..., :1]).expand_as(h)
        assert torch.equal(torch.autograd.grad(h, a, dh)[0], torch.autograd.grad(w, b, dh.contiguous())[0])


LINEAR = [(1, 32, 8), (1, 4096, 64), (2, 64, 24), (19, 2880, 2880), (63, 320, 72), (64, 256, 256), (65, 160, 264),
          (127, 4096, 520), (128, 512, 1000), (129, 96, 2056), (200, 2880, 640), (257, 1024, 384), (300, 14336, 256),
          (513, 544, 4096), (777, 1056, 1544), (1500, 352, 128)]


@pytest.mark.parametrize("T,K,N", LINEAR)
@pytest.mark.parametrize("bias", [None, BF16, F32])
def test_linear_values_and_gradients(dev, T, K, N, bias):
    print(f"linear T={T} K={K} N={N} bias={bias}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(T + K + N)
    x = (torch.randn((T, K), generator=gen, device=dev) * (1 + 9 * (torch.rand(K, generator=gen, device=dev) < 0.05))).to(BF16)
    w = (torch.randn((N, K), generator=gen, device=dev) * 0.05).to(BF16)
    dy = torch.randn((T, N), generator=gen, device=dev).to(BF16)
    ts = [x, w] + ([torch.randn(N, generator=gen, device=dev).to(bias)] if bias else [])
    leaves = [t.clone().requires_grad_() for t in ts]
    y = checkpointed_linear(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    xd, wd, gd = x.to(D), w.to(D), dy.to(D)
    b = ts[2].to(D) if bias else 0.0
    _near(y.detach(), xd @ wd.t() + b, xd.abs() @ wd.abs().t() + (b.abs() if bias else 0.0), K + 8, "y")
    _near(grads[0], gd @ wd, gd.abs() @ wd.abs(), N + 8, "dx")
    x8 = _encode(x)[0]
    _near(grads[1], gd.t() @ x8, gd.abs().t() @ x8.abs(), T + 8, "dw")
    if bias:
        assert grads[2].dtype == bias
        _near(grads[2], gd.sum(0), gd.abs().sum(0), T + 8, "dbias")
    for g, h in zip(grads, torch.autograd.grad(checkpointed_linear(*leaves), leaves, dy)):
        assert torch.equal(g, h)
    with torch.no_grad():
        assert torch.equal(checkpointed_linear(*ts), y)


def test_linear_one_gradient_alone(dev):
    """... is the one that the whole call gives, bit for bit; without the weight's no
    8 bits are kept."""
    gen = torch.Generator(device=dev).manual_seed(1)
    ts = [torch.randn(s, generator=gen, device=dev).to(BF16) for s in ((70, 96), (136, 96), (136,))]
    dy = torch.randn((70, 136), generator=gen, device=dev).to(BF16)
    leaves = [t.clone().requires_grad_() for t in ts]
    want = torch.autograd.grad(checkpointed_linear(*leaves), leaves, dy)
    for i in range(3):
        a = list(ts)
        a[i] = leaves[i]
        assert torch.equal(torch.autograd.grad(checkpointed_linear(*a), leaves[i], dy)[0], want[i])
    y = checkpointed_linear(leaves[0], ts[1])
    assert [t is None for t in y.grad_fn.saved_tensors] == [False, True, True]


def test_linear_gradient_against_differences(dev):
    """x of 8-bit values: the layer is linear in each operand, so differences of its
    float64 product along a direction are the gradient exactly."""
    gen = torch.Generator(device=dev).manual_seed(2)
    x = _encode(torch.randn((40, 64), generator=gen, device=dev).to(BF16))[0].to(BF16)
    w, dy = (torch.randn(s, generator=gen, device=dev).to(BF16) for s in ((48, 64), (40, 48)))
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(checkpointed_linear(a, b), (a, b), dy)
    f = lambda x, w: (x.to(D) @ w.to(D).t() * dy.to(D)).sum()  # noqa: E731
    v, u = torch.randn((40, 64), generator=gen, device=dev), torch.randn((48, 64), generator=gen, device=dev)
    for grad, vec, diff in ((dx, v, f(x.to(D) + v, w) - f(x, w)), (dw, u, f(x, w.to(D) + u) - f(x, w))):
        terms = (grad.to(D).abs() * vec.to(D).abs()).sum()
        assert ((grad.to(D) * vec.to(D)).sum() - diff).abs() <= torch.finfo(BF16).eps * terms


def test_linear_layouts_and_method(dev):
    gen = torch.Generator(device=dev).manual_seed(4)
    wide = torch.randn((4, 6, 232), generator=gen, device=dev).to(BF16)
    table = torch.randn((72, 168), generator=gen, device=dev).to(BF16)
    w = table[:, 8:104]  # rows 336 bytes apart
    for v in (wide[..., 8:104], wide[..., 3:99], wide.transpose(0, 1)[..., :96], wide[:1, :, :96].expand(4, 6, 96),
              wide[0, 0, :96], wide[:0, :, :96]):
        a, b = v.detach().requires_grad_(), w.detach().requires_grad_()
        c, d = v.clone(memory_format=torch.contiguous_format).requires_grad_(), w.contiguous().requires_grad_()
        y, z = checkpointed_linear(a, b), checkpointed_linear(c, d)
        assert y.shape == (*v.shape[:-1], 72) and torch.equal(y, z)
        dy = torch.ones_like(y[..., :1]).expand_as(y)
        for g, h in zip(torch.autograd.grad(y, (a, b), dy), torch.autograd.grad(z, (c, d), dy.contiguous())):
            assert torch.equal(g, h)
    layer = torch.nn.Module()
    layer.weight = torch.nn.Parameter(w.contiguous())
    method = UnquantizedLinearMethod()
    x = wide[..., :96].contiguous()
    y = method.apply_checkpointed(layer, x)
    # (the same product by other kernels: both within half a step of the exact sum)
    apart = (y - method.apply(layer, x)).abs().to(D)
    mag = x.to(D).abs() @ w.to(D).abs().t()
    assert (apart <= torch.finfo(BF16).eps * y.abs().to(D) + 4 * 96 * EPS * mag).all() and y.requires_grad
    y.sum().backward()
    assert layer.weight.grad.shape == layer.weight.shape


def test_nan_and_infinity_stay_in_their_rows_and_columns(dev):
    x = torch.randn((70, 96), device=dev).to(BF16)
    w, dy = torch.randn((136, 96), device=dev).to(BF16), torch.randn((70, 136), device=dev).to(BF16)
    x[3, 7], w[135, 5], dy[69, 2] = float("nan"), float("inf"), float("inf")
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(checkpointed_linear(a, b), (a, b), dy)
    keep = torch.ones(96, dtype=torch.bool, device=dev)
    keep[5] = False
    assert torch.isfinite(dx[:69][:, keep]).all() and not torch.isfinite(dx[:69, 5]).any()
    keep[5], keep[7] = True, False
    rows = torch.arange(136, device=dev) != 2
    assert torch.isfinite(dw[rows][:, keep]).all() and torch.isnan(dw[:, 7]).all() and not torch.isfinite(dw[2]).any()


def test_captured_and_on_two_streams(dev):
    def data(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        return [torch.randn(s, generator=g, device=dev).to(BF16) for s in ((200, 256), (512, 256), (256, 256), (200, 256))]

    def step(ts):
        x, w1, w2, dy = (t.detach().requires_grad_() for t in ts)
        y = checkpointed_linear(checkpointed_activation(checkpointed_linear(x, w1), "silu"), w2)
        return [y.detach(), *torch.autograd.grad(y, (x, w1, w2), dy.detach())]

    sets = [data(s) for s in (1, 2)]
    want = [step(ts) for ts in sets]
    static = [t.clone() for t in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in (1, 0, 1, 0):
        for s, t in zip(static, sets[i]):
            s.copy_(t)
        graph.replay()
        step(sets[1 - i])
        torch.cuda.synchronize()
        for x, y in zip(out, want[i]):
            assert torch.equal(x, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            for x, y in zip(res, want[i]):
                assert torch.equal(x, y)
