"""The norms before and after a block with its gate and residual, on the GPU
against float64.

Bounds, in units of EPS = 2^-24, a float32 rounding. A row's mean square is a sum of
positive terms at most 16 + 6 + 16 additions deep (a lane's values, the lanes of a
wavefront, the wavefronts), its square root halves that, and a normalized value
takes few more: 32 in all. `mag` adds the magnitudes of what a value is the sum of;
a row's dot product of a gradient adds 48 again. Sums over tokens are at most 128
additions deep (a workgroup's rows, the rows of a workgroup, 16 x 32 workgroups).
Results are rounded by half a step of their type. The next norm is that of h as it
is stored, so its reference starts from the h that the call returned."""

import pytest
import torch

from qmoe import ops
from qmoe.layers.block import block_norm, block_residual

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 2.0 ** -24
E = 1e-6


def _near(got, ref, mag, depth, what):
    half, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    lim = half * ref.abs() + depth * EPS * mag + tiny
    err = (got.double() - ref).abs()
    bad = ~(err <= lim)
    assert not bad.any(), f"{what}: {int(bad.sum())} beyond, first {got[bad][:3].tolist()} ref {ref[bad][:3].tolist()}"


def _rand(g, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device=g.device) * std + mean).to(dtype)


def _operands(dev, T, H, yt, rt, wt, gate, post, nxt, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[gate]
    return (_rand(g, (T, H), yt), _rand(g, (T, H), rt, 2.0),
            None if shape is None else _rand(g, shape, yt if gate == "full" else wt, 0.3, 0.5),
            _rand(g, (H,), wt, 0.1, 1.0) if post else None, _rand(g, (H,), wt, 0.1, 1.0) if nxt else None,
            _rand(g, (T, H), rt), _rand(g, (T, H), yt) if nxt else None)


def _check(y, r, gate, wp, wn, gh, gz, sc, rs, off, h, z, grads):
    D = torch.float64
    H = r.shape[-1]
    yd, rd, hd = y.double(), r.double(), h.double()
    one = torch.ones((), dtype=D, device=y.device)
    gd = one if gate is None else gate.double()
    ry = one if wp is None else (yd.square().mean(-1, keepdim=True) + E).rsqrt()
    cp = one if wp is None else wp.double() + off
    ny = yd * ry
    b = ny * cp
    ref = rs * rd + sc * gd * b
    _near(h, ref, (rs * rd).abs() + (sc * gd * b).abs(), 48, "h")
    G, mag = torch.zeros_like(rd), torch.zeros_like(rd)
    out = {}
    if wn is not None:
        rh = (hd.square().mean(-1, keepdim=True) + E).rsqrt()
        nh, cn = hd * rh, wn.double() + off
        _near(z, nh * cn, (nh * cn).abs(), 48, "z")
        if gz is not None:
            q = gz.double() * cn
            G = rh * (q - nh * (q * nh).mean(-1, keepdim=True))
            mag = rh * (q.abs() + nh.abs() * (q * nh).abs().mean(-1, keepdim=True))
            out["next"] = ((gz.double() * nh).sum(0), (gz.double() * nh).abs().sum(0), 176)
    if gh is not None:
        G, mag = G + gh.double(), mag + gh.double().abs()
    out["residual"] = (rs * G, abs(rs) * mag, 128)
    db, mdb = sc * gd * G, abs(sc) * gd.abs() * mag
    dg, mdg = sc * G * b, abs(sc) * mag * b.abs()
    if gate is not None:
        if gate.dim() == 1:
            out["gate"] = (dg.sum(0), mdg.sum(0), 288)
        elif gate.shape[-1] == 1 and H > 1:
            out["gate"] = (dg.sum(-1, keepdim=True), mdg.sum(-1, keepdim=True), 208)
        else:
            out["gate"] = (dg, mdg, 160)
    if wp is None:
        out["y"] = (db, mdb, 160)
    else:
        q, mq = db * cp, mdb * cp.abs()
        out["y"] = (ry * (q - ny * (q * ny).mean(-1, keepdim=True)),
                    ry * (mq + ny.abs() * (mq * ny.abs()).mean(-1, keepdim=True)), 256)
        out["post"] = ((db * ny).sum(0), (mdb * ny.abs()).sum(0), 320)
    for name, got in grads.items():
        if got is None:
            assert name not in out, name
            continue
        ref, mag, depth = out[name]
        _near(got, ref, mag, depth, f"gradient of {name}")


NAMES = ("y", "residual", "gate", "post", "next")
SIZES = [(1, 1), (1, 8), (2, 7), (3, 64), (5, 513), (9, 512), (1, 4096), (130, 1000), (70, 2880), (33, 4104), (3, 7168),
         (600, 136), (2, 8200), (3, 16384), (2, 16383), (1100, 24)]


def _run(T, H, ts, sc, rs, off, nxt, lead=None):
    a = [t if t is None else t.clone().requires_grad_() for t in ts[:5]]
    out = block_residual(*a, scale=sc, residual_scale=rs, eps=E, weight_offset=off)
    out = out if nxt else (out,)
    leaves = [t for t in a if t is not None]
    grads = iter(torch.autograd.grad(out, leaves, ts[5:5 + len(out)]))
    return out, {n: (None if t is None else next(grads)) for n, t in zip(NAMES, a)}


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post,nxt", [(False, False), (False, True), (True, False), (True, True)])
def test_values_and_gradients(dev, T, H, gate, post, nxt):
    kinds = [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F32, F32, F32), (F16, F32, F16), (BF16, BF16, F32)]
    yt, rt, wt = kinds[(T + H + len(gate) + 2 * post + nxt) % len(kinds)]
    print(f"block T={T} H={H} gate={gate} post={post} next={nxt} {yt} {rt} {wt}", flush=True)
    ts = _operands(dev, T, H, yt, rt, wt, gate, post, nxt, T + H)
    sc, rs, off = (1.0, 1.0, 0.0) if T % 2 else (0.5, -1.25, 1.0)
    out, grads = _run(T, H, ts, sc, rs, off, nxt)
    assert out[0].dtype == rt and (not nxt or out[1].dtype == yt)
    for n, t in zip(NAMES, ts):
        assert t is None or grads[n].dtype == t.dtype and grads[n].shape == t.shape
    _check(*ts, sc, rs, off, out[0].detach(), out[1].detach() if nxt else None, grads)
    with torch.no_grad():  # the same bits without gradients, and again
        plain = block_residual(*ts[:5], scale=sc, residual_scale=rs, eps=E, weight_offset=off)
    for x, w in zip(plain if nxt else (plain,), out):
        assert torch.equal(x, w)
    for n, v in _run(T, H, ts, sc, rs, off, nxt)[1].items():
        assert v is None or torch.equal(v, grads[n])


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("xt,zt", [(BF16, BF16), (F16, F16), (F32, F32), (F32, BF16), (F32, F16)])
def test_norm_alone(dev, T, H, xt, zt):
    g = torch.Generator(device=dev).manual_seed(H)
    x, w, gz = _rand(g, (T, H), xt, 3.0), _rand(g, (H,), BF16, 0.1), _rand(g, (T, H), zt)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    z = block_norm(a, b, E, 1.0, zt)
    dx, dw = torch.autograd.grad(z, (a, b), gz)
    assert z.dtype == zt and dx.dtype == xt and dw.dtype == BF16
    zero = torch.zeros_like(x)
    _check(zero.to(zt), x, None, None, w, None, gz, 1.0, 1.0, 1.0, x, z.detach(), {"residual": dx, "next": dw})


def test_only_one_result_used(dev):
    ts = _operands(dev, 20, 264, BF16, F32, F32, "token", True, True, 3)
    for use in (0, 1):
        a = [t.clone().requires_grad_() for t in ts[:5]]
        out = block_residual(*a, eps=E)
        grads = dict(zip(NAMES, torch.autograd.grad(out[use], a, ts[5 + use], allow_unused=use == 0)))
        assert (grads["next"] is None) == (use == 0)
        _check(*ts[:5], ts[5] if use == 0 else None, ts[6] if use else None, 1.0, 1.0, 0.0, out[0].detach(),
               out[1].detach(), grads)


@pytest.mark.parametrize("which", range(5))
def test_one_gradient_alone(dev, which):
    """... is the one that the whole call gives, bit for bit."""
    for gate in ("channel", "token", "full"):
        ts = _operands(dev, 37, 520, BF16, BF16, BF16, gate, True, True, 5)
        _, want = _run(37, 520, ts, 0.5, 2.0, 0.0, True)
        a = list(ts[:5])
        a[which] = a[which].clone().requires_grad_()
        out = block_residual(*a, scale=0.5, residual_scale=2.0, eps=E)
        (got,) = torch.autograd.grad(out, a[which], ts[5:7])
        assert torch.equal(got, want[NAMES[which]])


def test_gradient_against_differences(dev):
    """Central differences along a random direction, of step 2^-10, of float32 values
    summed in float64: off by the third derivative (of order 1 per unit of the
    direction) times the step squared, and by the values' rounding over it."""
    T, H = 3, 24
    for gate in ("channel", "token", "full"):
        ts = _operands(dev, T, H, F32, F32, F32, gate, True, True, 8)
        a = [t.clone().requires_grad_() for t in ts[:5]]
        h, z = block_residual(*a, scale=0.7, residual_scale=1.1, eps=E)
        grads = torch.autograd.grad((h, z), a, ts[5:7])
        g = torch.Generator(device=dev).manual_seed(1)
        for i in range(5):
            v = torch.randn(a[i].shape, generator=g, device=dev)
            step, f = 2.0 ** -10, []
            for sign in (1, -1):
                b = list(ts[:5])
                b[i] = ts[i] + sign * step * v
                vals = block_residual(*b, scale=0.7, residual_scale=1.1, eps=E)
                f.append(sum((x.double() * w.double()).sum() for x, w in zip(vals, ts[5:7])))
            slope = float((f[0] - f[1]) / (2 * step))
            terms = float(sum(w.double().abs().sum() for w in ts[5:7]))
            assert abs(slope - float((grads[i].double() * v.double()).sum())) <= terms * (64 * step ** 2 + 32 * EPS / step)


def test_layouts(dev):
    """Leading axes, padded and transposed rows, repeated rows, unaligned starts:
    the values of contiguous operands."""
    g = torch.Generator(device=dev).manual_seed(2)
    wide = _rand(g, (6, 5, 152), BF16)
    y, r, z = wide[..., 8:136], wide[..., 3:131], wide.transpose(0, 1)[..., 16:144].transpose(0, 1)
    w1, w2 = _rand(g, (260,), F32)[2:130], _rand(g, (256,), F32)[::2]
    gates = (_rand(g, (6, 5, 1), F32), _rand(g, (128,), F16), wide[..., 24:152], _rand(g, (6, 1, 1), BF16).expand(6, 5, 1))
    for a, b in ((y, r), (r, z), (y.contiguous(), wide[:1, :1, :128].expand(6, 5, 128))):
        for gate in gates:
            out = []
            for f in (lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)):
                leaves = [f(t.detach()).requires_grad_() for t in (a, b, gate, w1, w2)]
                res = block_residual(*leaves)
                grads = torch.autograd.grad(res, leaves, (f(z), f(y)))
                assert res[0].shape == a.shape and all(x.shape == t.shape for x, t in zip(grads, leaves))
                out.append([*res, *grads])
            for p, q in zip(*out):
                # (unaligned operands run another instance of the same sums)
                assert torch.allclose(p.float(), q.float(), rtol=2 * torch.finfo(p.dtype).eps, atol=1e-5)
    one = block_residual(y[0, 0], r[0, 0], norm_weight=w1, next_weight=w2)
    many = block_residual(y, r, norm_weight=w1, next_weight=w2)
    assert torch.equal(one[0], many[0][0, 0]) and torch.equal(one[1], many[1][0, 0])


def test_empty_rows_and_zeros(dev):
    w = torch.ones(16, device=dev, requires_grad=True)
    y = torch.zeros((0, 16), device=dev, requires_grad=True)
    h, z = block_residual(y, y.detach(), gate=w, norm_weight=w, next_weight=w)
    assert h.shape == z.shape == (0, 16)
    gy, gw = torch.autograd.grad(h.sum() + z.sum(), (y, w))
    assert gy.shape == (0, 16) and (gw == 0).all()
    x = torch.zeros((3, 16), device=dev, requires_grad=True)
    z = block_norm(x, w)
    assert (z == 0).all()
    gx, gw = torch.autograd.grad(z.sum(), (x, w))
    assert torch.allclose(gx, torch.full_like(gx, 1e3)) and (gw == 0).all()  # eps^(-1/2)


def test_nan_and_infinity_stay_in_their_row(dev):
    ts = _operands(dev, 6, 520, BF16, BF16, BF16, "channel", True, True, 4)
    bad = ts[0].clone()
    bad[2, 100], bad[4, 3] = float("nan"), float("inf")
    rest = torch.tensor([0, 1, 3, 5], device=dev)
    want, wg = _run(6, 520, ts, 1.0, 1.0, 0.0, True)
    got, gg = _run(6, 520, (bad, *ts[1:]), 1.0, 1.0, 0.0, True)
    for x, y in ((got[0], want[0]), (got[1], want[1]), (gg["y"], wg["y"]), (gg["residual"], wg["residual"])):
        assert torch.equal(x[rest], y[rest]) and torch.isnan(x[2]).any() and torch.isnan(x[4]).any()


def test_captured_and_on_two_streams(dev):
    sets = [_operands(dev, 300, 1032, BF16, F32, F32, "channel", True, True, s) for s in (1, 2)]
    want = [_run(300, 1032, ts, 1.0, 1.0, 0.0, True) for ts in sets]
    want = [[*o, *g.values()] for o, g in want]
    static = [t.clone() for t in sets[0]]

    def step(ts):
        a = [t.detach().requires_grad_() for t in ts[:5]]
        out = block_residual(*a, eps=E)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, a, ts[5:7])]

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


def test_kept_factors_and_refusals(dev):
    ts = _operands(dev, 4, 64, BF16, BF16, BF16, "token", True, True, 4)
    h, z, rstd = ops.block_residual(*ts[:5], keep=True)
    assert rstd.shape == (2, 4)
    ref = (ts[0].double().square().mean(-1) + E).rsqrt()
    assert ((rstd[0].double() - ref).abs() <= 32 * EPS * ref).all()
    with pytest.raises(ValueError):
        ops.block_residual_grad(ts[5], ts[6], ts[0], h, *ts[2:5], None)
    with pytest.raises(ValueError):
        ops.block_residual_grad(None, None, ts[0], h, *ts[2:5], rstd)
    with pytest.raises(ValueError):
        block_residual(ts[0].cpu(), ts[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_the_lowest_value(dev, dtype):
    """Their squares' sum is infinite, the row factor zero: zeros behind the norm, with
    weights and gates above one, and other rows as without them."""
    H = 512
    g = torch.Generator(device=dev).manual_seed(3)
    x = _rand(g, (5, H), dtype)
    low = x.clone()
    low[2] = torch.finfo(dtype).min
    w, gate = torch.full((H,), 2.0, device=dev), torch.full((H,), 3.0, device=dev)
    z, clean = block_norm(low, w), block_norm(x, w)
    assert not z[2].any() and torch.equal(z[[0, 1, 3, 4]], clean[[0, 1, 3, 4]])
    h, want = (block_residual(v, x, gate=gate, norm_weight=w) for v in (low, x))
    assert torch.equal(h[2], x[2]) and torch.equal(h[[0, 1, 3, 4]], want[[0, 1, 3, 4]])
