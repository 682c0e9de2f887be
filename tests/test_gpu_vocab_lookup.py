"""Vocabulary lookups and their gradient on the GPU against float64. Bounds:
one rounding to the output type is off by at most half a step (eps / 2 relative
to the value); a float32 sum of n terms by n 2^-24 of the sum of their
magnitudes; the scaling adds one or two float32 roundings."""

import pytest
import torch

from qmoe import ops
from qmoe.layers.quantization.fp8 import Fp8LinearMethod
from qmoe.layers.quantization.unquantized import UnquantizedLinearMethod
from qmoe.layers.vocab import embedding

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4, E5, I8 = (torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.float8_e5m2,
                              torch.int8)


def _half(t):
    return torch.finfo(t).eps / 2


def _table(dev, V, H, dtype, seed=0, pad=0):
    """A [V, H] table (rows `pad` values further apart) and its row scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn((V, H + pad), generator=g, device=dev)
    if dtype in (BF16, F32):
        return w.to(dtype)[:, :H], None
    w = (w * 40).round().clamp(-127, 127).to(I8) if dtype == I8 else w.to(dtype)
    return w[:, :H], torch.rand(V, generator=g, device=dev) * 0.02 + 1e-3


@pytest.mark.parametrize("N,V,H,pad", [(1, 1, 1, 0), (1, 1000, 4096, 0), (8, 777, 2880, 0), (7, 300, 2881, 0),
                                       (2000, 513, 520, 0), (33, 64, 512, 8), (5, 64, 512, 3), (1500, 1000, 9000, 0)])
@pytest.mark.parametrize("dtype", [BF16, F32, E4, E5, I8])
def test_lookup_values(dev, N, V, H, pad, dtype):
    w, s = _table(dev, V, H, dtype, pad=pad)
    g = torch.Generator(device=dev).manual_seed(1)
    ids = torch.randint(0, V, (N,), generator=g, device=dev)
    for out_dtype, scale, idt in ((BF16, 1.0, torch.int64), (F32, 53.66, torch.int32), (F16, 1.0, torch.int32)):
        got = embedding(ids.to(idt), w, s, scale=scale, out_dtype=out_dtype)
        ref = w.double()[ids] * scale
        if s is not None:
            ref = ref * s.to(out_dtype).double()[ids, None]
        assert got.dtype == out_dtype and got.shape == (N, H)
        if scale == 1.0:  # code x scale is exact in float32: one rounding
            assert torch.equal(got, ref.float().to(out_dtype))
        else:
            lim = (_half(out_dtype) + 3 * 2.0 ** -24) * ref.abs() + 1e-44
            assert ((got.double() - ref).abs() <= lim).all()


def test_lookup_shapes_bad_ids_and_empty(dev):
    w, _ = _table(dev, 50, 96, BF16)
    ids = torch.tensor([[0, 49, -1], [50, 3, 2 ** 40]], device=dev)
    out = embedding(ids, w)
    assert out.shape == (2, 3, 96)
    ok = (ids >= 0) & (ids < 50)
    assert torch.equal(out[ok], w[ids[ok]]) and out[~ok].isnan().all()
    assert embedding(ids[:0], w).shape == (0, 3, 96)


def test_lookup_rows_past_4_gib(dev):
    """Row offsets beyond 32 bits."""
    V, H = 1100000, 4096  # 4.5 GB of codes
    w = torch.zeros((V, H), dtype=I8, device=dev)
    s = torch.ones(V, device=dev)
    ids = torch.tensor([V - 1, 0, 1048576], device=dev)
    for k, i in enumerate(ids.tolist()):
        w[i] = k + 1
    assert torch.equal(embedding(ids, w, s)[:, 17].float().cpu(), torch.tensor([1.0, 2.0, 3.0]))


def _check_grad(dw, ids, g, V, scale, padding, before=None):
    """Against float64 sums, with the float32 summation bound."""
    H = g.shape[-1]
    flat, g = ids.reshape(-1), g.reshape(-1, H).double()
    keep = (flat >= 0) & (flat < V)
    if padding is not None:
        keep &= flat != padding
    ref, mag = (torch.zeros((V, H), dtype=torch.float64, device=g.device) for _ in range(2))
    ref.index_add_(0, flat[keep], g[keep])
    mag.index_add_(0, flat[keep], g[keep].abs())
    count = torch.bincount(flat[keep], minlength=V)[:, None]
    ref, lim = ref * scale, (count + 2) * 2.0 ** -24 * mag * abs(scale)
    if before is not None:
        lim = lim + 2.0 ** -24 * (ref.abs() + before.double().abs())
        ref = ref + before.double()
    lim = lim + _half(dw.dtype) * (ref.abs() + lim) + 1e-44
    assert ((dw.double() - ref).abs() <= lim).all()
    untouched = (count == 0).expand(V, H)
    assert torch.equal(dw[untouched], torch.zeros_like(dw[untouched]) if before is None else before[untouched])


@pytest.mark.parametrize("N,V,H", [(1, 1, 1), (1, 1000, 96), (64, 3, 64), (777, 5003, 1000), (3000, 131, 2880),
                                   (257, 600, 2881), (16, 140000, 64), (5000, 1, 72)])
@pytest.mark.parametrize("gdt,wdt,idt", [(BF16, BF16, torch.int64), (F32, F32, torch.int32), (BF16, F32, torch.int32)])
def test_lookup_grad(dev, N, V, H, gdt, wdt, idt):
    gen = torch.Generator(device=dev).manual_seed(N + V)
    ids = torch.randint(0, V, (N,), generator=gen, device=dev)
    g = torch.randn((N, H), generator=gen, device=dev).to(gdt)
    for padding in (None, int(ids[0])):
        dw = ops.vocab_lookup_grad(g, ids.to(idt), V, 1.75, padding, wdt)
        assert dw.dtype == wdt and dw.shape == (V, H)
        _check_grad(dw, ids, g, V, 1.75, padding)
        assert torch.equal(dw, ops.vocab_lookup_grad(g, ids.to(idt), V, 1.75, padding, wdt))  # the same bits again


@pytest.mark.parametrize("kind", ["one", "half", "natural", "bad"])
def test_lookup_grad_uneven_tokens(dev, kind):
    """One token only (a run over every chunk, more of one range than a
    wavefront keeps), a token that makes up half, natural frequencies, ids
    outside the table."""
    N, V, H = 20011, 4099, 264
    gen = torch.Generator(device=dev).manual_seed(5)
    ids = torch.randint(0, V, (N,), generator=gen, device=dev)
    if kind == "one":
        ids[:] = 77
    elif kind == "half":
        ids[torch.rand(N, generator=gen, device=dev) < 0.5] = V - 1
    elif kind == "natural":
        ids = (V ** torch.rand(N, generator=gen, device=dev, dtype=torch.float64)).long() - 1
    else:
        ids[::3], ids[1::3] = -7, V + 12
    g = torch.randn((N, H), generator=gen, device=dev).to(BF16)
    _check_grad(ops.vocab_lookup_grad(g, ids, V, dtype=F32), ids, g, V, 1.0, None)


def test_lookup_grad_into_touches_only_its_rows(dev):
    N, V, H = 500, 3001, 128
    gen = torch.Generator(device=dev).manual_seed(9)
    ids = torch.randint(0, V, (N,), generator=gen, device=dev)
    g = torch.randn((N, H), generator=gen, device=dev).to(BF16)
    for dt in (BF16, F32):
        wide = torch.randn((V, H + 8), generator=gen, device=dev).to(dt)
        before, beside = wide[:, :H].clone(), wide[:, H:].clone()
        out = ops.vocab_lookup_grad(g, ids, V, into=wide[:, :H])
        _check_grad(out, ids, g, V, 1.0, None, before)
        assert torch.equal(wide[:, H:], beside)


def test_lookup_grad_no_tokens(dev):
    g, ids = torch.empty((0, 64), dtype=BF16, device=dev), torch.empty((0,), dtype=torch.int64, device=dev)
    assert not ops.vocab_lookup_grad(g, ids, 33).any()
    into = torch.ones((33, 64), device=dev)
    assert torch.equal(ops.vocab_lookup_grad(g, ids, 33, into=into), torch.ones_like(into))


def test_lookup_autograd(dev):
    """Through autograd: against the formula, and against differences (the
    lookup is linear in the table)."""
    V, H = 41, 24
    w = torch.randn((V, H), device=dev, requires_grad=True)
    ids = torch.tensor([[1, 5, 1], [40, 2, 5]], device=dev)
    up = torch.randn((2, 3, H), device=dev)
    out = embedding(ids, w, scale=3.0, padding_idx=2, out_dtype=F32)
    (dw,) = torch.autograd.grad(out, w, up)
    _check_grad(dw, ids, up, V, 3.0, 2)
    e = torch.randn((V, H), device=dev)
    e[2] = 0
    moved = (embedding(ids, (w + e).detach(), scale=3.0, out_dtype=F32) - out.detach()).double()
    # differences of float32 outputs: 4 roundings of values up to ~12, 144 of them
    assert abs(float((moved * up.double()).sum() - (dw.double() * e.double()).sum())) < 144 * 4 * 2.0 ** -24 * 16 * 4
    wide = up.new_zeros((2, 3, 2 * H))[..., ::2]  # a strided gradient
    wide.copy_(up)
    assert torch.equal(torch.autograd.grad(embedding(ids, w, scale=3.0, padding_idx=2, out_dtype=F32), w, wide)[0], dw)


def test_lookup_streams_and_graph(dev):
    """On a side stream, and captured with its gradient and replayed with other
    ids, eager calls between the replays."""
    w, _ = _table(dev, 3000, 512, BF16)
    ids = torch.randint(0, 3000, (600,), device=dev)
    g = torch.randn((600, 512), device=dev).to(BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = embedding(ids, w), ops.vocab_lookup_grad(g, ids, 3000)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, w[ids])
    _check_grad(b, ids, g, 3000, 1.0, None)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = embedding(ids, w), ops.vocab_lookup_grad(g, ids, 3000)
    for _ in range(3):
        ids.copy_(torch.randint(0, 3000, (600,), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, w[ids])
        assert torch.equal(b, ops.vocab_lookup_grad(g, ids, 3000))


@pytest.mark.parametrize("dtype", [E4, I8, E5])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_fp8_method_embedding_keeps_its_results(dev, dtype, out_dtype):
    """The quant method's lookup gives the bits of its former gather, cast and
    product."""
    w, s = _table(dev, 700, 520, dtype)
    layer = torch.nn.Module()
    layer.weight, layer.weight_scale, layer.params_dtype = w, s, out_dtype
    ids = torch.randint(0, 700, (4, 9), device=dev)
    got = Fp8LinearMethod.embedding(None, layer, ids)
    was = w.view(torch.uint8)[ids].view(dtype).to(out_dtype) * s[ids].to(out_dtype).unsqueeze(-1)
    assert got.dtype == out_dtype and torch.equal(got, was)


def test_unquantized_method_embedding_and_tie(dev):
    m, emb, head = UnquantizedLinearMethod(), torch.nn.Module(), torch.nn.Module()
    m.create_weights(emb, 256, [300], 256, 300, BF16)
    emb.weight.data.normal_()
    m.process_weights_after_loading(emb)
    assert m.tie_weights(head, emb) is head and head.weight is emb.weight
    ids = torch.randint(0, 300, (17,), device=dev)
    x = m.embedding(emb, ids)
    assert torch.equal(x, emb.weight[ids])
    assert m.apply(head, x).shape == (17, 300)


def test_lookup_compiles(dev):
    w, _ = _table(dev, 100, 64, F32)
    w = w.clone().requires_grad_()
    ids = torch.randint(0, 100, (12,), device=dev)
    fn = torch.compile(lambda i, t: embedding(i, t, scale=2.0, out_dtype=F32) * 3.0, fullgraph=True, backend="eager")
    a, b = fn(ids, w), embedding(ids, w, scale=2.0, out_dtype=F32) * 3.0
    assert torch.equal(a, b)
    up = torch.randn_like(a)
    assert torch.equal(torch.autograd.grad(a, w, up)[0], torch.autograd.grad(b, w, up)[0])


@pytest.mark.parametrize("kind", ["one", "half", "natural", "bad", "rows"])
@pytest.mark.parametrize("N", [63, 1000, 1024, 1025])
def test_lookup_grad_few_tokens(dev, kind, N):
    """The same uneven tokens in short lists, around the sums' and the sort's
    chunks, and many tokens of few neighbouring rows."""
    V, H = 4099, 2120
    gen = torch.Generator(device=dev).manual_seed(6)
    ids = torch.randint(0, V, (N,), generator=gen, device=dev)
    if kind == "one":
        ids[:] = 77
    elif kind == "half":
        ids[torch.rand(N, generator=gen, device=dev) < 0.5] = V - 1
    elif kind == "natural":
        ids = (V ** torch.rand(N, generator=gen, device=dev, dtype=torch.float64)).long() - 1
    elif kind == "bad":
        ids[::3], ids[1::3] = -7, V + 12
    else:
        ids = ids % 16 + 48
    g = torch.randn((N, H), generator=gen, device=dev).to(BF16)
    for padding in (None, int(ids[0].clamp(0, V - 1))):
        dw = ops.vocab_lookup_grad(g, ids, V, 0.5, padding, F32)
        _check_grad(dw, ids, g, V, 0.5, padding)
    into = torch.randn((V, H), generator=gen, device=dev)
    before = into.clone()
    ops.vocab_lookup_grad(g, ids.int(), V, into=into)
    _check_grad(into, ids, g, V, 1.0, None, before)


@pytest.mark.parametrize("shape", [(0,), (7,), (2, 3), (1, 0, 4)])
def test_lookup_backward_takes_any_gradient(dev, shape):
    """Contiguous, broadcast and strided gradients, ids of any shape and stride,
    with and without a graph of the gradient (which ends there)."""
    V, H = 19, 40
    gen = torch.Generator(device=dev).manual_seed(3)
    w = torch.randn((V, H), generator=gen, device=dev, requires_grad=True)
    wide = torch.randint(0, V, (*shape, 2), generator=gen, device=dev)
    for ids in (wide[..., 0], wide[..., 0].contiguous(), wide[..., 0].contiguous().to(torch.int32)):
        up = torch.randn((*shape, H), generator=gen, device=dev)
        for g in (up, up[..., :1].expand(up.shape), torch.stack((up, up), -1)[..., 0]):
            for graph in (False, True):
                out = embedding(ids, w, out_dtype=F32)
                (dw,) = torch.autograd.grad(out, w, g, create_graph=graph)
                _check_grad(dw.detach(), ids.reshape(-1).long(), g.reshape(-1, H), V, 1.0, None)
        if graph and dw.requires_grad:
            with pytest.raises(RuntimeError, match="once_differentiable"):
                torch.autograd.grad(dw.sum(), w)


def test_method_embeddings_of_other_tables(dev):
    """Tables and scales that the kernel does not read as they are keep the
    methods' results: strided codes, parameters that ask for gradients, float32."""
    w, s = _table(dev, 60, 64, E4)
    ids = torch.randint(0, 60, (11,), device=dev)
    want = w.view(torch.uint8)[ids].view(E4).to(BF16) * s[ids].to(BF16).unsqueeze(-1)
    layer = torch.nn.Module()
    layer.params_dtype, layer.weight_scale = BF16, s
    for table in (w, w.t().contiguous().t(), w.clone().requires_grad_()):
        layer.weight = table
        assert torch.equal(Fp8LinearMethod.embedding(None, layer, ids), want)
    layer.weight, layer.weight_scale = w, s.clone().requires_grad_()
    out = Fp8LinearMethod.embedding(None, layer, ids)
    assert torch.equal(out, want) and out.requires_grad
    plain = torch.nn.Module()
    plain.weight = torch.randn((60, 64), device=dev)
    assert torch.equal(UnquantizedLinearMethod().embedding(plain, ids), plain.weight[ids])


@pytest.mark.parametrize("N", [65536, 65537, 70001])
def test_lookup_grad_long_lists(dev, N):
    """Around the token count from which a workgroup sums 64 entries instead of
    16; one token runs over hundreds of chunks."""
    V, H = 300, 40
    gen = torch.Generator(device=dev).manual_seed(7)
    ids = torch.randint(0, V, (N,), generator=gen, device=dev)
    ids[torch.rand(N, generator=gen, device=dev) < 0.4] = 123
    g = torch.randn((N, H), generator=gen, device=dev).to(BF16)
    dw = ops.vocab_lookup_grad(g, ids, V, 0.5, 7, F32)
    _check_grad(dw, ids, g, V, 0.5, 7)
    assert torch.equal(dw, ops.vocab_lookup_grad(g, ids, V, 0.5, 7, F32))
    # whole numbers: the sums are exact, so no entry is lost or taken twice
    g = torch.randint(-8, 9, (N, H), generator=gen, device=dev).float()
    want = torch.zeros((V, H), dtype=torch.float64, device=dev).index_add_(0, ids, g.double())
    assert torch.equal(ops.vocab_lookup_grad(g, ids.int(), V, dtype=F32).double(), want)
