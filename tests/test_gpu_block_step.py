"""The block operators and the balanced router together, as a training step and a
decode step use them, and under traces, transforms, hooks and recomputation."""

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.checkpoint import checkpoint

from qmoe import ops
from qmoe.layers.block import block_norm, block_residual, checkpointed_activation, checkpointed_linear
from qmoe.layers.fused_moe import few_token_moe
from qmoe.layers.moe_routing import balanced_experts

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
T, H, I, E, K = 150, 256, 544, 48, 4
NAMES = ("x", "norm", "router", "up", "down", "post", "gate", "next")


def _data(dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def rand(shape, std=1.0, mean=0.0, dtype=BF16):
        return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dtype)

    leaves = (rand((T, H), dtype=F32), rand(H, 0.1, 1.0, F32), rand((E, H), 0.05), rand((2 * I, H), 0.05),
              rand((H, I), 0.05), rand(H, 0.1, 1.0, F32), rand((T, 1), 0.3, 0.5), rand(H, 0.1, 1.0, F32))
    ups = (rand((T, H), dtype=F32), rand((T, H)), rand((T, K), dtype=F32), torch.tensor(0.01, device=dev))
    return leaves, ups


def _step(x, norm, router, up, down, post, gate, nxt):
    """A block with a router beside its MLP: (h, z, routing weights, balance loss, counts)."""
    n = block_norm(x, norm, out_dtype=BF16)
    w, _, loss, counts = balanced_experts(checkpointed_linear(n, router), K)
    y = checkpointed_linear(checkpointed_activation(checkpointed_linear(n, up), "silu"), down)
    h, z = block_residual(y, x, gate, post, nxt, scale=0.5)
    return h, z, w, loss, counts


def _grads(leaves, ups):
    a = [t.detach().requires_grad_() for t in leaves]
    out = _step(*a)
    return [t.detach() for t in out], list(torch.autograd.grad(out[:4], a, ups))


def _by_hand(leaves, ups):
    """The same step, backward pass written out with the operators' own gradients."""
    x, norm, router, up, down, post, gate, nxt = leaves
    gh, gz, gw, gl = ups
    _, n, rs0 = ops.block_residual(None, x, None, None, norm, z_dtype=BF16, keep=True)
    lg, c1, s1 = ops.linear_checkpoint(n, router)
    w, ids, loss, counts = ops.moe_balance(lg, K)
    gu, c2, s2 = ops.linear_checkpoint(n, up)
    act, c3, s3 = ops.act_checkpoint(gu, "silu")
    y, c4, s4 = ops.linear_checkpoint(act, down)
    h, z, rs1 = ops.block_residual(y, x, gate, post, nxt, 0.5, keep=True)
    dy, dx, dgate, dpost, dnext = ops.block_residual_grad(gh, gz, y, h, gate, post, nxt, rs1, 0.5)
    dact, ddown, _ = ops.linear_grad(dy, down, c4, s4)
    dn, dup, _ = ops.linear_grad(ops.act_checkpoint_grad(c3, s3, dact, "silu"), up, c2, s2)
    dn2, drouter, _ = ops.linear_grad(ops.moe_balance_grad(lg, ids, counts, gw, gl), router, c1, s1)
    _, dx2, _, _, dnorm = ops.block_residual_grad(None, dn + dn2, None, x, None, None, norm, rs0, z_dtype=BF16)
    return [h, z, w, loss, counts], [dx + dx2, dnorm, drouter, dup, ddown, dpost, dgate, dnext]


def _equal(a, b):
    for p, q in zip(a, b):
        assert p.dtype == q.dtype and torch.equal(p, q)


def test_a_step_is_its_operators(dev):
    """Bit for bit (the two gradients that meet at n and at x are one addition each)."""
    leaves, ups = _data(dev)
    out, grads = _grads(leaves, ups)
    ref, want = _by_hand(leaves, ups)
    _equal(out, ref)
    _equal(grads, want)
    with torch.no_grad():
        _equal(_step(*leaves), out)


def test_a_step_against_float64(dev):
    """The whole step's gradients against float64 autograd of the plain formulas:
    bf16 roundings of six stages and the 8 bits' 2^-4 per value of two factors, which
    are independent from value to value, leave a few per cent of a gradient's norm."""
    leaves, ups = _data(dev)
    _, grads = _grads(leaves, ups)
    a = [t.double().requires_grad_() for t in leaves]
    x, norm, router, up, down, post, gate, nxt = a

    def n(v, w):
        return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w

    p = n(x, norm)
    s = torch.softmax(p @ router.t(), -1)
    _, ids, _, counts = balanced_experts(checkpointed_linear(block_norm(leaves[0], leaves[1], out_dtype=BF16), leaves[2]), K)
    top = s.gather(1, ids.long())
    loss = E / (K * T * T) * (counts.double() * s.sum(0)).sum()
    g, u = (p @ up.t()).chunk(2, -1)
    h = x + 0.5 * gate * n((torch.nn.functional.silu(g) * u) @ down.t(), post)
    out = (h, n(h, nxt), top / top.sum(-1, keepdim=True), loss)
    want = torch.autograd.grad(out, a, [v.double() for v in ups])
    for name, got, ref in zip(NAMES, grads, want):
        assert (got.double() - ref).norm() <= 0.05 * ref.norm(), name


def test_a_captured_step(dev):
    sets = [_data(dev, s) for s in (1, 2)]
    want = [[*o, *g] for o, g in (_grads(*s) for s in sets)]
    leaves, ups = [t.clone() for t in sets[0][0]], [t.clone() for t in sets[0][1]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _grads(leaves, ups)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, g = _grads(leaves, ups)
        graphs.append(graph)
        outs.append([*o, *g])
    for i, k in ((1, 0), (0, 1), (1, 1), (0, 0), (1, 0)):
        for s, t in zip((*leaves, *ups), (*sets[i][0], *sets[i][1])):
            s.copy_(t)
        graphs[k].replay()
        _grads(*sets[1 - i])
        torch.cuda.synchronize()
        _equal(outs[k], want[i])


def test_a_decode_step(dev):
    """Norm, few-token experts, residual and the next norm of one and of 16 tokens."""
    g = torch.Generator(device=dev).manual_seed(3)
    w1, w2 = (torch.randn(s, generator=g, device=dev).to(BF16) * 0.05 for s in ((E, 512, H), (E, H, 256)))
    norm, nxt = (torch.rand(H, generator=g, device=dev) + 0.5 for _ in range(2))
    for t in (1, 16):
        x = torch.randn((t, H), generator=g, device=dev).to(BF16)
        lg = torch.randn((t, E), generator=g, device=dev)
        y = few_token_moe(block_norm(x, norm), lg, w1, w2, None, None, None, None, K, "silu")
        h, z = block_residual(y, x, next_weight=nxt)
        _, ids, _, counts = balanced_experts(lg, K)
        assert torch.equal(z, block_norm(h, nxt)) and int(counts.sum()) == t * K
        assert torch.equal(h, (x.float() + y.float()).to(BF16))
        assert torch.equal(ids, ops.moe_route(lg, K)[1])


def test_backward_again_and_second_derivatives(dev):
    leaves, ups = _data(dev)
    a = [t.detach().requires_grad_() for t in leaves]
    out = _step(*a)
    one = torch.autograd.grad(out[:4], a, ups, retain_graph=True)
    _equal(one, torch.autograd.grad(out[:4], a, ups, retain_graph=True))
    first = torch.autograd.grad(out[:4], a, ups, create_graph=True)
    _equal(first, one)
    for g in first:
        with pytest.raises(RuntimeError, match="no second derivative"):
            (g.sum() + out[0].sum()).backward(retain_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), a[0], retain_graph=True)


def test_saved_tensor_hooks_and_recomputation(dev):
    leaves, ups = _data(dev)
    out, want = _grads(leaves, ups)
    with torch.autograd.graph.save_on_cpu():
        _equal(_grads(leaves, ups)[1], want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
        _equal(_grads(leaves, ups)[1], want)
    a = [t.detach().requires_grad_() for t in leaves]
    again = checkpoint(_step, *a, use_reentrant=False)
    _equal(torch.autograd.grad(again[:4], a, ups), want)
    # an operand written after the forward pass is an error, not a wrong gradient
    a = [t.detach().clone().requires_grad_() for t in leaves]
    out = _step(*a)
    with torch.no_grad():
        a[4].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out[0], a[4], ups[0])


def test_strided_saved_operands(dev):
    """Operands that the forward pass reads where they lie, rows apart, and gradients
    with strides of their own."""
    g = torch.Generator(device=dev).manual_seed(5)
    wide = torch.randn((40, 3 * H), generator=g, device=dev).to(BF16)
    y, r = wide[:, :H].detach().requires_grad_(), wide[:, H:2 * H].detach().requires_grad_()
    w = torch.ones(H, device=dev, dtype=BF16)
    gh, gz = wide[:, 2 * H:], torch.ones((1, H), device=dev, dtype=BF16).expand(40, H)
    got = torch.autograd.grad(block_residual(y, r, norm_weight=w, next_weight=w), (y, r), (gh, gz))
    yc, rc = y.detach().contiguous().requires_grad_(), r.detach().contiguous().requires_grad_()
    _equal(got, torch.autograd.grad(block_residual(yc, rc, norm_weight=w, next_weight=w), (yc, rc),
                                    (gh.contiguous(), gz.contiguous())))


def _calls(dev):
    """name -> (function of one operand, two inputs)"""
    leaves, _ = _data(dev)
    x, norm, router, up, down, post, gate, nxt = leaves
    two = lambda t: (t, t.flip(0) + 1)  # noqa: E731
    y = torch.randn((T, H), device=dev).to(BF16)
    return {"norm": (lambda v: block_norm(v, norm, out_dtype=BF16), two(x)),
            "residual": (lambda v: torch.cat(block_residual(v, x.to(BF16), gate, post, nxt), -1), two(y)),
            "activation": (lambda v: checkpointed_activation(v, "swigluoai"), two(y)),
            "linear": (lambda v: checkpointed_linear(v, up), two(y)),
            "balance": (lambda v: torch.cat([t.float().flatten() for t in balanced_experts(v, K)]), two(x))}


WHICH = ["norm", "residual", "activation", "linear", "balance"]


@pytest.mark.parametrize("which", WHICH)
def test_traces_and_batches(dev, which):
    fn, (a, b) = _calls(dev)[which]
    wa, wb = fn(a), fn(b)
    for traced in (make_fx(fn)(a), make_fx(fn, pre_dispatch=True)(a),
                   make_fx(fn, tracing_mode="fake", _allow_non_fake_inputs=True)(a),
                   torch.jit.trace(fn, (a,), check_trace=False), torch.compile(fn, backend="eager", fullgraph=True)):
        assert torch.equal(traced(b), wb) and torch.equal(traced(a), wa)
    assert torch.equal(torch.vmap(fn)(torch.stack((a, b))), torch.stack((wa, wb)))
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Mode():
        assert torch.equal(fn(a), wa)
    assert len([s for s in seen if s.startswith("qmoe.")]) == 1
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fn(fw.make_dual(a, torch.ones_like(a)))


@pytest.mark.parametrize("which", WHICH)
def test_gradients_under_traces(dev, which):
    fn, (a, b) = _calls(dev)[which]

    def grad(v):
        leaf = v.detach().requires_grad_()
        out = fn(leaf)
        return torch.autograd.grad(out, leaf, torch.ones_like(out))[0]

    wa, wb = grad(a), grad(b)
    traced = make_fx(grad)(a)
    assert torch.equal(traced(b), wb) and torch.equal(traced(a), wa)
    compiled = torch.compile(lambda v: fn(v).float().sum(), backend="aot_eager")
    for v, want in ((a, wa), (b, wb)):
        leaf = v.detach().requires_grad_()
        # (the sum's gradient is ones)
        assert torch.equal(torch.autograd.grad(compiled(leaf), leaf)[0], want)
    with fw.dual_level():
        leaf = a.detach().requires_grad_()
        out = fn(leaf)
        scaled = out * fw.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(scaled.sum(), leaf)
