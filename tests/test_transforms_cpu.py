"""Gradients asked for inside functorch transforms are refused by the operators' own
error, before anything is launched; what asks for none goes on to the checks of its
operands (CPU tensors are refused there)."""

import pytest
import torch

from qmoe.layers.block import block_norm, block_residual, checkpointed_activation, checkpointed_linear
from qmoe.layers.moe_routing import balanced_experts
from qmoe.layers.quantization.unquantized import UnquantizedLinearMethod
from qmoe.layers.vocab import embedding, vocab_cross_entropy

BF16 = torch.bfloat16
W = torch.ones(32, dtype=BF16)
TABLE = torch.zeros((8, 32), dtype=BF16)
IDS = torch.zeros(4, dtype=torch.int64)
LAYER = torch.nn.Module()
LAYER.weight = torch.nn.Parameter(TABLE.clone())


def _first(v):
    return v[0] if isinstance(v, tuple) else v


# name -> function of rows [4, 32] that ask for a gradient
CALLS = {
    "block_norm": lambda x: block_norm(x, W),
    "block_residual": lambda x: block_residual(x, x.detach(), norm_weight=W, next_weight=W),
    "checkpointed_activation": checkpointed_activation,
    "checkpointed_linear": lambda x: checkpointed_linear(x, TABLE),
    "checkpointed_linear ": lambda x: UnquantizedLinearMethod().apply_checkpointed(LAYER, x),
    "balanced_experts": lambda x: balanced_experts(x, 2),
    "embedding": lambda x: embedding(IDS, x),
    "vocab_cross_entropy": lambda x: vocab_cross_entropy(x, TABLE, IDS),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("transform", ["grad", "vjp", "jacrev", "grad of a batch", "captured"])
def test_gradients_under_transforms_are_refused(name, transform):
    fn = CALLS[name]
    x = torch.zeros((4, 32), dtype=BF16)
    loss = lambda v: _first(fn(v)).float().sum()  # noqa: E731
    with pytest.raises(NotImplementedError, match=name.strip() + ".*functorch"):
        if transform == "grad":
            torch.func.grad(loss)(x)
        elif transform == "vjp":
            torch.func.vjp(loss, x)
        elif transform == "jacrev":
            torch.func.jacrev(loss)(x)
        elif transform == "grad of a batch":
            torch.vmap(torch.func.grad(loss))(x[None])
        else:  # an operand from outside the batch
            x.requires_grad_()
            torch.vmap(lambda v: v + _first(fn(x)).float().sum())(torch.zeros(2))


@pytest.mark.parametrize("name", [n for n in CALLS if n != "checkpointed_linear "])
def test_without_gradients_they_are_not(name):
    fn = CALLS[name]
    x = torch.zeros((2, 4, 32), dtype=BF16)
    with pytest.raises((ValueError, NotImplementedError)) as e:
        torch.vmap(lambda v: _first(fn(v)))(x)
    assert "functorch" not in str(e.value)
    with torch.no_grad(), pytest.raises((ValueError, NotImplementedError)) as e:
        torch.vmap(lambda v: _first(fn(v)))(x.requires_grad_())
    assert "functorch" not in str(e.value)
