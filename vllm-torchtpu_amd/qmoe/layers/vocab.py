"""The vocabulary table's two ends: token rows in, scored tokens out.

``embedding`` is the lookup behind the quant methods' ``embedding``
(`layers/adapter/quantization/fp8.py:1692-1698`) with the scaling that some
models put behind it, and its gradient for a bf16 or f32 table.

Both run as torch custom ops (``torch.ops.qmoe.vocab_lookup`` ...) under
`torch.compile` and fake tensors, and straight on the C ABI in eager mode: the
op's dispatch takes longer than a decode step's lookup. Gradients come from
`torch.autograd.Function`s around them.
"""

from typing import Optional

import torch

from qmoe import ops


def _eager(*ts):
    """Plain tensors outside of a trace: no dispatcher has to see the call."""
    return not torch.compiler.is_compiling() and all(
        t is None or type(t) in (torch.Tensor, torch.nn.Parameter) for t in ts)


# ---------------------------------------------------------------- lookup


@torch.library.custom_op("qmoe::vocab_lookup", mutates_args=())
def _lookup_op(ids: torch.Tensor, weight: torch.Tensor, weight_scale: Optional[torch.Tensor], scale: float,
               out_dtype: torch.dtype) -> torch.Tensor:
    return ops.vocab_lookup(ids, weight, weight_scale, scale, out_dtype)


@_lookup_op.register_fake
def _(ids, weight, weight_scale, scale, out_dtype):
    return weight.new_empty((*ids.shape, weight.shape[1]), dtype=out_dtype)


@torch.library.custom_op("qmoe::vocab_lookup_grad", mutates_args=())
def _lookup_grad_op(grad: torch.Tensor, ids: torch.Tensor, vocab: int, scale: float, padding_idx: Optional[int],
                    dtype: torch.dtype) -> torch.Tensor:
    return ops.vocab_lookup_grad(grad, ids, vocab, scale, padding_idx, dtype)


@_lookup_grad_op.register_fake
def _(grad, ids, vocab, scale, padding_idx, dtype):
    return grad.new_empty((vocab, grad.shape[-1]), dtype=dtype)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, out_dtype):
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, padding_idx, weight.dtype)
        return _lookup(ids, weight, None, scale, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        fn = ops.vocab_lookup_grad if _eager(grad, ids) else torch.ops.qmoe.vocab_lookup_grad
        return None, fn(grad, ids, *ctx.args), None, None, None


def _lookup(ids, weight, weight_scale, scale, out_dtype):
    fn = ops.vocab_lookup if _eager(ids, weight, weight_scale) else torch.ops.qmoe.vocab_lookup
    return fn(ids, weight, weight_scale, scale, out_dtype)


def embedding(ids, weight, weight_scale=None, scale=1.0, padding_idx=None, out_dtype=torch.bfloat16):
    """Rows ``ids`` (int32 or int64, any shape) of the table ``weight`` [V, H]:
    round(scale * s[id] * w[id]) as ``out_dtype`` [*ids.shape, H].

    The table is bf16 or f32, or 1-byte codes (e4m3, e5m2, int8) with one float32
    scale per row, which is rounded to ``out_dtype`` before the product. An id
    outside the table gives a row of NaN. A bf16 or f32 table that requires a
    gradient gets one (in its own type, from float32 sums in token order, the
    same bits on every call); ``padding_idx`` names the row that gets none."""
    ops._check_table(weight, weight_scale, "embedding")
    ops._check_ids(ids, "embedding: ids")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"embedding: padding_idx {padding_idx} is outside the table of {weight.shape[0]} rows")
    scale = float(scale)
    if weight.requires_grad and torch.is_grad_enabled():
        if weight_scale is not None:
            raise NotImplementedError("embedding: no gradient for a table of 1-byte codes")
        if out_dtype == torch.float16:
            raise NotImplementedError("embedding: gradients flow through bf16 or f32 outputs, not f16")
        return _Embedding.apply(ids, weight, scale, padding_idx, out_dtype)
    return _lookup(ids, weight, weight_scale, scale, out_dtype)
