"""The vocabulary table's two ends: token rows in, scored tokens out.

``embedding`` is the lookup behind the quant methods' ``embedding``
(`layers/adapter/quantization/fp8.py:1692-1698`) with the scaling that some
models put behind it, and its gradient for a bf16 or f32 table.
``vocab_cross_entropy`` scores tokens against the output projection (the tied
table of `fp8.py:1679-1681`) without the [T, V] logits, and its gradients.

Both run as torch custom ops (``torch.ops.qmoe.vocab_lookup`` ...) under a
trace, a dispatch mode, a functorch transform and fake tensors, and straight on
the C ABI in eager mode: the op's dispatch takes longer than a decode step's
lookup. Gradients come from `torch.autograd.Function`s around them; there is no
forward-mode derivative, and a tangent is refused.
"""

from typing import Optional, Tuple

import torch

from qmoe import ops


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
    def backward(ctx, grad):
        # (autograd runs this with gradients off; with create_graph the decorator puts the error for a second pass behind it)
        if torch.is_grad_enabled():
            return _Embedding._once(ctx, grad)
        return _Embedding._grads(ctx, grad)

    @staticmethod
    def _grads(ctx, grad):
        (ids,) = ctx.saved_tensors
        vocab, scale, padding_idx, dtype = ctx.args
        if torch.compiler.is_compiling() or ops.watched() or type(grad) is not torch.Tensor or not grad.is_contiguous() or \
                not ids.is_contiguous() or grad.get_device() != torch.cuda.current_device():
            ops.refuse_tangents("embedding's gradient", grad)
            fn = ops.vocab_lookup_grad if ops.eager_call(grad, ids) else torch.ops.qmoe.vocab_lookup_grad
            return None, fn(grad, ids, vocab, scale, padding_idx, dtype), None, None, None
        H = grad.shape[-1]
        dw = ops.lookup_grad_run(grad, H, ids if ids.dim() == 1 else ids.view(-1), vocab, H, scale,
                                 -1 if padding_idx is None else padding_idx, dtype)
        return None, dw, None, None, None

    _once = staticmethod(torch.autograd.function.once_differentiable(_grads.__func__))


def _lookup(ids, weight, weight_scale, scale, out_dtype):
    if ops.eager_call(ids, weight, weight_scale):
        return ops.vocab_lookup(ids, weight, weight_scale, scale, out_dtype)
    ops.refuse_tangents("embedding", weight, weight_scale)
    ops._check_table(weight, weight_scale, "embedding")
    ops._check_ids(ids, "embedding: ids")
    return torch.ops.qmoe.vocab_lookup(ids, weight, weight_scale, scale, out_dtype)


def embedding(ids, weight, weight_scale=None, scale=1.0, padding_idx=None, out_dtype=torch.bfloat16):
    """Rows ``ids`` (int32 or int64, any shape) of the table ``weight`` [V, H]:
    round(scale * s[id] * w[id]) as ``out_dtype`` [*ids.shape, H].

    The table is bf16 or f32, or 1-byte codes (e4m3, e5m2, int8) with one float32
    scale per row, which is rounded to ``out_dtype`` before the product. An id
    outside the table gives a row of NaN. A bf16 or f32 table that requires a
    gradient gets one (in its own type, from float32 sums in a fixed order: the
    same bits for the same ids and gradients); ``padding_idx`` names the row that
    gets none."""
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"embedding: padding_idx {padding_idx} is outside the table of {weight.shape[0]} rows")
    scale = float(scale)
    if torch.is_grad_enabled() and (weight.requires_grad or (weight_scale is not None and weight_scale.requires_grad)):
        if weight_scale is not None:
            raise NotImplementedError("embedding: no gradient for a table of 1-byte codes or its scales")
        if out_dtype == torch.float16:
            raise NotImplementedError("embedding: gradients flow through bf16 or f32 outputs, not f16")
        return _Embedding.apply(ids, weight, scale, padding_idx, out_dtype)
    return _lookup(ids, weight, weight_scale, scale, out_dtype)


# ---------------------------------------------------------------- cross entropy


@torch.library.custom_op("qmoe::vocab_loss", mutates_args=())
def _loss_op(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, weight_scale: Optional[torch.Tensor],
             ignore_index: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return ops.vocab_loss(x, weight, targets, weight_scale, ignore_index)


@_loss_op.register_fake
def _(x, weight, targets, weight_scale, ignore_index):
    return x.new_empty(targets.shape, dtype=torch.float32), x.new_empty(targets.shape, dtype=torch.float32)


@torch.library.custom_op("qmoe::vocab_loss_grad", mutates_args=())
def _loss_grad_op(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, g_loss: torch.Tensor,
                  g_lse: Optional[torch.Tensor], weight_scale: Optional[torch.Tensor], ignore_index: int, need_x: bool,
                  need_weight: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """(a gradient that is not asked for comes back empty)"""
    dx, dw = ops.vocab_loss_grad(x, weight, targets, lse, g_loss, g_lse, weight_scale, ignore_index, need_x, need_weight)
    return (x.new_empty(0) if dx is None else dx), (x.new_empty(0) if dw is None else dw)


@_loss_grad_op.register_fake
def _(x, weight, targets, lse, g_loss, g_lse, weight_scale, ignore_index, need_x, need_weight):
    return x.new_empty(x.shape if need_x else 0), x.new_empty(weight.shape if need_weight else 0)


class _VocabCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, weight_scale, ignore_index):
        loss, lse = _loss(x, weight, targets, weight_scale, ignore_index)
        ctx.save_for_backward(x, weight, targets, weight_scale, lse)
        ctx.ignore_index = ignore_index
        ctx.set_materialize_grads(False)
        return loss, lse

    @staticmethod
    def backward(ctx, g_loss, g_lse):
        if torch.is_grad_enabled():  # (as above)
            return _VocabCrossEntropy._once(ctx, g_loss, g_lse)
        return _VocabCrossEntropy._grads(ctx, g_loss, g_lse)

    @staticmethod
    def _grads(ctx, g_loss, g_lse):
        x, weight, targets, weight_scale, lse = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        if g_loss is None and g_lse is None:
            return None, None, None, None, None
        if g_loss is None:
            g_loss = torch.zeros_like(g_lse)
        fn = ops.vocab_loss_grad
        if not ops.eager_call(x, weight, g_loss, g_lse):
            ops.refuse_tangents("vocab_cross_entropy's gradients", g_loss, g_lse)
            fn = torch.ops.qmoe.vocab_loss_grad
        dx, dw = fn(x, weight, targets, lse, g_loss, g_lse, weight_scale, ctx.ignore_index, need_x, need_w)
        return (dx if need_x else None), (dw if need_w else None), None, None, None

    _once = staticmethod(torch.autograd.function.once_differentiable(_grads.__func__))


def _loss(x, weight, targets, weight_scale, ignore_index):
    if ops.eager_call(x, weight, targets, weight_scale):
        return ops.vocab_loss(x, weight, targets, weight_scale, ignore_index)
    ops.refuse_tangents("vocab_cross_entropy", x, weight, weight_scale)
    ops._check_loss(x, weight, targets, weight_scale, "vocab_cross_entropy")
    return torch.ops.qmoe.vocab_loss(x, weight, targets, weight_scale, ignore_index)


def unpadded_rows(weight, weight_scale, vocab_size):
    """The first ``vocab_size`` rows of a table and their scales (None: all); the
    rows of a table padded beyond its vocabulary have logits too, which are not
    the model's."""
    if vocab_size is None:
        return weight, weight_scale
    if not 0 < vocab_size <= weight.shape[0]:
        raise ValueError(f"cross_entropy: vocab_size {vocab_size} of a table of {weight.shape[0]} rows")
    return weight[:vocab_size], None if weight_scale is None else weight_scale.reshape(-1)[:vocab_size]


def vocab_cross_entropy(x, weight, targets, weight_scale=None, ignore_index=-100):
    """Cross entropy of the targets (int32 or int64 [...]) under softmax(x .
    w^T): (loss, lse), float32 of the targets' shape, without the logits in
    memory. ``-loss`` is the targets' log-probability, ``lse`` the log of the
    sum of exponentials.

    ``x`` is bf16 [..., H]; ``weight`` [V, H] bf16, or 1-byte codes (e4m3, e5m2,
    int8) with one float32 scale per row, the layout `Fp8LinearMethod` keeps an
    embedding table in; H a multiple of 8. ``ignore_index`` marks tokens that
    are not scored (loss 0, no gradient of the loss; padding rows may hold
    anything); another target outside the table gives a NaN loss.

    Differentiable in ``x`` and in a bf16 ``weight`` through both results
    (gradients in bf16; a table of codes is frozen). The sums' order is fixed:
    the same bits on every call."""
    ignore_index = int(ignore_index)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (weight_scale is not None and weight_scale.requires_grad)):
        if weight_scale is not None and (weight.requires_grad or weight_scale.requires_grad):
            raise NotImplementedError("vocab_cross_entropy: no gradient for a table of 1-byte codes or its scales")
        return _VocabCrossEntropy.apply(x, weight, targets, weight_scale, ignore_index)
    return _loss(x, weight, targets, weight_scale, ignore_index)
