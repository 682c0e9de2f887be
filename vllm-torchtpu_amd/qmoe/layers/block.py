"""What stands around the products of a transformer block, for training and
serving: the norms before and after it with its gate and the residual
(``block_norm``, ``block_residual``), and a gated activation and a linear layer
whose inputs wait for the backward pass in 8 bits (``checkpointed_activation``,
``checkpointed_linear``). The reference serves only and leaves norms to the model:
no counterpart.

Each runs straight on the C ABI in eager mode and as a torch custom op
(``torch.ops.qmoe.block_residual`` ...) under a trace, a dispatch mode, `torch.vmap` and
fake tensors, as the vocabulary's operators do. Gradients come from
`torch.autograd.Function`s; there is no second derivative and no forward-mode
derivative, and a tangent is refused, as is a gradient that is asked for inside a
functorch transform (`torch.func.grad` ...; through a batch of `torch.vmap`, whose
operands do not say that they require one, the backward pass is an error).

8 bits: per 32 columns e4m3 codes and a power of two, the least with which none
of them saturates. A value is off by at most 2^-4 of itself, or 2^-10 of the
power of two where that is more; infinities and NaN become NaN.
"""

from typing import Optional, Tuple

import torch

from qmoe import ops


def _wants(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ---------------------------------------------------------------- norms, gate, residual


@torch.library.custom_op("qmoe::block_residual", mutates_args=())
def _block_op(y: Optional[torch.Tensor], residual: torch.Tensor, gate: Optional[torch.Tensor],
              norm_weight: Optional[torch.Tensor], next_weight: Optional[torch.Tensor], scale: float,
              residual_scale: float, eps: float, weight_offset: float, z_dtype: torch.dtype,
              keep: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(a result that the call has not comes back empty)"""
    out = ops.block_residual(y, residual, gate, norm_weight, next_weight, scale, residual_scale, eps, weight_offset, z_dtype,
                             keep)
    return tuple(residual.new_empty(0) if t is None else t for t in out)


@_block_op.register_fake
def _(y, residual, gate, norm_weight, next_weight, scale, residual_scale, eps, weight_offset, z_dtype, keep):
    return (residual.new_empty(0 if y is None else residual.shape),
            residual.new_empty(0) if next_weight is None else residual.new_empty(residual.shape, dtype=z_dtype),
            residual.new_empty((2, residual.numel() // residual.shape[-1]), dtype=torch.float32) if keep else
            residual.new_empty(0))


@torch.library.custom_op("qmoe::block_residual_grad", mutates_args=())
def _block_grad_op(g_h: Optional[torch.Tensor], g_z: Optional[torch.Tensor], y: Optional[torch.Tensor], h: torch.Tensor,
                   gate: Optional[torch.Tensor], norm_weight: Optional[torch.Tensor], next_weight: Optional[torch.Tensor],
                   rstd: torch.Tensor, scale: float, residual_scale: float, eps: float, weight_offset: float,
                   z_dtype: torch.dtype, need_y: bool, need_residual: bool, need_gate: bool, need_norm: bool,
                   need_next: bool
                   ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    out = ops.block_residual_grad(g_h, g_z, y, h, gate, norm_weight, next_weight, rstd, scale, residual_scale, eps,
                                  weight_offset, z_dtype, (need_y, need_residual, need_gate, need_norm, need_next))
    return tuple(h.new_empty(0) if t is None else t for t in out)


@_block_grad_op.register_fake
def _(g_h, g_z, y, h, gate, norm_weight, next_weight, rstd, scale, residual_scale, eps, weight_offset, z_dtype,
      need_y, need_residual, need_gate, need_norm, need_next):
    wanted = ((y, need_y), (h, need_residual), (gate, need_gate), (norm_weight, need_norm),
              (next_weight, need_next and g_z is not None))
    return tuple(h.new_empty(0) if t is None or not n else t.new_empty(t.shape) for t, n in wanted)


class _Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, gate, norm_weight, next_weight, args):
        h, z, rstd, desc = _block(y, residual, gate, norm_weight, next_weight, args, True)
        saved = (y, residual if y is None else h, gate, norm_weight, next_weight, rstd)
        ctx.save_for_backward(*saved)
        ctx.args = args
        ctx.run = None if desc is None else ops.block_saved(desc, *saved)
        ctx.set_materialize_grads(False)
        return h, z

    @staticmethod
    def backward(ctx, g_h, g_z):
        if torch.is_grad_enabled():  # (a backward pass that records itself)
            return ops.once("block_residual", _Block._grads, ctx, g_h, g_z)
        return _Block._grads(ctx, g_h, g_z)

    @staticmethod
    def _grads(ctx, g_h, g_z):
        if g_h is None and g_z is None:
            return (None,) * 6
        saved, need = ctx.saved_tensors, ctx.needs_input_grad[:5]
        if ctx.run is not None and ops.plain_grad(g_h, g_z):
            grads = ops.block_grad_plain(ctx.run, g_h, g_z, saved, need)
            if grads is not None:
                return (*grads, None)
        if ops.eager_call(g_h, g_z, *saved):
            return (*ops.block_residual_grad(g_h, g_z, *saved, *ctx.args, need), None)
        ops.refuse_tangents("block_residual's gradients", g_h, g_z)
        grads = torch.ops.qmoe.block_residual_grad(g_h, g_z, *saved, *ctx.args, *need)
        there = (saved[0], saved[1], saved[2], saved[3], saved[4] if g_z is not None else None)
        return (*(g if n and t is not None else None for g, n, t in zip(grads, need, there)), None)


def _block(y, residual, gate, norm_weight, next_weight, args, keep):
    ts = (y, residual, gate, norm_weight, next_weight)
    if ops.eager_call(*ts):
        return ops.block_residual_desc(*ts, *args, keep)
    ops.refuse_tangents("block_residual", *ts)
    ops._check_block(*ts, args[-1], "block_residual")
    h, z, rstd = torch.ops.qmoe.block_residual(*ts, *args, keep)
    return None if y is None else h, None if next_weight is None else z, rstd if keep else None, None


def block_norm(x, weight, eps=1e-6, weight_offset=0.0, out_dtype=None):
    """The norm before a block: x (mean x^2 + eps)^(-1/2) (weight_offset + weight)
    over the last axis of ``x`` [..., H] (bf16, f16 or f32; H up to 16384), statistics in
    float32 (a row whose squares add up to infinity there gives zeros), rounded once to ``out_dtype`` (``x``'s type; of a float32 ``x`` also bf16
    or f16). Differentiable in ``x`` and ``weight``, with gradients of their types."""
    args = (1.0, 1.0, float(eps), float(weight_offset), x.dtype if out_dtype is None else out_dtype)
    if weight is None:
        raise ValueError("block_norm: a weight is required")
    if _wants(x, weight):
        ops.refuse_transforms("block_norm")
        return _Block.apply(None, x, None, None, weight, args)[1]
    return _block(None, x, None, None, weight, args, False)[1]


def block_residual(y, residual, gate=None, norm_weight=None, next_weight=None, scale=1.0, residual_scale=1.0, eps=1e-6,
                   weight_offset=0.0):
    """What follows a block with output ``y`` [..., H]:

        h = residual_scale residual + scale gate n(y; norm_weight),   z = n(h; next_weight)

    n: the norm of `block_norm`; without ``norm_weight`` y itself. Returns h, or (h, z)
    with ``next_weight``, the norm before the next block. h has the residual's type, y's
    or float32, and is rounded as it is stored before its norm; z has y's type.
    ``gate``: one value per channel [H], per token [..., 1] (either bf16, f16 or f32) or
    per element [..., H] (y's type), multiplied as it is; the two weights have one type.

    Differentiable in all five tensors through both results, with gradients of their
    types, from float32 sums in a fixed order. A gradient that reaches h only gives
    ``next_weight`` none."""
    if y is None:
        raise ValueError("block_residual: needs the block's output")
    args = (float(scale), float(residual_scale), float(eps), float(weight_offset), y.dtype)
    ts = (y, residual, gate, norm_weight, next_weight)
    if _wants(*ts):
        ops.refuse_transforms("block_residual")
        h, z = _Block.apply(*ts, args)
    else:
        h, z = _block(*ts, args, False)[:2]
    return h if next_weight is None else (h, z)


# ---------------------------------------------------------------- gated activation


@torch.library.custom_op("qmoe::act_checkpoint", mutates_args=())
def _act_op(gate_up: torch.Tensor, activation: str, keep: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    out = ops.act_checkpoint(gate_up, activation, keep)
    return tuple(gate_up.new_empty(0) if t is None else t for t in out)


@_act_op.register_fake
def _(gate_up, activation, keep):
    n = gate_up.shape[-1]
    T, I = gate_up.numel() // n, n // 2
    h = gate_up.new_empty((*gate_up.shape[:-1], I))
    if not keep:
        return h, gate_up.new_empty(0), gate_up.new_empty(0)
    return (h, gate_up.new_empty((T, n), dtype=torch.uint8),
            gate_up.new_empty((T, 2, (I + 31) // 32), dtype=torch.uint8))


@torch.library.custom_op("qmoe::act_checkpoint_grad", mutates_args=())
def _act_grad_op(codes: torch.Tensor, scales: torch.Tensor, grad: torch.Tensor, activation: str) -> torch.Tensor:
    return ops.act_checkpoint_grad(codes, scales, grad, activation)


@_act_grad_op.register_fake
def _(codes, scales, grad, activation):
    return grad.new_empty((*grad.shape[:-1], 2 * grad.shape[-1]))


class _Activation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate_up, activation):
        h, codes, scales = _act(gate_up, activation, True)
        ctx.save_for_backward(codes, scales)
        ctx.activation = activation
        ctx.run = None
        if ops.eager_call(gate_up) and h.numel():
            I = h.shape[-1]
            ctx.run = (codes.data_ptr(), scales.data_ptr(), h.shape, h.numel() // I, I, *ops.act_code(activation))
        return h

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():  # (as above)
            return ops.once("checkpointed_activation", _Activation._grads, ctx, grad)
        return _Activation._grads(ctx, grad)

    @staticmethod
    def _grads(ctx, grad):
        codes, scales = ctx.saved_tensors
        run = ctx.run
        if run is not None and ops.plain_grad(grad) and codes.data_ptr() == run[0] and scales.data_ptr() == run[1]:
            return ops.act_grad_run(codes, scales, grad, run[4], *run[2:]), None
        fn = ops.act_checkpoint_grad
        if not ops.eager_call(grad, codes, scales):
            ops.refuse_tangents("checkpointed_activation's gradient", grad)
            fn = torch.ops.qmoe.act_checkpoint_grad
        return fn(codes, scales, grad, ctx.activation), None


def _act(gate_up, activation, keep):
    if ops.eager_call(gate_up):
        return ops.act_checkpoint(gate_up, activation, keep)
    ops.refuse_tangents("checkpointed_activation", gate_up)
    ops._check_act(gate_up, activation, "checkpointed_activation")
    return torch.ops.qmoe.act_checkpoint(gate_up, activation, keep)


def checkpointed_activation(gate_up, activation="silu"):
    """act(gate, up) of ``gate_up`` [..., 2 I] ([gate | up], bf16 or f16) -> [..., I] of
    its type, ``activation`` as in the fused expert products ("silu", "swigluoai",
    "gelu", "silu_and_mul_with_clamp", "situ:...").

    When a gradient is asked for, the 8 bits of gate and up are kept instead of
    their 16 (2 I + 2 ceil(I / 32) bytes a row), and the derivatives are those at the
    8-bit values; a clamp passes the gradient up to its limits. The result itself comes
    from the 16-bit values."""
    if _wants(gate_up):
        ops.refuse_transforms("checkpointed_activation")
        return _Activation.apply(gate_up, activation)
    return _act(gate_up, activation, False)[0]


# ---------------------------------------------------------------- linear layer


@torch.library.custom_op("qmoe::linear_checkpoint", mutates_args=())
def _linear_op(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
               keep: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    out = ops.linear_checkpoint(x, weight, bias, keep)
    return tuple(x.new_empty(0) if t is None else t for t in out)


@_linear_op.register_fake
def _(x, weight, bias, keep):
    K = x.shape[-1]
    T = x.numel() // K
    y = x.new_empty((*x.shape[:-1], weight.shape[0]))
    if not keep:
        return y, x.new_empty(0), x.new_empty(0)
    return y, x.new_empty((T, K), dtype=torch.uint8), x.new_empty((T, K // 32), dtype=torch.uint8)


@torch.library.custom_op("qmoe::linear_grad", mutates_args=())
def _linear_grad_op(grad: torch.Tensor, weight: torch.Tensor, codes: Optional[torch.Tensor],
                    scales: Optional[torch.Tensor], need_x: bool, need_weight: bool,
                    bias_dtype: Optional[torch.dtype]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    out = ops.linear_grad(grad, weight, codes, scales, need_x, need_weight, bias_dtype)
    return tuple(grad.new_empty(0) if t is None else t for t in out)


@_linear_grad_op.register_fake
def _(grad, weight, codes, scales, need_x, need_weight, bias_dtype):
    return (grad.new_empty((*grad.shape[:-1], weight.shape[1]) if need_x else 0),
            grad.new_empty(weight.shape if need_weight else 0),
            grad.new_empty(0) if bias_dtype is None else grad.new_empty(weight.shape[0], dtype=bias_dtype))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        keep = ctx.needs_input_grad[1]
        y, codes, scales = _linear(x, weight, bias, keep)
        ctx.save_for_backward(weight, *((codes, scales) if keep else (None, None)))
        ctx.bias_dtype = bias.dtype if bias is not None and ctx.needs_input_grad[2] else None
        ctx.run = None
        if ops.eager_call(x, weight, bias) and y.numel():
            N, K = weight.shape
            at = (codes.data_ptr(), scales.data_ptr()) if keep else (0, 0)
            ctx.run = (weight.data_ptr(), *at, N, y.shape, y.numel() // N, N, K)
        return y

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():  # (as above)
            return ops.once("checkpointed_linear", _Linear._grads, ctx, grad)
        return _Linear._grads(ctx, grad)

    @staticmethod
    def _grads(ctx, grad):
        weight, codes, scales = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        run = ctx.run
        if run is not None and ops.plain_grad(grad) and grad.data_ptr() % 16 == 0 and weight.data_ptr() == run[0] and \
                (codes is None or (codes.data_ptr() == run[1] and scales.data_ptr() == run[2])):
            return ops.linear_grad_run(grad, *run[3:], weight, codes, scales, need_x, need_w, ctx.bias_dtype)
        fn = ops.linear_grad
        if not ops.eager_call(grad, weight, codes, scales):
            ops.refuse_tangents("checkpointed_linear's gradients", grad)
            fn = torch.ops.qmoe.linear_grad
        dx, dw, db = fn(grad, weight, codes, scales, need_x, need_w, ctx.bias_dtype)
        return (dx if need_x else None), (dw if need_w else None), (db if ctx.bias_dtype is not None else None)


def _linear(x, weight, bias, keep):
    if ops.eager_call(x, weight, bias):
        return ops.linear_checkpoint(x, weight, bias, keep)
    ops.refuse_tangents("checkpointed_linear", x, weight, bias)
    ops._check_linear(x, weight, bias, "checkpointed_linear")
    return torch.ops.qmoe.linear_checkpoint(x, weight, bias, keep)


def checkpointed_linear(x, weight, bias=None):
    """x weight^T + bias: bf16 ``x`` [..., K] and ``weight`` [N, K] (K a multiple of 32, N
    of 8), bias [N] bf16 or f32 -> bf16 [..., N]: float32 sums, the bias added before
    the one rounding.

    When the weight's gradient is asked for, the 8 bits of ``x`` are kept instead of
    its 16 (33/32 bytes a value), and that gradient is dy^T x8; those of ``x`` and the
    bias are exact. bf16 gradients (the bias's in its type) from float32 sums in a
    fixed order."""
    if _wants(x, weight, bias):
        ops.refuse_transforms("checkpointed_linear")
        return _Linear.apply(x, weight, bias)
    return _linear(x, weight, bias, False)[0]
