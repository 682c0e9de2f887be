"""MoE routing (the reference's `moe_routing` / `router_topk` adapters).

``select_experts`` mirrors `layers/adapter/moe_routing.py:232-323`,
``route`` mirrors `:150-186`, and ``rowmax_select`` mirrors
`layers/adapter/router_topk.py:42-50`. Scores, the sort-free top-k (ties to
the lowest expert id), grouped selection, renormalization and scaling all run
in one HIP kernel (`qmoe_moe_route`), registered as the torch custom op
``torch.ops.qmoe.moe_route`` with a fake implementation (the reference
registers its router op the same way, `layers/adapter/router_topk.py:36-39`).

``balanced_experts`` is the router in training: the same choice with the balance
loss, per-expert counts and the logits' gradient (no reference counterpart, which
serves only).
"""

from typing import Optional, Tuple

import torch

from qmoe import ops


@torch.library.custom_op("qmoe::moe_route", mutates_args=())
def _moe_route_op(logits: torch.Tensor, topk: int, scoring_func: str, renormalize: bool,
                  bias: Optional[torch.Tensor], routed_scaling_factor: float, num_expert_group: int,
                  topk_group: int, weights_f32: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return ops.moe_route(logits, topk, scoring_func, renormalize, bias, routed_scaling_factor,
                         num_expert_group, topk_group, weights_f32)


@_moe_route_op.register_fake
def _(logits, topk, scoring_func, renormalize, bias, routed_scaling_factor, num_expert_group, topk_group,
      weights_f32):
    T = logits.numel() // logits.shape[-1]
    w = logits.new_empty((T, topk), dtype=torch.float32 if weights_f32 else torch.bfloat16)
    return w, logits.new_empty((T, topk), dtype=torch.int32)


@torch.library.custom_op("qmoe::moe_route_hash", mutates_args=())
def _moe_route_hash_op(logits: torch.Tensor, topk: int, table: torch.Tensor, input_ids: torch.Tensor,
                       scoring_func: str, renormalize: bool,
                       routed_scaling_factor: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return ops.moe_route_hash(logits, topk, table, input_ids, scoring_func, renormalize, routed_scaling_factor)


@_moe_route_hash_op.register_fake
def _(logits, topk, table, input_ids, scoring_func, renormalize, routed_scaling_factor):
    T = logits.numel() // logits.shape[-1]
    return (logits.new_empty((T, topk), dtype=torch.bfloat16), logits.new_empty((T, topk), dtype=torch.int32))


def _route(logits, topk, scoring_func, renormalize, bias=None, routed_scaling_factor=1.0,
           num_expert_group=1, topk_group=1, weights_f32=False):
    """Host-side checks (raised at trace time), then the custom op."""
    if scoring_func not in ops._SCORING:
        raise NotImplementedError(f"FusedMoE does not support {scoring_func} scoring function for TPU.")
    if topk > logits.shape[-1]:
        raise ValueError(f"topk k={topk} exceeds the expert count {logits.shape[-1]}")
    return torch.ops.qmoe.moe_route(logits, int(topk), scoring_func, bool(renormalize), bias,
                                    float(routed_scaling_factor), int(num_expert_group or 1),
                                    int(topk_group or 1), bool(weights_f32))


def rowmax_select(scores: torch.Tensor, topk: int):
    """Top-k of float scores without a sort: (values f32 [R, k], ids int32).

    Scores at or below -3e38 (and NaN) are clamped to -3e38; a row with no
    score above it returns NaN values (`layers/core/rowmax_topk.py:28-61`).
    """
    n = scores.shape[-1]
    if topk > n:
        raise ValueError(f"topk k={topk} exceeds the expert count {n}")
    w, ids = _route(scores.float(), topk, "none", False, weights_f32=True)
    return w.reshape(*scores.shape[:-1], topk), ids.reshape(*scores.shape[:-1], topk)


def routing_params(layer):
    """The layer's routing settings as `select_experts` reads them: (bias,
    routed_scaling_factor, num_expert_group, topk_group); grouped selection
    only when `use_grouped_topk` with num_expert_group > 1 and topk_group <
    num_expert_group (`moe_routing.py:276-299`)."""
    bias = getattr(layer, "e_score_correction_bias", None) if layer is not None else None
    rsf = getattr(layer, "routed_scaling_factor", 1.0) if layer is not None else 1.0
    ng, tg = 1, 1
    if (layer is not None and getattr(layer, "use_grouped_topk", False)
            and layer.num_expert_group > 1 and layer.topk_group < layer.num_expert_group):
        ng, tg = layer.num_expert_group, layer.topk_group
    return bias, (rsf if rsf is not None else 1.0), ng, tg


def select_experts(hidden_states, router_logits, *, topk, renormalize, scoring_fn, layer=None,
                   input_ids=None):
    """(topk_weights in the hidden dtype, topk_ids int32), `moe_routing.py:232-323`.

    Grouped selection (`layer.use_grouped_topk` with ``num_expert_group > 1``
    and ``topk_group < num_expert_group``) uses the DeepSeek-V3 rule that the
    reference delegates to upstream vLLM (`:276-299`).
    """
    table = getattr(layer, "hash_indices_table", None) if layer is not None else None
    if table is not None and input_ids is not None:
        # DeepSeek-V4 hash routing (`moe_routing.py:259-274`): ids from the
        # table row of each token's input id, weights from its scores
        rsf = getattr(layer, "routed_scaling_factor", 1.0)
        if scoring_fn not in ops._SCORING:
            raise NotImplementedError(f"FusedMoE does not support {scoring_fn} scoring function for TPU.")
        w, ids = torch.ops.qmoe.moe_route_hash(router_logits, int(topk), table, input_ids, scoring_fn,
                                               bool(renormalize), float(rsf if rsf is not None else 1.0))
        return w.to(hidden_states.dtype), ids
    bias, rsf, ng, tg = routing_params(layer)
    w, ids = _route(router_logits, topk, scoring_fn, renormalize, bias=bias, routed_scaling_factor=rsf,
                    num_expert_group=ng, topk_group=tg)
    return w.to(hidden_states.dtype), ids


def route(layer, hidden_states, router_logits, input_ids=None):
    """Routing entry of the MoE methods, `moe_routing.py:150-186`: a
    model-supplied ``custom_routing_function`` wins, else `select_experts`."""
    topk = layer.moe_config.experts_per_token
    custom = getattr(layer, "custom_routing_function", None)
    if custom is not None:
        return custom(hidden_states=hidden_states, gating_output=router_logits, topk=topk,
                      renormalize=layer.renormalize)
    return select_experts(hidden_states, router_logits, topk=topk, renormalize=layer.renormalize,
                          scoring_fn=layer.scoring_func, layer=layer, input_ids=input_ids)


# ---------------------------------------------------------------- balanced routing


@torch.library.custom_op("qmoe::moe_balance", mutates_args=())
def _balance_op(logits: torch.Tensor, topk: int, scoring_func: str, renormalize: bool, bias: Optional[torch.Tensor],
                routed_scaling_factor: float, num_expert_group: int, topk_group: int,
                token_mask: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return ops.moe_balance(logits, topk, scoring_func, renormalize, bias, routed_scaling_factor, num_expert_group,
                           topk_group, token_mask)


@_balance_op.register_fake
def _(logits, topk, scoring_func, renormalize, bias, routed_scaling_factor, num_expert_group, topk_group, token_mask):
    T, E = logits.shape
    return (logits.new_empty((T, topk), dtype=torch.float32), logits.new_empty((T, topk), dtype=torch.int32),
            logits.new_empty((), dtype=torch.float32), logits.new_empty(E, dtype=torch.int32))


@torch.library.custom_op("qmoe::moe_balance_grad", mutates_args=())
def _balance_grad_op(logits: torch.Tensor, topk_ids: torch.Tensor, counts: torch.Tensor, g_weights: Optional[torch.Tensor],
                     g_loss: Optional[torch.Tensor], scoring_func: str, renormalize: bool, routed_scaling_factor: float,
                     token_mask: Optional[torch.Tensor]) -> torch.Tensor:
    return ops.moe_balance_grad(logits, topk_ids, counts, g_weights, g_loss, scoring_func, renormalize,
                                routed_scaling_factor, token_mask)


@_balance_grad_op.register_fake
def _(logits, topk_ids, counts, g_weights, g_loss, scoring_func, renormalize, routed_scaling_factor, token_mask):
    return torch.empty_like(logits)


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, args, bias, token_mask):
        w, ids, loss, counts = _balance(logits, topk, args, bias, token_mask)
        ctx.save_for_backward(logits, ids, counts, token_mask)
        ctx.args = args[:3]
        ctx.run = None
        if ops.eager_call(logits, bias, token_mask) and logits.numel() and logits.is_contiguous() and \
                (token_mask is None or token_mask.is_contiguous()):
            at = ops._addresses((logits, ids, counts, token_mask))
            ctx.run = (at, *logits.shape, topk, ops._SCORING[args[0]], *args[1:3])
        ctx.mark_non_differentiable(ids, counts)
        ctx.set_materialize_grads(False)
        return w, ids, loss, counts

    @staticmethod
    def backward(ctx, g_w, g_ids, g_loss, g_counts):
        if torch.is_grad_enabled():  # (a backward pass that records itself)
            return ops.once("balanced_experts", _Balance._grads, ctx, g_w, g_ids, g_loss, g_counts)
        return _Balance._grads(ctx, g_w, g_ids, g_loss, g_counts)

    @staticmethod
    def _grads(ctx, g_w, g_ids, g_loss, g_counts):
        if g_w is None and g_loss is None:
            return (None,) * 5
        logits, ids, counts, mask = saved = ctx.saved_tensors
        run = ctx.run
        if run is not None and ops.plain_grad(g_w, g_loss) and ops._addresses(saved) == run[0]:
            return ops.balance_grad_run(logits, ids, counts, g_w, g_loss, *run[1:], mask), None, None, None, None
        fn = ops.moe_balance_grad
        if not ops.eager_call(logits, ids, counts, g_w, g_loss, mask):
            ops.refuse_tangents("balanced_experts' gradient", g_w, g_loss)
            fn = torch.ops.qmoe.moe_balance_grad
        return fn(logits, ids, counts, g_w, g_loss, *ctx.args, mask), None, None, None, None


def _balance(logits, topk, args, bias, token_mask):
    scoring_func, renormalize, rsf, ng, tg = args
    if ops.eager_call(logits, bias, token_mask):
        return ops.moe_balance(logits, topk, scoring_func, renormalize, bias, rsf, ng, tg, token_mask)
    ops.refuse_tangents("balanced_experts", logits, bias)
    ops._check_balance(logits, topk, scoring_func, bias, ng, tg, token_mask, "balanced_experts")
    return torch.ops.qmoe.moe_balance(logits, topk, scoring_func, renormalize, bias, rsf, ng, tg, token_mask)


def balanced_experts(router_logits, topk, scoring_func="softmax", renormalize=True, e_score_correction_bias=None,
                     routed_scaling_factor=1.0, num_expert_group=1, topk_group=1, token_mask=None):
    """Routing for training, and for watching a server's load: (topk_weights f32
    [T, k], topk_ids int32 [T, k], balance_loss f32 [], expert_counts int32 [E]) of
    router logits [T, E] (bf16, f32, or another float type taken as f32).

    Experts and weights as `select_experts` chooses them (scoring "softmax",
    "sigmoid" or "sqrtsoftplus"), the weights not rounded. Over the N tokens of
    ``token_mask`` (bool [T]; None: all), with f[e] the share of their k N routes that
    expert e has and P[e] the mean of their scores' share of e (softmax: the score; else
    over the row's sum, of at least 1e-20):

        balance_loss = E sum_e f[e] P[e]          (1 for an even load; 0 for N = 0)

    ``expert_counts`` are those routes. A token outside the mask gets weights 0, and no
    gradient whatever its logits are. Differentiable in the logits through the
    weights and the loss (through P; the choice and f are constants), in their type, by
    `torch.autograd` (under functorch transforms the call is refused where a gradient is
    asked for); the correction bias only chooses and has no gradient. The sums' order is
    fixed. The fused expert layers here serve only: a gradient of the weights comes from
    experts that are differentiable themselves."""
    if torch.is_grad_enabled() and e_score_correction_bias is not None and e_score_correction_bias.requires_grad:
        raise NotImplementedError("balanced_experts: no gradient for the correction bias, which only chooses")
    if router_logits.dtype not in (torch.bfloat16, torch.float32) and router_logits.is_floating_point():
        router_logits = router_logits.float()
    args = (scoring_func, bool(renormalize), float(routed_scaling_factor), int(num_expert_group or 1),
            int(topk_group or 1))
    topk = int(topk)
    if torch.is_grad_enabled() and router_logits.requires_grad:
        ops.refuse_transforms("balanced_experts")
        return _Balance.apply(router_logits, topk, args, e_score_correction_bias, token_mask)
    return _balance(router_logits, topk, args, e_score_correction_bias, token_mask)
