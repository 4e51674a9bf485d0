"""The router of a MoE layer, on B200 (sm_100a): what stands before hex_moe, expert_mlp and int8_moe.

  route            softmax or sigmoid scores, a bias that balances the choice, groups of experts of which a
                   token may use a few, the k best, their weights renormalised and scaled; differentiable
  route_backward   its gradient for the logits

hex_moe.route_topk is the plain softmax form of a served Qwen3 layer and stays as it is.  The loads that a
balancing bias follows are `experts.expert_plan(ids, E)[0].diff()`.

Inputs must be CUDA tensors on an sm_100 device; there is no CPU path.  Calls run on the current stream of
the inputs' device, synchronise nothing and can be captured in CUDA graphs.
"""

from __future__ import annotations

import torch

from blackhole_b200 import _lib
from blackhole_b200.experts import _INDEX, _call, _recorded, _rows2d, _run
from blackhole_b200.hex_moe import _DT, _ptr

SCORING = {"softmax": _lib.SOFTMAX, "sigmoid": _lib.SIGMOID}
MAX_EXPERTS, MAX_TOPK = 2048, 32

_route, _route_backward = _lib.lib.hexmoe_route, _lib.lib.hexmoe_route_backward


def _check(what: str, logits: torch.Tensor, scoring: str) -> tuple[torch.Tensor, int, int]:
    """logits with contiguous rows, their row stride, and the code of the scoring."""
    if not logits.is_cuda:
        raise ValueError(f"{what} runs on CUDA only")
    if logits.dtype not in _DT:
        raise ValueError(f"{what}: unsupported logits dtype {logits.dtype}")
    if scoring not in SCORING:
        raise ValueError(f"{what}: scoring must be one of {sorted(SCORING)}, got {scoring!r}")
    if logits.dim() == 2 and logits.shape[1] > MAX_EXPERTS:
        raise ValueError(f"{what}: {logits.shape[1]} experts, at most {MAX_EXPERTS}")
    return *_rows2d(logits, "logits"), SCORING[scoring]


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, options):
        weights, ids = route(logits, k, **options)
        ctx.mark_non_differentiable(ids)
        ctx.save_for_backward(logits, ids)
        ctx.options = {name: options[name] for name in ("scoring", "renormalize", "scale")}
        return weights, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, _):
        return route_backward(dweights, *ctx.saved_tensors, **ctx.options), None, None


def route(logits: torch.Tensor, k: int, *, scoring: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          topk_groups: int | None = None, group_top: int = 2, renormalize: bool = True,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Every token's k experts and their weights from logits [T, E] (f32, bf16 or fp16; at most 2048 experts,
    k <= 32): (weights f32 [T, k], ids int32 [T, k]), differentiable in the logits (once).

    scoring      scores are softmax(logits) over all experts, or sigmoid(logits)
    bias         float32 [E]: added to the scores for the choice, not to the weights; it gets no gradient
    groups       experts in so many equal runs of ids (at most 32), of which the topk_groups with the largest
                 sums of their group_top (1 or 2) best scores, bias included, are open to the token
    renormalize  the weights of a token's experts sum to 1
    scale        a factor on the weights

    The experts come in the order of their scores, bias included (without a bias: of their logits), ties by the
    lower id, as 64-bit arithmetic decides.  An expert whose logit is -inf is masked: its score is 0, which is
    also what its group is valued by (with its bias), and it is taken after all others of the open groups; a token with
    nothing else there has weights 0.  A row with a NaN (softmax: or +inf) has NaN weights of valid ids."""
    res = _call.route(logits, k, SCORING.get(scoring), bias, groups, topk_groups, group_top, renormalize, scale)
    if res is not None:
        return res
    options = dict(scoring=scoring, bias=bias, groups=groups, topk_groups=topk_groups, group_top=group_top,
                   renormalize=renormalize, scale=scale)
    if _recorded(logits):
        return _Route.apply(logits, k, options)
    logits, ld, code = _check("route", logits, scoring)
    T, E = logits.shape
    dev = logits.device
    open_groups = groups if topk_groups is None else topk_groups
    for name, value in (("k", k), ("groups", groups), ("topk_groups", open_groups), ("group_top", group_top)):
        if not 1 <= value <= MAX_TOPK:
            raise ValueError(f"route: {name} {value} outside 1..{MAX_TOPK}")
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (E,) or bias.device != dev:
            raise ValueError(f"route: bias must be float32 [{E}] on {dev}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
        bias = bias.detach().contiguous()
    weights = torch.empty(T, k, dtype=torch.float32, device=dev)
    ids = torch.empty(T, k, dtype=torch.int32, device=dev)
    _run(_route, dev, logits.data_ptr(), _DT[logits.dtype], ld, T, E, k, code, _ptr(bias), groups,
         open_groups, group_top, renormalize, scale, weights.data_ptr(), ids.data_ptr())
    return weights, ids


def route_backward(dweights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, *, scoring: str = "softmax",
                   renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """The gradient of route's weights for the logits: dlogits [T, E] in their type, from dweights float32 [T, k]
    and the ids [T, k] (int32 or int64) that route gave, with the same scoring, renormalize and scale.  The choice
    itself (bias, groups) has no gradient.  ids outside 0..E-1 have no part.  A softmax's row with a NaN or +inf has a
    NaN gradient; with sigmoid scores only the chosen logits are looked at.  Not differentiable itself."""
    dlogits = _call.route_backward(dweights, logits, ids, SCORING.get(scoring), renormalize, scale)
    if dlogits is not None:
        return dlogits
    logits, ld, code = _check("route_backward", logits, scoring)
    T, E = logits.shape
    dev = logits.device
    if ids.dtype not in _INDEX or ids.dim() != 2 or ids.shape[0] != T or ids.shape[1] > MAX_TOPK or ids.device != dev:
        raise ValueError(f"route_backward: ids must be int32 or int64 [{T}, k <= {MAX_TOPK}] on {dev}, got {ids.dtype} {tuple(ids.shape)} "
                         f"on {ids.device}")
    if dweights.dtype != torch.float32 or dweights.shape != ids.shape or dweights.device != dev:
        raise ValueError(f"route_backward: dweights must be float32 {list(ids.shape)} on {dev}, got {dweights.dtype} "
                         f"{tuple(dweights.shape)} on {dweights.device}")
    dweights, ids = dweights.contiguous(), ids.contiguous()
    dlogits = torch.empty(T, E, dtype=logits.dtype, device=dev)
    _run(_route_backward, dev, dweights.data_ptr(), logits.data_ptr(), _DT[logits.dtype], ld, T, E, ids.shape[1],
         ids.data_ptr(), _INDEX[ids.dtype], code, renormalize, scale, dlogits.data_ptr(), E)
    return dlogits
