"""The router beside the experts: choice, balance loss and counts, with gradients (csrc/router.hip).

The pager takes ``topk_weights`` and ``topk_ids`` as they are (the reference
has them from vLLM, experts.py:380-400). This module makes them from the
router's logits, and says how they are spread:

    topk_weights, topk_ids = choose_experts(logits, topk)
    loss, counts = balance_loss(logits, topk_ids)
    topk_weights, topk_ids, loss, counts = choose_and_balance(logits, topk)   # both in one pass

``topk_ids`` go to ``moe.fused_moe``, ``PagedExperts.forward`` and the tables
as they are: an id of -1 (a padded token, or fewer experts left than topk) adds
nothing there. ``counts`` tell which experts a traffic prefers, which decides
the tables' hit rates; the loss trains a router towards or away from it.

The weights and the loss are differentiable by the logits (backward, first
order); ids and counts are not. The expert calls of this package return tensors
without a graph: a gradient of ``topk_weights`` comes from experts that are run
elsewhere, and beside frozen experts served here a router is trained by the loss
alone. All calls run on the current stream of the logits' device, allocate their
results with torch and can be captured in a graph.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from vllm_expert_pager import _native as nat

SCORING = {"softmax": 0, "sigmoid": 1}
MAX_TOPK = 64
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _logits(logits: torch.Tensor) -> torch.Tensor:
    nat.require_device(logits, "logits")
    if logits.dtype not in _DTYPES or logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be a 2-D float32, bfloat16 or float16 tensor, got {logits.dtype} "
                         f"{tuple(logits.shape)}")
    # Rows may be apart (a slice of a wider projection); within a row they are consecutive.
    if not logits.is_contiguous() and (logits.stride(1) != 1 or logits.stride(0) < logits.shape[1]):
        logits = logits.contiguous()
    return logits


def _scoring(scoring: str) -> int:
    code = SCORING.get(scoring)
    if code is None:
        raise ValueError(f"scoring {scoring!r}: one of {sorted(SCORING)}")
    return code


def _pick(logits: torch.Tensor, topk: int, bias: torch.Tensor | None, groups: int,
          topk_groups: int) -> torch.Tensor | None:
    E = logits.shape[1]
    if not 1 <= topk <= min(MAX_TOPK, E):
        raise ValueError(f"topk must be in [1, {min(MAX_TOPK, E)}] for {E} experts, got {topk}")
    if groups < 1 or E % groups or not 1 <= topk_groups <= groups or topk > E // groups * topk_groups:
        raise ValueError(f"{topk_groups} of {groups} groups do not fit topk={topk} of {E} experts")
    if bias is None:
        return None
    nat.require_same_device(bias, logits, "bias")
    if tuple(bias.shape) != (E,) or not bias.is_floating_point():
        raise ValueError(f"bias must be a floating-point tensor of {E} entries, got {bias.dtype} {tuple(bias.shape)}")
    return bias.detach().to(torch.float32).contiguous()


def _mask(mask: torch.Tensor | None, logits: torch.Tensor) -> torch.Tensor | None:
    if mask is None:
        return None
    nat.require_same_device(mask, logits, "mask")
    if mask.dtype != torch.bool or tuple(mask.shape) != (logits.shape[0],):
        raise ValueError(f"mask must be a bool tensor of {logits.shape[0]} tokens, got {mask.dtype} {tuple(mask.shape)}")
    return mask.contiguous()


def _offsets(seq_offsets: torch.Tensor | None, logits: torch.Tensor) -> tuple[torch.Tensor | None, int]:
    if seq_offsets is None:
        return None, 1
    nat.require_same_device(seq_offsets, logits, "seq_offsets")
    if seq_offsets.dtype not in (torch.int32, torch.int64) or seq_offsets.dim() != 1 or not (
            2 <= seq_offsets.numel() <= 65535):
        raise ValueError("seq_offsets must be a 1-D int32 or int64 tensor of 2 to 65535 entries, got "
                         f"{seq_offsets.dtype} {tuple(seq_offsets.shape)}")
    num_seqs = seq_offsets.numel() - 1
    if seq_offsets.dtype == torch.int64:  # an offset behind every row stays one
        seq_offsets = seq_offsets.clamp(-1, 2**31 - 1).to(torch.int32)
    return seq_offsets.contiguous(), num_seqs


def _stats(logits: torch.Tensor, num_seqs: int, per_seq: bool):
    """(workspace, its bytes, counts, tokens, loss) of a balance pass."""
    T, E = logits.shape
    nbytes = int(nat.lib().xp_router_workspace_bytes(T, E, num_seqs))
    dev = logits.device
    return (torch.empty((nbytes,), dtype=torch.uint8, device=dev), nbytes,
            torch.empty((num_seqs, E) if per_seq else (E,), dtype=torch.int32, device=dev),
            torch.empty((num_seqs + 1,), dtype=torch.int32, device=dev),
            torch.empty((), dtype=torch.float32, device=dev))


def _fp32(grad: torch.Tensor | None) -> torch.Tensor | None:
    if grad is None or (grad.dtype == torch.float32 and grad.is_contiguous()):
        return grad
    return grad.to(torch.float32).contiguous()


def _backward(ctx, grad_weights, grad_loss):
    """The logits' gradient through the weights and the loss (either may be None)."""
    if grad_weights is None and grad_loss is None:
        return None
    logits, ids, counts, tokens, mask, offsets = ctx.saved_tensors
    T, E = logits.shape
    grad = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
    gw, gl = _fp32(grad_weights), _fp32(grad_loss)
    through = gl is not None
    nat.call_on(
        logits, "xp_router_backward", logits.data_ptr(), _DTYPES[logits.dtype], T, E, logits.stride(0), ctx.topk,
        ctx.scoring, ctx.renormalize, ctx.scale, nat.ptr(mask), nat.ptr(offsets), ctx.num_seqs, ids.data_ptr(),
        ids.element_size(), nat.ptr(gw), counts.data_ptr() if through else None,
        tokens.data_ptr() if through else None, nat.ptr(gl), grad.data_ptr(),
    )
    return grad


def _choose(logits, topk, scoring, renormalize, bias, groups, topk_groups, scale, mask):
    T, E = logits.shape
    weights = logits.new_empty((T, topk), dtype=torch.float32)
    ids = logits.new_empty((T, topk), dtype=torch.int32)
    nat.call_on(
        logits, "xp_router_choose", logits.data_ptr(), _DTYPES[logits.dtype], T, E, logits.stride(0), topk, scoring,
        renormalize, nat.ptr(bias), groups, topk_groups, scale, nat.ptr(mask), weights.data_ptr(), ids.data_ptr(),
    )
    return weights, ids


class _Choose(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, scoring, renormalize, bias, groups, topk_groups, scale, mask):
        weights, ids = _choose(logits, topk, scoring, renormalize, bias, groups, topk_groups, scale, mask)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(ids)
        ctx.save_for_backward(logits, ids, None, None, mask, None)
        ctx.topk, ctx.scoring, ctx.renormalize, ctx.scale, ctx.num_seqs = topk, scoring, renormalize, scale, 1
        return weights, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, _ids):
        return _backward(ctx, grad_weights, None), *(None,) * 8


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, scoring, mask, offsets, num_seqs):
        T, E = logits.shape
        topk = ids.shape[1]
        work, nbytes, counts, tokens, loss = _stats(logits, num_seqs, offsets is not None)
        nat.call_on(
            logits, "xp_router_balance", logits.data_ptr(), _DTYPES[logits.dtype], T, E, logits.stride(0), topk, scoring,
            ids.data_ptr(), ids.element_size(), nat.ptr(mask), nat.ptr(offsets), num_seqs, work.data_ptr(), nbytes,
            counts.data_ptr(), tokens.data_ptr(), loss.data_ptr(),
        )
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(counts)
        ctx.save_for_backward(logits, ids, counts, tokens, mask, offsets)
        ctx.topk, ctx.scoring, ctx.renormalize, ctx.scale, ctx.num_seqs = topk, scoring, False, 1.0, num_seqs
        return loss, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss, _counts):
        return _backward(ctx, None, grad_loss), *(None,) * 5


class _ChooseBalance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk, scoring, renormalize, bias, groups, topk_groups, scale, mask, offsets, num_seqs):
        T, E = logits.shape
        weights = torch.empty((T, topk), dtype=torch.float32, device=logits.device)
        ids = torch.empty((T, topk), dtype=torch.int32, device=logits.device)
        work, nbytes, counts, tokens, loss = _stats(logits, num_seqs, offsets is not None)
        nat.call_on(
            logits, "xp_router_choose_balance", logits.data_ptr(), _DTYPES[logits.dtype], T, E, logits.stride(0), topk,
            scoring, renormalize, nat.ptr(bias), groups, topk_groups, scale, nat.ptr(mask), nat.ptr(offsets), num_seqs,
            weights.data_ptr(), ids.data_ptr(), work.data_ptr(), nbytes, counts.data_ptr(), tokens.data_ptr(),
            loss.data_ptr(),
        )
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(ids, counts)
        ctx.save_for_backward(logits, ids, counts, tokens, mask, offsets)
        ctx.topk, ctx.scoring, ctx.renormalize, ctx.scale = topk, scoring, renormalize, scale
        ctx.num_seqs = num_seqs
        return weights, ids, loss, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, _ids, grad_loss, _counts):
        return _backward(ctx, grad_weights, grad_loss), *(None,) * 10


def choose_experts(
    logits: torch.Tensor,
    topk: int,
    *,
    scoring: str = "softmax",
    renormalize: bool = True,
    bias: torch.Tensor | None = None,
    groups: int = 1,
    topk_groups: int = 1,
    scale: float = 1.0,
    mask: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(topk_weights, topk_ids)`` (fp32 and int32, ``(T, topk)``) of the router's logits ``(T, E)``.

    ``scoring`` is the softmax over the experts or the sigmoid of each.
    Experts come in descending order, equal ones by the lower index; a masked
    logit (NaN or -inf) is never chosen, and where fewer than ``topk`` are
    left the id is -1 and the weight 0. ``renormalize`` divides a token's
    weights by their sum, ``scale`` multiplies them. ``bias`` (``(E,)``) is
    added to the scores for the choice alone. With ``groups`` > 1 only the
    ``topk_groups`` best groups of ``E / groups`` consecutive experts are
    chosen from: by their best expert, or with a bias by the sum of their best
    two. ``mask`` (bool, ``(T,)``): False marks padding, whose ids are -1.
    At most 2048 experts, 64 chosen, and 64 groups (of at most 1024 experts).
    """
    code = _scoring(scoring)
    logits = _logits(logits)
    bias = _pick(logits, topk, bias, groups, topk_groups)
    args = (logits, topk, code, bool(renormalize), bias, groups, topk_groups, float(scale), _mask(mask, logits))
    # Inside a level of forward mode the function is taken as well: it refuses a tensor that carries a tangent.
    if (logits.requires_grad and torch.is_grad_enabled()) or getattr(forward_ad, "_current_level", 0) >= 0:
        return _Choose.apply(*args)
    return _choose(*args)  # serving: no graph, and none of its cost (a third of a one-token call's host time)


def balance_loss(
    logits: torch.Tensor,
    topk_ids: torch.Tensor,
    *,
    scoring: str = "softmax",
    mask: torch.Tensor | None = None,
    seq_offsets: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, counts)`` of a choice ``topk_ids`` ``(T, topk)`` made from ``logits`` ``(T, E)``.

    ``counts[e]`` (int32) is how often expert e is chosen. With n tokens,
    ``f_e = E counts_e / (topk n)`` and ``P_e`` the mean probability of e
    (softmax, or the sigmoid over its sum), the loss (an fp32 scalar) is
    ``sum_e f_e P_e``: 1 for an even spread. With ``seq_offsets`` (ascending,
    ``(B + 1,)``) sequence s holds the rows ``[seq_offsets[s],
    seq_offsets[s + 1])``, counts are ``(B, E)``, and the loss is the mean over
    the sequences that have tokens; rows outside of all are padding. Padding,
    and ids outside ``[0, E)``, count nowhere. Every sequence is given the same
    number of workgroups, so lengths of one order are summed fastest.
    """
    code = _scoring(scoring)
    logits = _logits(logits)
    nat.require_same_device(topk_ids, logits, "topk_ids")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != logits.shape[0] or not 1 <= topk_ids.shape[1] <= MAX_TOPK:
        raise ValueError(f"topk_ids must be ({logits.shape[0]}, 1 to {MAX_TOPK}), got {tuple(topk_ids.shape)}")
    if topk_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    offsets, num_seqs = _offsets(seq_offsets, logits)
    return _Balance.apply(logits, topk_ids.contiguous(), code, _mask(mask, logits), offsets, num_seqs)


def choose_and_balance(
    logits: torch.Tensor,
    topk: int,
    *,
    scoring: str = "softmax",
    renormalize: bool = True,
    bias: torch.Tensor | None = None,
    groups: int = 1,
    topk_groups: int = 1,
    scale: float = 1.0,
    mask: torch.Tensor | None = None,
    seq_offsets: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(topk_weights, topk_ids, loss, counts)``: ``choose_experts`` and the ``balance_loss`` of its choice.

    One pass over the logits forward and one backward. Rows outside of every
    sequence of ``seq_offsets`` are padding (ids -1, weights 0).
    """
    code = _scoring(scoring)
    logits = _logits(logits)
    bias = _pick(logits, topk, bias, groups, topk_groups)
    offsets, num_seqs = _offsets(seq_offsets, logits)
    return _ChooseBalance.apply(logits, topk, code, bool(renormalize), bias, groups, topk_groups, float(scale),
                                _mask(mask, logits), offsets, num_seqs)
