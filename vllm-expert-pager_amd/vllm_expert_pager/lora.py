"""Low-rank adapters of many requests beside the experts' projections (csrc/lora.hip).

The experts are frozen fp8 rows that the pager moves between tiers; a
fine-tuned variant of them is served as a pair of small matrices per expert
and projection, which stay in HBM, addressed by expert id, whatever slot the
expert's rows are in:

    y[t, k] = W_e x  +  scale_l B_le (A_le x)      l = adapter of token t, e = topk_ids[t, k]

``LowRankAdapters`` holds the adapters of one projection, ``low_rank`` computes
the second term for a batch in which every request may have an adapter of its
own (or none), on top of ``base``, the shared projection's output. With one
expert and no ``topk_ids`` it is the adapter of a dense projection. The gate
and up projections, which share their input, are one ``LowRankAdapters`` of two
slices. ``ExpertAdapters`` is the pair of them that the expert FFN takes
(``moe.fused_moe``, ``moe.run_experts``, ``PagedExperts.forward``).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from vllm_expert_pager import _native as nat

MAX_RANK = 128
DIRECT_PAIRS = 256  # pairs up to which the launch groups them itself (no workspace)
_DTYPES = {torch.bfloat16: 1, torch.float16: 2}


class LowRankAdapters:
    """Adapters ``0 .. adapters - 1`` of one projection, for each of ``experts`` experts.

    ``out_features`` covers all ``slices`` (2 for gate and up: gate columns,
    then up columns), each with matrices of its own. ``in_features`` and
    ``out_features / slices`` are multiples of 8, ranks at most ``max_rank``
    (128 at most); an adapter of a smaller rank is read only as far as its
    rank. Every adapter starts out empty (adds nothing).
    """

    def __init__(self, adapters: int, experts: int, in_features: int, out_features: int, max_rank: int, *,
                 slices: int = 1, dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        if dtype not in _DTYPES:
            raise ValueError(f"adapters are bfloat16 or float16, got {dtype}")
        if not 1 <= max_rank <= MAX_RANK:
            raise ValueError(f"max_rank must be in [1, {MAX_RANK}], got {max_rank}")
        if adapters < 1 or experts < 1 or adapters * experts >= 1 << 20:
            raise ValueError(f"{adapters} adapters of {experts} experts: at least one, fewer than 2^20 together")
        if not 1 <= slices <= 16 or out_features % slices:
            raise ValueError(f"{out_features} columns in {slices} slices")
        n = out_features // slices
        if in_features < 8 or in_features % 8 or n < 8 or n % 8:
            raise ValueError(f"in_features={in_features} and the {n} columns of a slice must be multiples of 8")
        self.adapters, self.experts, self.slices = adapters, experts, slices
        self.in_features, self.out_features, self.columns = in_features, out_features, n
        self.max_rank, self.dtype = max_rank, dtype
        # Storage: ranks in whole matrix-instruction steps, zeros behind what an adapter has.
        self.rank_rows = 16 if max_rank <= 16 else -(-max_rank // 32) * 32
        # A by blocks of 16 ranks and 32 inputs, each in the matrix instruction's lane order.
        self.a = torch.zeros((adapters, experts, slices, self.rank_rows // 16, -(-in_features // 32), 4, 16, 8),
                             dtype=dtype, device=device)
        self.b = torch.zeros((adapters, experts, slices, -(-n // 32) * 32, self.rank_rows), dtype=dtype, device=device)
        self.scales = torch.zeros((adapters,), dtype=torch.float32, device=device)
        self.ranks = torch.zeros((adapters,), dtype=torch.int32, device=device)

    @property
    def device(self) -> torch.device:
        return self.a.device

    @torch.no_grad()  # a copy: matrices that are parameters elsewhere leave no graph in the stack
    def load(self, adapter: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Put an adapter in place: ``a`` ``(experts, slices, r, in_features)`` and ``b`` ``(experts, slices,
        out_features / slices, r)``; without the slices' dimension for one slice, without the experts' for one
        expert. ``scale`` multiplies its output (alpha / r). On the current stream, as any other copy; bringing A
        into the kernels' order costs up to as much again as copying both."""
        self._index(adapter)
        lead = (self.experts, self.slices)
        # What may stand before a matrix: both dimensions, or without one (or both) of size 1.
        leads = {lead, lead[: 1 if lead[1] == 1 else 2], lead[1 if lead[0] == 1 else 0 :], () if lead == (1, 1) else lead}
        a, b = (t.reshape(lead + tuple(t.shape[-2:])) if tuple(t.shape[:-2]) in leads and t.dim() >= 2 else t
                for t in (a, b))
        r = a.shape[-2] if a.dim() == 4 else -1
        if tuple(a.shape) != (*lead, r, self.in_features) or tuple(b.shape) != (*lead, self.columns, r):
            raise ValueError(f"adapter matrices {tuple(a.shape)} and {tuple(b.shape)} do not fit {self.experts} experts, "
                             f"{self.slices} slices, {self.in_features} inputs and {self.columns} columns")
        if not 1 <= r <= self.max_rank:
            raise ValueError(f"rank {r} (at most {self.max_rank})")
        steps = self.a.shape[4]
        whole = torch.zeros((*lead, self.rank_rows, 32 * steps), dtype=self.dtype, device=self.a.device)
        whole[:, :, :r, : self.in_features] = a
        self.a[adapter] = whole.view(*lead, -1, 16, steps, 4, 8).permute(0, 1, 2, 4, 5, 3, 6)
        self.b[adapter, :, :, : self.columns, :r] = b
        self.b[adapter, :, :, :, r:] = 0
        self.scales[adapter] = float(scale)
        self.ranks[adapter] = r

    def clear(self, adapter: int) -> None:
        """Empty an adapter's place (its requests get the shared projection alone)."""
        self._index(adapter)
        self.a[adapter] = 0
        self.b[adapter] = 0
        self.scales[adapter] = 0
        self.ranks[adapter] = 0

    def _index(self, adapter: int) -> None:
        if not 0 <= adapter < self.adapters:
            raise ValueError(f"adapter {adapter} of {self.adapters}")


@dataclass
class ExpertAdapters:
    """The adapters of an expert layer: ``gate_up`` (two slices: gate, up) and ``down``; either may be None."""

    gate_up: LowRankAdapters | None = None
    down: LowRankAdapters | None = None

    def check(self, hidden: int, intermediate: int, experts: int, device: torch.device) -> None:
        """ValueError unless the stacks fit an expert layer of these sizes."""
        for stack, what, shape in ((self.gate_up, "gate_up", (experts, 2, hidden, intermediate)),
                                   (self.down, "down", (experts, 1, intermediate, hidden))):
            if stack is None:
                continue
            have = (stack.experts, stack.slices, stack.in_features, stack.columns)
            if have != shape or stack.dtype != torch.bfloat16 or stack.device != device:
                raise ValueError(f"{what} adapters of (experts, slices, inputs, columns) {have} in {stack.dtype} on "
                                 f"{stack.device} do not fit a layer of {shape} in torch.bfloat16 on {device}")
        if self.gate_up is not None and self.down is not None and self.gate_up.adapters != self.down.adapters:
            raise ValueError(f"{self.gate_up.adapters} gate_up and {self.down.adapters} down adapters")


@dataclass
class AdaptedBatch:
    """A batch's pairs with their adapters, as ``moe.run_experts`` takes them.

    ``gate_up`` holds the pairs' gate and up terms ``(T * topk, 2I)``, made
    once per layer call: they depend on tokens and ids alone, so the experts
    may then run in any number of chunks. ``listing`` is the pairs by adapter
    and expert, shared by both projections of a call in one piece.
    """

    adapters: ExpertAdapters
    adapter_ids: torch.Tensor
    topk_ids: torch.Tensor
    gate_up: torch.Tensor | None
    listing: torch.Tensor | None

    def down(self, acts: torch.Tensor, expert_map: torch.Tensor | None, slots: int) -> torch.Tensor | None:
        """The down projection's terms ``(T * topk, H)`` of the pairs whose expert ``expert_map`` places in a slot
        (None: all), from their activations ``(T * topk, I)``; the other rows are left unwritten."""
        stack = self.adapters.down
        if stack is None:
            return None
        T, topk = self.topk_ids.shape
        out = torch.empty((T * topk, stack.out_features), dtype=stack.dtype, device=acts.device)
        listing = self.listing
        if expert_map is not None:
            nat.require_same_device(expert_map, stack.a, "expert_map")
            if expert_map.dtype != torch.int32 or not expert_map.is_contiguous() or expert_map.numel() < stack.experts:
                raise ValueError(f"expert_map must be a contiguous int32 tensor of {stack.experts} entries, got "
                                 f"{expert_map.dtype} {tuple(expert_map.shape)}")
            listing = group(stack, self.adapter_ids, self.topk_ids, expert_map, slots)
        apply(acts, stack, self.adapter_ids, self.topk_ids, T, topk, True, None, out, expert_map=expert_map, slots=slots,
              listing=listing)
        return out


def adapt(x: torch.Tensor, adapters: ExpertAdapters, adapter_ids: torch.Tensor, topk_ids: torch.Tensor,
          intermediate: int, experts: int) -> AdaptedBatch:
    """The adapters' part of a layer call that its tokens ``x`` ``(T, H)`` decide, before any expert runs."""
    nat.require_device(x, "x")
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise ValueError(f"x must be a 2-D bfloat16 tensor, got {x.dtype} {tuple(x.shape)}")
    T, H = x.shape
    adapters.check(H, intermediate, experts, x.device)
    adapter_ids, topk_ids = _ids(adapter_ids, "adapter_ids", x), _ids(topk_ids, "topk_ids", x)
    if tuple(adapter_ids.shape) != (T,) or topk_ids.dim() != 2 or topk_ids.shape[0] != T:
        raise ValueError(f"adapter_ids must be ({T},) and topk_ids ({T}, topk), got {tuple(adapter_ids.shape)} and "
                         f"{tuple(topk_ids.shape)}")
    some = adapters.gate_up if adapters.gate_up is not None else adapters.down
    if some is None or T == 0:
        return AdaptedBatch(adapters, adapter_ids, topk_ids, None, None)
    listing = group(some, adapter_ids, topk_ids, None, 0)
    terms = None
    if adapters.gate_up is not None:
        terms = torch.empty((topk_ids.numel(), 2 * intermediate), dtype=x.dtype, device=x.device)
        apply(x.contiguous(), adapters.gate_up, adapter_ids, topk_ids, T, topk_ids.shape[1], False, None, terms,
              listing=listing)
    return AdaptedBatch(adapters, adapter_ids, topk_ids, terms, listing)


def _ids(t: torch.Tensor, what: str, like: torch.Tensor) -> torch.Tensor:
    nat.require_same_device(t, like, what)
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what} must be int32 or int64, got {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _rows(t: torch.Tensor, shape: tuple[int, int], what: str, stack: LowRankAdapters) -> None:
    nat.require_same_device(t, stack.a, what)
    if t.dtype != stack.dtype or t.shape != shape:
        raise ValueError(f"{what} must be {stack.dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
    # Rows may be apart; each starts on 16 bytes and is consecutive.
    if t.data_ptr() % 16 or not t.is_contiguous() and t.numel() and (
            t.stride(1) != 1 or (shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) < shape[1]))):
        raise ValueError(f"{what} must have consecutive rows that start on 16 bytes, got strides {t.stride()}")


def _stride(t: torch.Tensor | None) -> int:
    return 0 if t is None or t.shape[0] <= 1 else t.stride(0)


def low_rank(
    x: torch.Tensor,
    stack: LowRankAdapters,
    adapter_ids: torch.Tensor,
    topk_ids: torch.Tensor | None = None,
    *,
    base: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``base + scale * B (A x)`` per pair, ``(T * topk, out_features)`` (zeros for ``base`` None).

    ``adapter_ids`` ``(T,)`` is each token's adapter; one outside ``[0,
    adapters)`` (-1) has none. ``topk_ids`` ``(T, topk)`` are the pairs'
    experts (None for a projection of one expert: topk 1); a pair with an id
    outside ``[0, experts)`` gets ``base``. ``x`` has a row per token, or one
    per pair (``T * topk`` rows, the experts' activations). ``out`` may be
    ``base`` itself (the same rows), and must not overlap ``x`` or ``base``
    otherwise. Types are the stack's; the result is rounded once and carries no
    gradient.
    """
    nat.require_device(stack.a, "the adapters")
    adapter_ids = _ids(adapter_ids, "adapter_ids", stack.a)
    if adapter_ids.dim() != 1:
        raise ValueError(f"adapter_ids must be 1-D, got {tuple(adapter_ids.shape)}")
    T, topk = adapter_ids.shape[0], 1
    if topk_ids is not None:
        topk_ids = _ids(topk_ids, "topk_ids", stack.a)
        if topk_ids.dim() != 2 or topk_ids.shape[0] != T or topk_ids.shape[1] < 1:
            raise ValueError(f"topk_ids must be ({T}, topk), got {tuple(topk_ids.shape)}")
        topk = topk_ids.shape[1]
    elif stack.experts != 1:
        raise ValueError(f"adapters of {stack.experts} experts need topk_ids")
    P = T * topk
    per_pair = x.dim() == 2 and x.shape[0] == P and topk > 1 and P != T
    _rows(x, (P if per_pair else T, stack.in_features), "x", stack)
    if base is not None:
        _rows(base, (P, stack.out_features), "base", stack)
    if out is None:
        out = stack.a.new_empty((P, stack.out_features))
    else:
        _rows(out, (P, stack.out_features), "out", stack)
    if P:
        apply(x, stack, adapter_ids, topk_ids, T, topk, per_pair, base, out)
    return out


def group(stack: LowRankAdapters, adapter_ids: torch.Tensor, topk_ids: torch.Tensor, expert_map: torch.Tensor | None,
          slots: int) -> torch.Tensor | None:
    """The listing of a call's pairs by adapter and expert, for several ``apply`` calls; None where they need none."""
    T, topk = topk_ids.shape
    if T * topk <= DIRECT_PAIRS:
        return None
    nbytes = int(nat.lib().xp_lora_workspace_bytes(T * topk, stack.adapters, stack.experts))
    work = torch.empty((nbytes,), dtype=torch.uint8, device=stack.a.device)
    nat.call_on(stack.a, "xp_lora_group", adapter_ids.data_ptr(), adapter_ids.element_size(), topk_ids.data_ptr(),
                topk_ids.element_size(), T, topk, nat.ptr(expert_map), slots, stack.adapters, stack.experts,
                work.data_ptr(), nbytes)
    return work


def apply(x: torch.Tensor, stack: LowRankAdapters, adapter_ids: torch.Tensor, topk_ids: torch.Tensor | None, T: int,
          topk: int, per_pair: bool, base: torch.Tensor | None, out: torch.Tensor, *,
          expert_map: torch.Tensor | None = None, slots: int = 0, listing: torch.Tensor | None = None) -> None:
    """One launch of the adapters over checked arguments; ``listing`` is ``group``'s of the same ids."""
    grouped = listing is not None
    nbytes = 0
    if grouped:
        nbytes = listing.numel()
    elif T * topk > DIRECT_PAIRS:
        nbytes = int(nat.lib().xp_lora_workspace_bytes(T * topk, stack.adapters, stack.experts))
        listing = torch.empty((nbytes,), dtype=torch.uint8, device=stack.a.device)
    nat.call_on(
        stack.a, "xp_lora_apply", x.data_ptr(), _DTYPES[stack.dtype], _stride(x), per_pair, T, topk, stack.in_features,
        stack.a.data_ptr(), stack.b.data_ptr(), stack.scales.data_ptr(), stack.ranks.data_ptr(), stack.adapters,
        stack.experts, stack.slices, stack.columns, stack.rank_rows, adapter_ids.data_ptr(),
        adapter_ids.element_size(), nat.ptr(topk_ids), 4 if topk_ids is None else topk_ids.element_size(),
        nat.ptr(expert_map), slots, nat.ptr(base), _stride(base), out.data_ptr(), _stride(out), nat.ptr(listing),
        nbytes, grouped,
    )
