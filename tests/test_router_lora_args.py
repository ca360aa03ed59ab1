"""Refusals of the router and adapter calls, and the layout of loaded adapters (CPU, no kernel is launched)."""

import pytest
import torch

from vllm_expert_pager import _native as nat
from vllm_expert_pager import lora, moe, router

P = 1 << 20  # an address that a refused call never reads


def _refused(name, *args):
    with pytest.raises(ValueError):
        nat.call(name, *args)


CHOOSE = dict(logits=P, dtype=0, T=4, E=16, stride=16, topk=2, scoring=0, renorm=1, bias=None, groups=1, keep=1,
              scale=1.0, mask=None, weights=P, ids=P, stream=None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(dtype=3), dict(dtype=-1), dict(T=-1), dict(T=1 << 31), dict(E=0), dict(E=2049), dict(stride=15),
    dict(topk=0), dict(topk=17), dict(E=128, stride=128, topk=65), dict(scoring=2), dict(groups=0), dict(groups=3),
    dict(groups=4, keep=5), dict(groups=4, keep=0), dict(groups=8, keep=1, topk=3), dict(E=1280, stride=1280, groups=2),
    dict(E=128, stride=128, groups=128, keep=128), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e300),
    dict(weights=None), dict(ids=None),
])
def test_choose_refuses(bad):
    _refused("xp_router_choose", *{**CHOOSE, **bad}.values())


BALANCE = dict(logits=P, dtype=0, T=4, E=16, stride=16, topk=2, scoring=0, ids=P, eb=4, mask=None, offsets=None, seqs=1,
               work=P, nbytes=1 << 30, counts=P, tokens=P, loss=P, stream=None)


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(E=4096, stride=4096), dict(topk=0), dict(topk=65), dict(scoring=5), dict(eb=2), dict(ids=None),
    dict(seqs=0), dict(seqs=2), dict(offsets=P, seqs=65535), dict(work=None), dict(work=P + 4), dict(nbytes=64),
    dict(counts=None), dict(tokens=None), dict(loss=None),
])
def test_balance_refuses(bad):
    _refused("xp_router_balance", *{**BALANCE, **bad}.values())


BACK = dict(logits=P, dtype=0, T=4, E=16, stride=16, topk=2, scoring=0, renorm=1, scale=1.0, mask=None, offsets=None,
            seqs=1, ids=P, eb=4, gw=P, counts=P, tokens=P, gl=P, grad=P, stream=None)


@pytest.mark.parametrize("bad", [
    dict(dtype=7), dict(topk=0), dict(ids=None), dict(eb=3), dict(counts=None), dict(tokens=None), dict(gl=None),
    dict(grad=None), dict(seqs=3), dict(scale=float("nan")),
])
def test_backward_refuses(bad):
    _refused("xp_router_backward", *{**BACK, **bad}.values())


APPLY = dict(x=P, dtype=1, x_stride=64, per_pair=0, T=4, topk=2, K=64, a=P, b=P, scales=P, ranks=P, adapters=3, experts=8,
             slices=1, n=32, R=16, who=P, web=4, ids=P, eb=4, emap=None, slots=0, base=None, base_stride=0, out=P,
             out_stride=32, work=None, nbytes=0, grouped=0, stream=None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(dtype=0), dict(x_stride=60), dict(x_stride=56), dict(T=-1), dict(topk=0), dict(T=1 << 30, topk=4),
    dict(K=60), dict(K=0), dict(a=None), dict(b=P + 2), dict(scales=None), dict(ranks=None), dict(adapters=0),
    dict(adapters=1 << 19), dict(slices=0), dict(slices=17), dict(n=12), dict(R=48), dict(R=144), dict(who=None),
    dict(web=2), dict(ids=None), dict(eb=1), dict(base=P + 8, base_stride=32), dict(base=P, base_stride=24), dict(out=None),
    dict(out_stride=24), dict(out_stride=36), dict(base=P, base_stride=40), dict(T=129), dict(T=129, work=P, nbytes=64), dict(T=129, work=P + 16, nbytes=1 << 30),
])
def test_apply_refuses(bad):
    _refused("xp_lora_apply", *{**APPLY, **bad}.values())


def test_workspace_sizes():
    lib = nat.lib()
    assert lib.xp_lora_workspace_bytes(0, 4, 4) == 0 and lib.xp_lora_workspace_bytes(10, 0, 4) == 0
    assert lib.xp_lora_workspace_bytes(1000, 4, 4) >= 1000 * 12
    assert lib.xp_router_workspace_bytes(-1, 4, 1) == 0 and lib.xp_router_workspace_bytes(5, 0, 1) == 0
    assert lib.xp_router_workspace_bytes(0, 4, 1) > 0


def test_host_tensors_are_refused():
    z, ids = torch.zeros((4, 8)), torch.zeros((4, 2), dtype=torch.int32)
    for call in (lambda: router.choose_experts(z, 2), lambda: router.balance_loss(z, ids),
                 lambda: router.choose_and_balance(z, 2)):
        with pytest.raises(ValueError):
            call()
    stack = lora.LowRankAdapters(1, 1, 16, 16, 4, device="cpu")
    with pytest.raises(ValueError):
        lora.low_rank(torch.zeros((4, 16), dtype=torch.bfloat16), stack, ids[:, 0])
    with pytest.raises(ValueError):
        lora.adapt(torch.zeros((4, 16), dtype=torch.bfloat16), lora.ExpertAdapters(), ids[:, 0], ids, 128, 8)
    w = torch.zeros((1, 256, 128), dtype=torch.uint8)
    with pytest.raises(ValueError):  # adapters without their ids
        moe.fused_moe(torch.zeros((4, 128), dtype=torch.bfloat16), torch.zeros((4, 1)), ids[:, :1], w, w, w, w,
                      adapters=lora.ExpertAdapters())


@pytest.mark.parametrize("K, n, r, rank_rows", [(72, 40, 3, 16), (64, 32, 16, 16), (40, 8, 17, 32), (96, 48, 70, 96)])
def test_layout_of_loaded_adapters(K, n, r, rank_rows):
    """Block [i][k] of a holds rank 16 i + m, input 32 k + 8 q + c at [q][m][c]; b by columns; zeros elsewhere."""
    L, E, S = 2, 3, 2
    stack = lora.LowRankAdapters(L, E, K, S * n, r, slices=S, device="cpu")
    g = torch.Generator().manual_seed(0)
    a, b = torch.randn((E, S, r, K), generator=g), torch.randn((E, S, n, r), generator=g)
    stack.load(1, a, b, 0.25)
    assert stack.rank_rows == rank_rows
    steps = -(-K // 32)
    whole = torch.zeros((E, S, rank_rows, 32 * steps), dtype=torch.bfloat16)
    for i in range(rank_rows // 16):
        for k in range(steps):
            for q in range(4):
                whole[:, :, 16 * i : 16 * i + 16, 32 * k + 8 * q : 32 * k + 8 * q + 8] = stack.a[1, :, :, i, k, q]
    assert torch.equal(whole[:, :, :r, :K], a.bfloat16())
    assert whole[:, :, r:].abs().sum() == 0 and whole[:, :, :, K:].abs().sum() == 0
    assert torch.equal(stack.b[1, :, :, :n, :r], b.bfloat16())
    assert stack.b[1, :, :, n:].abs().sum() == 0 and stack.b[1, :, :, :, r:].abs().sum() == 0
    assert stack.a[0].abs().sum() == 0 and stack.scales.tolist() == [0.0, 0.25] and stack.ranks.tolist() == [0, r]


@pytest.mark.parametrize("E, S, fits, bad", [
    (2, 1, [(2, 1), (2,)], [(1, 2), (), (2, 1, 1)]), (1, 2, [(1, 2), (2,)], [(2, 1), ()]), (1, 1, [(1, 1), (1,), ()], [(1, 1, 1), (2,)]),
    (2, 3, [(2, 3)], [(3, 2), (6,), (1, 6)]),
])
def test_shapes_of_loaded_adapters(E, S, fits, bad):
    """The experts' and the slices' dimension are left out only where they are 1, and never taken for each other."""
    stack = lora.LowRankAdapters(1, E, 16, S * 8, 4, slices=S, device="cpu")
    a, b = torch.randn((E * S, 3, 16)), torch.randn((E * S, 8, 3))
    stack.load(0, a.view(E, S, 3, 16), b.view(E, S, 8, 3))
    want = stack.a.clone(), stack.b.clone()
    for lead in fits:
        stack.clear(0)
        stack.load(0, a.view(*lead, 3, 16), b.view(*lead, 8, 3))
        assert torch.equal(stack.a, want[0]) and torch.equal(stack.b, want[1])
    for lead in bad:
        n = 1
        for d in lead:
            n *= d
        with pytest.raises(ValueError):
            stack.load(0, torch.randn((n, 3, 16)).view(*lead, 3, 16), torch.randn((n, 8, 3)).view(*lead, 8, 3))


def test_loaded_parameters_keep_no_graph():
    """Matrices that are trained elsewhere (parameters) are copied: the stack takes no part in their graph."""
    stack = lora.LowRankAdapters(2, 3, 16, 8, 4, device="cpu")
    a, b = torch.nn.Parameter(torch.randn((3, 4, 16))), torch.nn.Parameter(torch.randn((3, 8, 4)))
    stack.load(1, a, b * 2)
    for t in (stack.a, stack.b, stack.scales, stack.ranks):
        assert not t.requires_grad and t.grad_fn is None
    assert torch.equal(stack.b[1, :, 0, :8, :4], (b * 2).detach().bfloat16())
    stack.load(1, a, b)
    stack.clear(0)
    assert torch.equal(stack.b[1, :, 0, :8, :4], b.detach().bfloat16())


@pytest.mark.parametrize("bad", [
    torch.zeros((7,), dtype=torch.int32), torch.zeros((0,), dtype=torch.int32), torch.zeros((8,), dtype=torch.int64),
    torch.zeros((16,), dtype=torch.int32)[::2],
])
def test_expert_map_of_an_adapted_chunk(bad):
    """The kernels read an entry per expert of the adapters: a shorter map, or one of other values, is refused."""
    stack = lora.LowRankAdapters(2, 8, 16, 8, 4, device="cpu")
    ids = torch.zeros((3, 2), dtype=torch.int32)
    batch = lora.AdaptedBatch(lora.ExpertAdapters(down=stack), ids[:, 0].contiguous(), ids, None, None)
    with pytest.raises(ValueError, match="expert_map"):
        batch.down(torch.zeros((6, 16), dtype=torch.bfloat16), bad, 8)


@pytest.mark.parametrize("T, E, topk", [((1 << 28) + 1, 8, 2), ((1 << 26) + 1, 600, 2), ((1 << 31) - 1, 1, 1)])
def test_more_rows_than_a_launch_has_threads_for(T, E, topk):
    for name, args in (("xp_router_choose", CHOOSE), ("xp_router_backward", BACK)):
        with pytest.raises(nat.NativeError, match="launch grid"):
            nat.call(name, *{**args, "T": T, "E": E, "stride": E, "topk": topk}.values())
