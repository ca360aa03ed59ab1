"""The expert layer with its router and low-rank adapters: router.py, lora.py, moe.py and pager.py together.

Tolerance against the oracle: that of the layer without adapters
(tests/test_moe_gpu.py): the adapters' terms are rounded to bf16 before they
enter, here as in the oracle, but for terms next to a rounding boundary, whose
flips move a gate or up value by at most one bf16 step of the term, the same
kind of flip that those bounds are made for. The oracle takes every product in
64 bits.
"""

import numpy as np
import pytest
import torch

from oracle import moe_ref as M
from test_moe_gpu import _check_close
from test_pager_gpu import Model, routing, same

pytestmark = pytest.mark.gpu


def _mods():
    from vllm_expert_pager import lora, moe, router

    return lora, moe, router


def _adapters(L, E, H, I, rank, seed, which="both"):
    lora = _mods()[0]
    g = torch.Generator(device="cuda").manual_seed(seed)
    mats = {}
    made = lora.ExpertAdapters()
    for name, slices, k, n in (("gate_up", 2, H, I), ("down", 1, I, H)):
        if which not in ("both", name):
            continue
        stack = lora.LowRankAdapters(L, E, k, slices * n, rank, slices=slices)
        setattr(made, name, stack)
        for i in range(L):
            r = max(1, rank - 3 * i)
            a = (torch.randn((E, slices, r, k), generator=g, device="cuda") / k**0.5).to(torch.bfloat16)
            b = (0.3 * torch.randn((E, slices, n, r), generator=g, device="cuda")).to(torch.bfloat16)
            stack.load(i, a, b, 0.5)
            mats[name, i] = (a.double().cpu().numpy(), b.double().cpu().numpy())
    return made, mats


def _oracle(x, tw, ids, who, weights, mats, act):
    """The layer pair by pair; x (T, H) holds bf16 values."""
    w13, w13s, w2, w2s = weights
    T, topk = ids.shape
    E, I = w13.shape[0], w13.shape[1] // 2
    contrib = np.zeros((T * topk, x.shape[1]), np.float32)
    xd = M.dequant_rows(*M.quant_groups(x))
    for p in range(T * topk):
        t, e, a = p // topk, int(ids.reshape(-1)[p]), int(who[p // topk])
        if not 0 <= e < E:
            continue
        h = M.dequant_weight(w13[e], w13s[e]) @ xd[t]
        if ("gate_up", a) in mats:
            ma, mb = mats["gate_up", a]
            d = np.concatenate([0.5 * (mb[e, s] @ (ma[e, s] @ x[t].astype(np.float64))) for s in (0, 1)])
            h = h + M.bf16(d)
        h = M.bf16(h.astype(np.float32))
        act_row = M.bf16(M.bf16(M.activation(h[:I], act)) * h[I:])
        y = M.dequant_weight(w2[e], w2s[e]) @ M.dequant_rows(*M.quant_groups(act_row[None]))[0]
        if ("down", a) in mats:
            ma, mb = mats["down", a]
            y = y + M.bf16(0.5 * (mb[e, 0] @ (ma[e, 0] @ act_row.astype(np.float64))))
        contrib[p] = M.bf16((y * tw.reshape(-1)[p]).astype(np.float32))
    return M.topk_sum(contrib, ids, E)


@pytest.mark.parametrize("which", ["both", "gate_up", "down"])
@pytest.mark.parametrize("E, T, topk, H, I, rank, act", [
    (8, 6, 2, 256, 128, 8, "silu"), (16, 40, 4, 384, 256, 20, "gelu"), (64, 150, 4, 512, 256, 16, "silu"),
    (64, 100, 2, 384, 128, 5, "gelu"),
])
def test_layer_against_the_oracle(E, T, topk, H, I, rank, act, which):
    _, moe, _ = _mods()
    rng = np.random.default_rng(E + T)
    weights = M.random_experts(rng, E, H, I)
    dev = [torch.from_numpy(a).cuda() for a in weights]
    made, mats = _adapters(3, E, H, I, rank, T, which)
    x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(torch.bfloat16).cuda()
    ids = np.stack([rng.permutation(E)[:topk] for _ in range(T)]).astype(np.int64)
    ids[0, 0] = -1
    tw = rng.random((T, topk)).astype(np.float32)
    who = rng.integers(-1, 3, T).astype(np.int32)
    args = (x, torch.from_numpy(tw).cuda(), torch.from_numpy(ids).cuda(), *dev)
    out = moe.fused_moe(*args, activation=act, adapters=made, adapter_ids=torch.from_numpy(who).cuda())
    ref = _oracle(x.float().cpu().numpy(), tw, ids, who, weights, mats, act)
    _check_close(out.float().cpu().numpy(), ref, f"{which} E={E} T={T}")
    # A token without an adapter gets the bits of the layer without adapters; another does not.
    plain = moe.fused_moe(*args, activation=act)
    none = torch.from_numpy(who < 0).cuda()
    assert same(out[none], plain[none]) and not same(out[~none], plain[~none])


@pytest.mark.parametrize("compress, R", [(True, 16), (False, 64)])
def test_pager_with_adapters_matches_one_shot(tmp_path, compress, R):
    """Decode steps, and prefills through the working slab in chunks, give the one-shot layer's bits."""
    _, moe, _ = _mods()
    m = Model(tmp_path, 64, 16, R, 8, compress)
    try:
        H, I = 256, 128
        made, _ = _adapters(4, m.E, H, I, 16, 3)
        rng = np.random.default_rng(1)
        layer = m.layers[0]
        for T in (1, 3, 40, 2, 200):
            x, tw, ids = routing(rng, T, m.E, 4)
            who = torch.from_numpy(rng.integers(-1, 4, T)).cuda()
            out = layer.forward(x, tw, ids, adapters=made, adapter_ids=who)
            want = moe.fused_moe(x, tw, ids, *m.weights[0], adapters=made, adapter_ids=who)
            assert same(out, want), f"{T} tokens"
            assert same(layer.forward(x, tw, ids), m.one_shot(0, x, tw, ids))
    finally:
        m.close()


def test_router_to_experts_in_a_graph():
    """Logits to layer output in one captured graph (a padded batch), replayed on changed tokens; and eagerly."""
    lora, moe, router = _mods()
    E, H, I, T, topk = 32, 256, 128, 24, 4
    rng = np.random.default_rng(0)
    dev = [torch.from_numpy(a).cuda() for a in M.random_experts(rng, E, H, I)]
    made, _ = _adapters(2, E, H, I, 8, 1)
    sets = []
    for i in range(3):
        z = torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32)).to(torch.bfloat16).cuda()
        x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(torch.bfloat16).cuda()
        who = torch.from_numpy(rng.integers(-1, 2, T)).cuda()
        sets.append((z, x, who, torch.arange(T, device="cuda") < T - 3 * i))

    def layer(z, x, who, mask):
        tw, ids, loss, counts = router.choose_and_balance(z, topk, mask=mask)
        return moe.fused_moe(x, tw, ids, *dev, adapters=made, adapter_ids=who), loss, counts

    want = [layer(*s) for s in sets]
    for (y, _, counts), s in zip(want, sets):
        assert int(counts.sum()) == topk * int(s[3].sum())
        assert (y[~s[3]] == 0).all() and y[s[3]].abs().sum() > 0
    buf = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(*buf)
    for i in (1, 0, 2, 1):
        for d, s in zip(buf, sets[i]):
            d.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        layer(*sets[0])[0].sum().item()


def test_refusals():
    lora, moe, _ = _mods()
    rng = np.random.default_rng(0)
    E, H, I = 4, 256, 128
    dev = [torch.from_numpy(a).cuda() for a in M.random_experts(rng, E, H, I)]
    x = torch.zeros((3, H), dtype=torch.bfloat16, device="cuda")
    tw, ids = torch.ones((3, 2), device="cuda"), torch.zeros((3, 2), dtype=torch.int64, device="cuda")
    who = torch.zeros((3,), dtype=torch.int32, device="cuda")

    def call(made, who=who):
        return moe.fused_moe(x, tw, ids, *dev, adapters=made, adapter_ids=who)

    S = lora.LowRankAdapters
    for made in (lora.ExpertAdapters(gate_up=S(1, E, H, 2 * I, 4)), lora.ExpertAdapters(down=S(1, E, H, I, 4)),
                 lora.ExpertAdapters(down=S(1, E + 1, I, H, 4)),
                 lora.ExpertAdapters(down=S(1, E, I, H, 4, dtype=torch.float16)),
                 lora.ExpertAdapters(S(1, E, H, 2 * I, 4, slices=2), S(2, E, I, H, 4))):
        with pytest.raises(ValueError):
            call(made)
    good = lora.ExpertAdapters(down=S(1, E, I, H, 4))
    none = moe.fused_moe(x[:0], tw[:0], ids[:0], *dev, adapters=good, adapter_ids=who[:0])
    assert tuple(none.shape) == (0, H)
    for bad in (None, who[:2], who.cpu(), who.float()):
        with pytest.raises(ValueError):
            call(good, bad)
    with pytest.raises(ValueError):
        call(None)
    assert same(call(good), moe.fused_moe(x, tw, ids, *dev))  # an adapter that was never loaded
    assert same(call(lora.ExpertAdapters()), moe.fused_moe(x, tw, ids, *dev))


@pytest.mark.parametrize("which", ["both", "gate_up", "down"])
@pytest.mark.parametrize("L, E, T, topk, H, I, rank, act", [(4, 64, 150, 4, 256, 128, 16, "silu"),
                                                            (5, 64, 120, 4, 384, 256, 30, "gelu")])
def test_layer_of_many_groups_against_the_oracle(L, E, T, topk, H, I, rank, act, which):
    """256 groups of (adapter, expert) and more: the adapters' terms by tiles of 64 pairs; one expert that most tokens
    choose, so that tiles are filled."""
    _, moe, _ = _mods()
    rng = np.random.default_rng(L + T)
    weights = M.random_experts(rng, E, H, I)
    dev = [torch.from_numpy(a).cuda() for a in weights]
    made, mats = _adapters(L, E, H, I, rank, T, which)
    x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(torch.bfloat16).cuda()
    ids = np.stack([rng.permutation(E)[:topk] for _ in range(T)]).astype(np.int64)
    ids[:, 1][(ids != 7).all(1)] = 7
    ids[0, 0] = -1
    tw = rng.random((T, topk)).astype(np.float32)
    who = np.where(rng.random(T) < 0.6, 1, rng.integers(-1, L, T)).astype(np.int32)
    assert L * E >= 256 and ((who == 1)[:, None] & (ids == 7)).sum() > 64
    args = (x, torch.from_numpy(tw).cuda(), torch.from_numpy(ids).cuda(), *dev)
    out = moe.fused_moe(*args, activation=act, adapters=made, adapter_ids=torch.from_numpy(who).cuda())
    ref = _oracle(x.float().cpu().numpy(), tw, ids, who, weights, mats, act)
    _check_close(out.float().cpu().numpy(), ref, f"{which} L={L} E={E} T={T}")
    plain = moe.fused_moe(*args, activation=act)
    none = torch.from_numpy(who < 0).cuda()
    assert same(out[none], plain[none]) and not same(out[~none], plain[~none])
