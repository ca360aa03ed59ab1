"""GPU parity of the low-rank adapters (csrc/lora.hip) against the products in 64 bits.

Tolerance, per value, with U = 2^-24 and h = half a step of the type (bf16
2^-8, fp16 2^-11, relative): the inner product u_r is an fp32 sum of K products
of which each carries at most K roundings, |du_r| <= 2 K U sum_k |A x| (the
matrix unit's sums are taken to lose up to twice an fp32 add's rounding); u
enters the second product as two values of the type, losing h^2 of it (bf16
2^-16); that product adds 2 R U of its terms' magnitude. The result is rounded
once: h of itself. All magnitudes are taken from sum |B| (|A| |x|).
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}  # half the least step


def _lora():
    from vllm_expert_pager import lora

    return lora


def _stack(L, E, K, n, ranks, slices, dtype, max_rank, seed, scale=1.7):
    """A loaded stack, its matrices per adapter, and the scales."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    stack = _lora().LowRankAdapters(L, E, K, slices * n, max_rank, slices=slices, dtype=dtype)
    mats = []
    for i in range(L):
        r = ranks[i % len(ranks)]
        if r == 0:
            mats.append(None)
            continue
        a = (torch.randn((E, slices, r, K), generator=g, device="cuda") / K**0.5).to(dtype)
        b = (0.5 * torch.randn((E, slices, n, r), generator=g, device="cuda")).to(dtype)
        stack.load(i, a, b, scale / (i + 1))
        mats.append((a, b, np.float32(scale / (i + 1))))
    return stack, mats


def _ref(x, mats, adapter, ids, slices, n, K, base, per_pair, dtype):
    """(value, bound) in 64 bits."""
    T = adapter.numel()
    k = 1 if ids is None else ids.shape[1]
    P = T * k
    out = torch.zeros((P, slices * n), dtype=torch.float64, device="cuda") if base is None else base.double()
    mag = torch.zeros_like(out)
    h = HALF[dtype]
    for p in range(P):
        a, e = int(adapter[p // k]), 0 if ids is None else int(ids.reshape(-1)[p])
        if not 0 <= a < len(mats) or mats[a] is None or not 0 <= e < mats[a][0].shape[0]:
            continue
        ma, mb, sc = mats[a]
        xr = x[p if per_pair else p // k].double()
        r = ma.shape[2]
        for s in range(slices):
            A, B = ma[e, s].double(), mb[e, s].double()
            out[p, s * n : (s + 1) * n] += float(sc) * (B @ (A @ xr))
            mag[p, s * n : (s + 1) * n] += abs(float(sc)) * (2 * (K + r) * U + h * h) * (B.abs() @ (A.abs() @ xr.abs()))
    return out, mag + 4 * U * out.abs() + h * 1.01 * out.abs() + TINY[dtype]


CASES = [
    # T, E, topk, K, n, slices, ranks, max_rank, L, dtype, per_pair, with base
    (1, 1, 1, 8, 8, 1, [1], 1, 1, torch.bfloat16, False, False),
    (1, 16, 8, 256, 128, 2, [16], 16, 3, torch.bfloat16, False, False),
    (5, 1, 1, 40, 24, 1, [4, 7], 8, 2, torch.float16, False, True),
    (64, 1, 1, 264, 136, 1, [16, 0, 64, 33], 64, 5, torch.float16, False, True),
    (65, 1, 1, 264, 136, 1, [16, 0, 64, 33], 64, 5, torch.bfloat16, False, True),
    (8, 64, 8, 512, 256, 1, [32, 5], 32, 4, torch.bfloat16, True, False),
    (40, 8, 3, 384, 120, 2, [96, 70], 96, 3, torch.bfloat16, False, True),
    (200, 4, 2, 136, 512, 1, [128, 100, 1], 128, 3, torch.float16, True, False),
    (300, 1, 1, 1000, 72, 3, [12], 12, 1, torch.bfloat16, False, False),
    (130, 256, 4, 128, 64, 1, [8], 8, 20, torch.bfloat16, False, False),
    (17, 4, 4, 2048, 2048, 2, [64], 64, 2, torch.bfloat16, False, True),
]


@pytest.mark.parametrize("T, E, topk, K, n, slices, ranks, max_rank, L, dtype, per_pair, with_base", CASES)
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_against_the_products(T, E, topk, K, n, slices, ranks, max_rank, L, dtype, per_pair, with_base, wide):
    g = torch.Generator(device="cuda").manual_seed(T + K)
    stack, mats = _stack(L, E, K, n, ranks, slices, dtype, max_rank, 5)
    P = T * topk
    x = torch.randn((P if per_pair else T, K), generator=g, device="cuda").to(dtype)
    base = torch.randn((P, slices * n), generator=g, device="cuda").to(dtype) if with_base else None
    adapter = torch.randint(-2, L + 1, (T,), generator=g, device="cuda").to(wide)  # some of them out of range
    adapter[0] = 0
    ids = None
    if E > 1:
        ids = torch.rand((T, E), generator=g, device="cuda").argsort(1)[:, :topk].to(wide)
        ids[0, 0] = 0
        if T > 3:
            ids[1, 0], ids[2, 0] = -1, E
            ids[3] = 1  # the same expert several times
    got = _lora().low_rank(x, stack, adapter, ids, base=base)
    ref, bound = _ref(x, mats, adapter, ids, slices, n, K, base, per_pair, dtype)
    assert got.dtype == dtype and tuple(got.shape) == (P, slices * n)
    err = (got.double() - ref).abs()
    assert (err <= bound).all(), float((err / bound).max())
    # Pairs without an adapter: base as it was, or zeros.
    k = topk
    none = torch.tensor([not 0 <= int(adapter[p // k]) < L or (ids is not None and not 0 <= int(ids.reshape(-1)[p]) < E)
                         for p in range(P)], device="cuda")
    assert torch.equal(got[none], base[none] if base is not None else torch.zeros_like(got[none]))


@pytest.mark.parametrize("L, E, T, topk, dtype", [
    (20, 256, 900, 4, torch.bfloat16),  # thousands of groups, some of many pairs
    (2, 1, 6000, 1, torch.bfloat16),  # two groups of thousands
    (3, 2, 20000, 1, torch.float16),  # tiles of 64 by the number of pairs
    (1, 40, 130, 2, torch.bfloat16),  # just above what a workgroup groups itself
    (1, 40, 128, 2, torch.bfloat16),  # and the most that it does
])
def test_any_order_and_any_split(L, E, T, topk, dtype):
    """The order of the tokens changes no bit, nor does a second run; calls of a few tokens each agree within the
    roundings: their sums run over other parts of K, two fp32 sums of K products apart at most, then one rounding."""
    lora = _lora()
    g = torch.Generator(device="cuda").manual_seed(0)
    K, n = 128, 64
    stack, mats = _stack(L, E, K, n, [16, 3], 1, dtype, 16, 1)
    x = torch.randn((T, K), generator=g, device="cuda").to(dtype)
    adapter = torch.randint(-1, L, (T,), generator=g, device="cuda")
    adapter[::3] = L // 2
    ids = torch.rand((T, E), generator=g, device="cuda").argsort(1)[:, :topk].to(torch.int32).contiguous()
    if E > 11:
        ids[::2, 0] = 11
    experts = ids if E > 1 else None
    whole = lora.low_rank(x, stack, adapter, experts)
    assert torch.equal(whole, lora.low_rank(x, stack, adapter, experts))
    turn = torch.randperm(T, generator=g, device="cuda")
    turned = lora.low_rank(x[turn], stack, adapter[turn], None if experts is None else experts[turn])
    assert torch.equal(whole.view(T, topk, n)[turn], turned.view(T, topk, n))
    step = 16
    some = range(0, min(T, 2000), step)
    parts = torch.cat([lora.low_rank(x[t : t + step], stack, adapter[t : t + step],
                                     None if experts is None else experts[t : t + step]) for t in some])
    a, b = whole[: parts.shape[0]].double(), parts.double()
    # sum |B| (|A| |x|) is at most the largest row sum of B times that of A times the largest |x|
    reach = max(float(m[2]) * m[1].double().abs().sum(-1).max().item() * m[0].double().abs().sum(-1).max().item()
                for m in mats) * x.double().abs().max().item()
    assert ((a - b).abs() <= 2 * HALF[dtype] * 1.01 * torch.maximum(a.abs(), b.abs()) + 4 * (K + 16) * U * reach).all()


@pytest.mark.parametrize("T", [3, 200])
def test_in_place_strides_and_rows_behind(T):
    """out = base in place, rows apart in every tensor, and the rows behind them left as they were."""
    lora = _lora()
    g = torch.Generator(device="cuda").manual_seed(2)
    stack, _ = _stack(3, 1, 64, 40, [8], 1, torch.bfloat16, 8, 3)
    wide = torch.randn((T + 2, 96), generator=g, device="cuda").to(torch.bfloat16)
    x = wide[1 : T + 1, 16:80]
    y = torch.randn((T + 2, 56), generator=g, device="cuda").to(torch.bfloat16)
    before = y.clone()
    adapter = torch.randint(-1, 3, (T,), generator=g, device="cuda").to(torch.int32)
    want = lora.low_rank(x.contiguous(), stack, adapter, base=y[1 : T + 1, 8:48].contiguous())
    out = lora.low_rank(x, stack, adapter, base=y[1 : T + 1, 8:48], out=y[1 : T + 1, 8:48])
    assert torch.equal(out, want) and out.data_ptr() == y[1:, 8:].data_ptr()
    before[1 : T + 1, 8:48] = want
    assert torch.equal(y, before)


def test_loading_and_clearing():
    """A place that is loaded again with a smaller rank holds nothing of the old adapter; a cleared one adds nothing."""
    lora = _lora()
    g = torch.Generator(device="cuda").manual_seed(4)
    stack = lora.LowRankAdapters(2, 3, 72, 48, 40, slices=2)
    fresh = lora.LowRankAdapters(2, 3, 72, 48, 40, slices=2)
    big = [torch.randn(s, generator=g, device="cuda") for s in ((3, 2, 40, 72), (3, 2, 24, 40))]
    small = [torch.randn(s, generator=g, device="cuda") for s in ((3, 2, 3, 72), (3, 2, 24, 3))]
    stack.load(1, *big, 2.0)
    stack.load(1, *small, 0.5)
    fresh.load(1, *small, 0.5)
    for name in ("a", "b", "scales", "ranks"):
        assert torch.equal(getattr(stack, name), getattr(fresh, name))
    x = torch.randn((5, 72), generator=g, device="cuda").to(torch.bfloat16)
    ids = torch.tensor([[0, 1], [2, 1], [0, 2], [1, 0], [2, 0]], device="cuda")
    who = torch.ones((5,), dtype=torch.int32, device="cuda")
    assert lora.low_rank(x, stack, who, ids).abs().sum() > 0
    stack.clear(1)
    assert (lora.low_rank(x, stack, who, ids) == 0).all()
    assert (lora.low_rank(x, stack, who - 1, ids) == 0).all()  # never loaded
    one = lora.LowRankAdapters(1, 1, 72, 24, 8)
    one.load(0, torch.ones((4, 72)), torch.ones((24, 4)))  # without the experts' and slices' dimensions, from the host
    assert (lora.low_rank(torch.ones_like(x), one, who - 1) == 288).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_extreme_values(dtype):
    """Infinite and NaN tokens stay in their rows, and unused ranks and columns add nothing to them; huge and tiny
    inner products keep their precision in fp16."""
    lora = _lora()
    stack = lora.LowRankAdapters(1, 1, 40, 8, 5, dtype=dtype)
    a, b = torch.ones((5, 40)), torch.ones((8, 5))
    stack.load(0, a, b, 1.0)
    x = torch.ones((70, 40), dtype=dtype, device="cuda")
    x[1, 39] = float("inf")
    x[2, 0] = float("nan")
    x[3] = 60000.0  # u = 2.4e6, beyond fp16; the result is infinite there
    x[4] = 2.0**-24
    who = torch.zeros((70,), dtype=torch.int32, device="cuda")
    y = lora.low_rank(x, stack, who)
    assert (y[0] == 200).all() and (y[5:] == 200).all()
    assert torch.isinf(y[1]).all() and torch.isnan(y[2]).all()
    want = (x[3, 0].double() * 200).to(dtype)
    assert torch.equal(y[3], want.expand(8))
    assert torch.equal(y[4], torch.full((8,), 200 * 2.0**-24, dtype=torch.float64, device="cuda").to(dtype))
    stack.load(0, a, b, 2.0**-12)  # u beyond fp16, the result inside it: no overflow on the way
    y = lora.low_rank(x, stack, who)
    want = (x[3, 0].double() * 200 * 2.0**-12).to(dtype)
    assert torch.equal(y[3], want.expand(8))


def test_no_tokens():
    lora = _lora()
    stack = lora.LowRankAdapters(2, 4, 16, 16, 4)
    x = torch.empty((0, 16), dtype=torch.bfloat16, device="cuda")
    ids = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    assert tuple(lora.low_rank(x, stack, ids[:, 0].contiguous(), ids).shape) == (0, 16)


@pytest.mark.parametrize("T", [4, 100, 200])
def test_graph_and_stream(T):
    """Captured and replayed on changed tokens, adapters and experts; a call on a side stream."""
    lora = _lora()
    g = torch.Generator(device="cuda").manual_seed(6)
    stack, _ = _stack(4, 16, 128, 64, [16, 7], 2, torch.bfloat16, 16, 9)
    sets = []
    for _ in range(3):
        x = torch.randn((T, 128), generator=g, device="cuda").to(torch.bfloat16)
        who = torch.randint(-1, 4, (T,), generator=g, device="cuda")
        ids = torch.rand((T, 16), generator=g, device="cuda").argsort(1)[:, :2].contiguous()
        sets.append((x, who, ids, lora.low_rank(x, stack, who, ids)))
    buf = [t.clone() for t in sets[0][:3]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lora.low_rank(buf[0], stack, buf[1], buf[2])
    for i in (1, 2, 0, 1):
        for d, s in zip(buf, sets[i]):
            d.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, sets[i][3])
        lora.low_rank(sets[0][0], stack, sets[0][1], sets[0][2]).sum().item()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = lora.low_rank(*sets[2][:1], stack, *sets[2][1:3])
    side.synchronize()
    assert torch.equal(y, sets[2][3])


def test_refusals():
    lora = _lora()
    for bad in (dict(max_rank=129), dict(max_rank=0), dict(in_features=12), dict(out_features=20), dict(adapters=0),
                dict(adapters=1 << 12, experts=1 << 8), dict(slices=3), dict(dtype=torch.float32)):
        how = {**dict(adapters=2, experts=4, in_features=16, out_features=32, max_rank=8), **bad}
        with pytest.raises(ValueError):
            lora.LowRankAdapters(**how)
    s = lora.LowRankAdapters(2, 4, 16, 32, 8)
    for a, b in (((4, 1, 9, 16), (4, 1, 32, 9)), ((4, 1, 4, 16), (4, 1, 32, 5)), ((3, 1, 4, 16), (4, 1, 32, 4)),
                 ((4, 1, 4, 8), (4, 1, 32, 4))):
        with pytest.raises(ValueError):
            s.load(0, torch.zeros(a), torch.zeros(b))
    with pytest.raises(ValueError):
        s.load(2, torch.zeros((4, 1, 4, 16)), torch.zeros((4, 1, 32, 4)))
    with pytest.raises(ValueError):
        s.clear(-1)
    x = torch.zeros((3, 16), dtype=torch.bfloat16, device="cuda")
    who = torch.zeros((3,), dtype=torch.int32, device="cuda")
    ids = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    bad = [
        lambda: lora.low_rank(x, s, who),  # four experts, no ids
        lambda: lora.low_rank(x[:2], s, who, ids),
        lambda: lora.low_rank(x.half(), s, who, ids),
        lambda: lora.low_rank(x.cpu(), s, who, ids),
        lambda: lora.low_rank(x, s, who.cpu(), ids),
        lambda: lora.low_rank(x, s, who.float(), ids),
        lambda: lora.low_rank(x, s, who, ids[:2]),
        lambda: lora.low_rank(x, s, who[:, None], ids),
        lambda: lora.low_rank(x.t().contiguous().t(), s, who, ids),
        lambda: lora.low_rank(x, s, who, ids, base=torch.zeros((5, 32), dtype=torch.bfloat16, device="cuda")),
        lambda: lora.low_rank(x, s, who, ids, out=torch.zeros((6, 32), device="cuda")),
        lambda: lora.low_rank(torch.zeros((3, 20), dtype=torch.bfloat16, device="cuda")[:, :16], s, who, ids),
        lambda: lora.low_rank(torch.zeros((3, 24), dtype=torch.bfloat16, device="cuda")[:, 4:20], s, who, ids),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_offsets_past_32_bits():
    """More than 2^31 values of x and of the result: the last rows get what a call of their own gives."""
    lora = _lora()
    g = torch.Generator(device="cuda").manual_seed(8)
    T, K, n, tail = (1 << 20) + 256, 2048, 2048, 256
    stack, _ = _stack(2, 1, K, n, [8], 1, torch.bfloat16, 8, 3)
    x = torch.zeros((T, K), dtype=torch.bfloat16, device="cuda")
    x[-tail:] = torch.randn((tail, K), generator=g, device="cuda").to(torch.bfloat16)
    assert x.numel() > 1 << 31
    who = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    who[-tail:] = torch.arange(tail, device="cuda") % 3 - 1
    y = lora.low_rank(x, stack, who)
    own = lora.low_rank(x[-tail:].contiguous(), stack, who[-tail:].contiguous())
    d = (y[-tail:].double() - own.double()).abs()
    assert (d <= 2 * 1.01 * HALF[torch.bfloat16] * own.double().abs() + 1e-4).all()  # other parts of K, one rounding each
    assert y[: T - tail].abs().max() == 0 and own[who[-tail:] >= 0].abs().sum() > 0


# Tiles of 64 pairs: listings of 256 groups or of 16384 pairs at least. A call that lists for itself takes 16-pair tiles
# instead where it has one slice (or three) of rank 16, the large cases of test_any_order_and_any_split among them, or
# rank 96 or 128; from a listing of lora.group it gets tiles of 64 too.

GROUP_SIZES = [1, 16, 17, 33, 63, 64, 65, 130]


def _grouped_batch(L, E, topk, sizes, seed):
    """(adapter, ids) whose groups have these sizes; tokens without an adapter and pairs without an expert among them,
    in random order."""
    rng = np.random.default_rng(seed)
    cells = rng.permutation(L * E)[: len(sizes)]
    adapter, ids = [], []
    for cell, size in zip(cells, sizes):
        a, e = divmod(int(cell), E)
        for left in range(size, 0, -topk):
            row = [e] * min(left, topk) + [-1] * (topk - min(left, topk))
            adapter.append(a)
            ids.append(rng.permutation(row))
    for a in (-1, L, -1, 0, 0):
        adapter.append(a)
        ids.append(rng.integers(0, E, topk) if not 0 <= a < L else np.full(topk, E))
    order = rng.permutation(len(adapter))
    return (torch.from_numpy(np.array(adapter)[order]).to(torch.int32).cuda(),
            torch.from_numpy(np.stack(ids)[order].astype(np.int64)).cuda())


def _ref_by_group(x, mats, adapter, ids, slices, n, K, base, per_pair, dtype):
    """_ref, a group of pairs at a time."""
    T, k = ids.shape
    out = torch.zeros((T * k, slices * n), dtype=torch.float64, device="cuda") if base is None else base.double()
    mag, h = torch.zeros_like(out), HALF[dtype]
    a, e = adapter.cpu().numpy().repeat(k), ids.cpu().numpy().reshape(-1)
    for i, m in enumerate(mats):
        if m is None:
            continue
        for j in range(m[0].shape[0]):
            p = np.flatnonzero((a == i) & (e == j))
            if not p.size:
                continue
            p = torch.from_numpy(p).cuda()
            rows = x[p if per_pair else p // k].double()
            r, sc = m[0].shape[2], float(m[2])
            for s in range(slices):
                A, B = m[0][j, s].double().t().contiguous(), m[1][j, s].double().t().contiguous()
                c = slice(s * n, (s + 1) * n)
                out[p, c] += sc * ((rows @ A) @ B)
                mag[p, c] += abs(sc) * (2 * (K + r) * U + h * h) * ((rows.abs() @ A.abs()) @ B.abs())
    return out, mag + 4 * U * out.abs() + h * 1.01 * out.abs() + TINY[dtype]


def _check_grouped(got, ref, bound, adapter, ids, L, E, base):
    err = (got.double() - ref).abs()
    assert (err <= bound).all(), float((err / bound).max())
    k = ids.shape[1]
    a, e = adapter.repeat_interleave(k), ids.reshape(-1)
    none = (a < 0) | (a >= L) | (e < 0) | (e >= E)
    assert torch.equal(got[none], base[none] if base is not None else torch.zeros_like(got[none]))


TILES = [
    # K, n, slices, ranks, max_rank
    (72, 40, 2, [16, 5], 16),
    (1000, 264, 2, [9, 16], 16),
    (200, 72, 2, [32, 0, 20], 32),
    (520, 136, 1, [32, 17], 32),
    (72, 200, 3, [32, 3], 32),
    (200, 264, 1, [64, 33, 40], 64),
    (1000, 40, 2, [64, 2], 64),
    (264, 72, 1, [96, 65], 96),
    (136, 520, 2, [128, 100, 7], 128),
]


@pytest.mark.parametrize("topk, per_pair, with_base", [(1, False, True), (2, False, False), (3, True, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K, n, slices, ranks, max_rank", TILES)
def test_tiles_of_64_pairs(K, n, slices, ranks, max_rank, dtype, topk, per_pair, with_base):
    L, E = 4, 64
    g = torch.Generator(device="cuda").manual_seed(K + n)
    stack, mats = _stack(L, E, K, n, ranks, slices, dtype, max_rank, 5)
    adapter, ids = _grouped_batch(L, E, topk, GROUP_SIZES, K + topk)
    P = ids.numel()
    assert L * E >= 256 and P > 256
    x = torch.randn((P if per_pair else P // topk, K), generator=g, device="cuda").to(dtype)
    base = torch.randn((P, slices * n), generator=g, device="cuda").to(dtype) if with_base else None
    got = _lora().low_rank(x, stack, adapter, ids, base=base)
    ref, bound = _ref_by_group(x, mats, adapter, ids, slices, n, K, base, per_pair, dtype)
    _check_grouped(got, ref, bound, adapter, ids, L, E, base)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K, n, slices, max_rank", [(72, 264, 1, 16), (520, 40, 3, 16), (200, 72, 1, 32),
                                                        (264, 72, 1, 96), (136, 520, 2, 128)])
def test_tiles_of_64_pairs_from_a_listing(K, n, slices, max_rank, dtype):
    """From a listing that several projections share, whole and by an expert_map; pairs whose expert has no slot keep
    what stood in their rows."""
    lora, (L, E, topk) = _lora(), (4, 64, 2)
    g = torch.Generator(device="cuda").manual_seed(K)
    stack, mats = _stack(L, E, K, n, [max_rank, 3], slices, dtype, max_rank, 6)
    adapter, ids = _grouped_batch(L, E, topk, GROUP_SIZES, K)
    P = ids.numel()
    x = torch.randn((P, K), generator=g, device="cuda").to(dtype)
    ref, bound = _ref_by_group(x, mats, adapter, ids, slices, n, K, None, True, dtype)
    out = torch.full((P, slices * n), 3.0, dtype=dtype, device="cuda")
    lora.apply(x, stack, adapter, ids, P // topk, topk, True, None, out,
               listing=lora.group(stack, adapter, ids, None, 0))
    _check_grouped(out, ref, bound, adapter, ids, L, E, None)
    emap = torch.arange(E, dtype=torch.int32, device="cuda") % 2 * 40 + torch.arange(E, dtype=torch.int32, device="cuda") - 8
    slots = 50  # experts below 8 (even) have none, and those whose entry is 50 or more
    out.fill_(3.0)
    lora.apply(x, stack, adapter, ids, P // topk, topk, True, None, out, expert_map=emap, slots=slots,
               listing=lora.group(stack, adapter, ids, emap, slots))
    e = ids.reshape(-1)
    at = emap[e.clamp(0, E - 1)]
    routed = (e >= 0) & (e < E) & (at >= 0) & (at < slots)
    assert routed.any() and not routed.all()
    assert ((out.double() - ref).abs() <= bound)[routed].all()
    assert (out[~routed] == 3).all()


@pytest.mark.parametrize("max_rank, slices, dtype", [(32, 1, torch.float16), (16, 2, torch.bfloat16),
                                                     (64, 1, torch.bfloat16), (128, 1, torch.float16)])
def test_tiles_of_64_pairs_by_their_number(max_rank, slices, dtype):
    """Few groups of thousands of pairs each, the last tile of a group in part."""
    T, L, K, n = 16384 + 37, 3, 136, 72
    g = torch.Generator(device="cuda").manual_seed(max_rank)
    stack, mats = _stack(L, 1, K, n, [max_rank, 7], slices, dtype, max_rank, 8)
    x = torch.randn((T, K), generator=g, device="cuda").to(dtype)
    adapter = torch.randint(-1, L, (T,), generator=g, device="cuda")
    ids = torch.zeros((T, 1), dtype=torch.int32, device="cuda")
    got = _lora().low_rank(x, stack, adapter)
    ref, bound = _ref_by_group(x, mats, adapter, ids, slices, n, K, None, False, dtype)
    _check_grouped(got, ref, bound, adapter, ids, L, 1, None)
