"""GPU parity of the router kernels (csrc/router.hip) against plain formulas in 64 bits.

Tolerances, per value (U = 2^-24, half a step of fp32):
- weights: the terms e^(z - m) carry the exponential's error (the library's
  fp32 exp: 1 ulp, two half steps) and that of the rounded difference z - m,
  |z - m| U absolute; the sum over E terms in a tree of lanes and at most 32
  serial adds adds (32 + 6) U; then a division and a product: relative error
  below (64 + |z - m|) U. The logits are within +-8 of each other but for the
  extreme rows, whose bound takes their own span.
- loss: P_e sums fp32 probabilities serially over at most T / parts rows and
  joins them in 64 bits: (rows + 64 + span) U relative, all terms positive.
- gradient: p (G - sum G p): the difference of sums of the magnitude max|G|,
  error (2 x 64 + E) U p max|G|, then half a step of the gradient's type.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
NEG = -math.inf


def _router():
    from vllm_expert_pager import router

    return router


def _logits(T, E, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * (torch.randn((T, E), generator=g) + 0.4 * torch.randn((E,), generator=g))).to(dtype)


def _score(z, scoring):
    """(score, p) in 64 bits; masked logits (NaN, -inf) have neither."""
    live = z > NEG  # False for NaN
    if scoring == "softmax":
        m = np.max(np.where(live, z, NEG), axis=1, keepdims=True)
        with np.errstate(invalid="ignore", over="ignore"):
            d = np.where(z == m, 0.0, z - m)
        e = np.where(live, np.exp(np.where(live, d, 0.0)), 0.0)
        p = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
        return p, p
    with np.errstate(over="ignore"):
        s = np.where(live, 1.0 / (1.0 + np.exp(-np.where(live, z, 0.0))), 0.0)
    return s, s / np.maximum(s.sum(1, keepdims=True), 1e-300)


def _choose_ref(z, k, scoring="softmax", renorm=True, bias=None, groups=1, keep=1, scale=1.0, mask=None):
    T, E = z.shape
    score, _ = _score(z, scoring)
    key = np.where(z > NEG, z if bias is None else score + bias, NEG)
    key = np.where(key > NEG, key, NEG)
    ids = np.full((T, k), -1)
    w = np.zeros((T, k))
    for t in range(T):
        if mask is not None and not mask[t]:
            continue
        kt = key[t].copy()
        if groups > 1:
            worth = []
            for g in kt.reshape(groups, -1):
                best = sorted((v for v in g if v > NEG), reverse=True)
                worth.append(NEG if not best else best[0] if bias is None else sum(best[:2]))
            order = sorted((g for g in range(groups) if worth[g] > NEG), key=lambda g: (-worth[g], g))[:keep]
            kt = np.where(np.isin(np.arange(E) // (E // groups), order), kt, NEG)
        best = sorted((e for e in range(E) if kt[e] > NEG), key=lambda e: (-kt[e], e))[:k]
        ids[t, : len(best)] = best
        w[t, : len(best)] = score[t, best]
    if renorm:  # by the logarithms of the scores, which do not underflow
        live = ids >= 0
        chosen = np.where(live, np.take_along_axis(z, np.maximum(ids, 0), 1), 0.0)
        log = np.minimum(chosen, 0) - np.log1p(np.exp(-np.abs(chosen))) if scoring == "sigmoid" else chosen
        log = np.where(live, log, NEG)
        top = log.max(1, keepdims=True)
        w = np.where(live, np.exp(np.where(live, log, 0.0) - np.where(top > NEG, top, 0.0)), 0.0)
        w = w / np.maximum(w.sum(1, keepdims=True), 1.0)
    return w * scale, ids


def _span(z):
    """The rows' largest |z - m| among finite logits."""
    live = np.isfinite(z)
    top, least = np.where(live, z, NEG).max(1, keepdims=True), np.where(live, z, math.inf).min(1, keepdims=True)
    return np.where(live.any(1, keepdims=True), top - np.where(live.any(1, keepdims=True), least, 0.0), 0.0)


def _check_weights(w, ref, z):
    got = w.detach().double().cpu().numpy()
    bound = (64 + _span(z)) * U * np.abs(ref) + 2.0**-149
    assert (np.abs(got - ref) <= bound).all(), float((np.abs(got - ref) / bound).max())


CHOICES = [
    # T, E, k, dtype, options
    (1, 1, 1, torch.float32, {}),
    (1, 256, 8, torch.bfloat16, {}),
    (3, 2, 2, torch.float16, {"renorm": False}),
    (65, 60, 4, torch.float16, {"renorm": False}),
    (130, 61, 7, torch.bfloat16, {"scale": 2.5}),
    (64, 128, 6, torch.float32, {"scoring": "sigmoid"}),
    (33, 160, 6, torch.float32, {"scoring": "sigmoid", "renorm": False, "scale": 16.0}),
    (257, 256, 8, torch.float32, {"scoring": "sigmoid", "bias": True, "groups": 8, "keep": 4, "scale": 2.5}),
    (70, 256, 8, torch.bfloat16, {"scoring": "sigmoid", "bias": True, "groups": 8, "keep": 3}),
    (40, 96, 5, torch.float32, {"groups": 12, "keep": 2}),
    (40, 64, 3, torch.bfloat16, {"groups": 64, "keep": 3}),
    (37, 64, 3, torch.float32, {"bias": True}),
    (12, 1000, 10, torch.float32, {"bias": True, "groups": 10, "keep": 7}),
    (9, 2048, 64, torch.bfloat16, {}),
    (7, 513, 33, torch.float32, {"renorm": False}),
    (5, 1025, 1, torch.float32, {"scoring": "sigmoid", "renorm": False}),
]


@pytest.mark.parametrize("T, E, k, dtype, how", CHOICES)
def test_choice(T, E, k, dtype, how):
    router = _router()
    logits = _logits(T, E, dtype, T + E)
    how = dict(how)
    bias = None
    if how.pop("bias", False):
        bias = 0.2 * torch.randn((E,), generator=torch.Generator().manual_seed(E))
    renorm, keep = how.pop("renorm", True), how.pop("keep", 1)
    w, ids = router.choose_experts(logits.cuda(), k, renormalize=renorm, topk_groups=keep,
                                   bias=None if bias is None else bias.cuda(), **how)
    z = logits.double().numpy()
    rw, rids = _choose_ref(z, k, renorm=renorm, keep=keep, bias=None if bias is None else bias.double().numpy(), **how)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    assert np.array_equal(ids.cpu().numpy(), rids)
    _check_weights(w, rw, z)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("bias", [False, True])
def test_ties_masks_and_extremes(scoring, renorm, bias):
    """Ties to the lowest index (-0 and 0 among them), masked logits, rows with fewer than topk or none, padding."""
    router = _router()
    E, k = 37, 5
    z = np.zeros((12, E), np.float32)
    z[0, 3::2] = -0.0
    z[1] = NEG
    z[2] = np.nan
    z[3, 4:] = NEG
    z[4] = np.arange(E) % 3
    z[5] = -3.0e38
    z[6] = np.linspace(-200, 200, E)
    z[7, ::2] = NEG
    z[7, 1] = np.nan
    z[8, 6] = 80.0
    z[9] = -90.0 - np.arange(E) % 4
    z[10] = 3.0e38
    z[11] = np.random.default_rng(0).standard_normal(E)
    mask = np.ones(12, bool)
    mask[11] = False
    b = np.zeros(E, np.float32) if bias else None
    w, ids = router.choose_experts(torch.from_numpy(z).cuda(), k, scoring=scoring, renormalize=renorm,
                                   bias=None if b is None else torch.from_numpy(b).cuda(),
                                   mask=torch.from_numpy(mask).cuda())
    zz = z.astype(np.float64)
    rw, rids = _choose_ref(zz, k, scoring, renorm, None if b is None else b.astype(np.float64), mask=mask)
    assert np.array_equal(ids.cpu().numpy(), rids)
    got = w.cpu().double().numpy()
    assert np.isfinite(got).all()
    # Scores below the least fp32 (2^-149) are 0 there; a row of them renormalises by what 64 bits hold.
    finite = np.minimum(_span(zz), 1e4)
    assert (np.abs(got - rw) <= (64 + finite) * U * rw + 2.0**-148).all()
    assert (rids[[1, 2, 11]] == -1).all() and (got[[1, 2, 11]] == 0).all()
    assert (rids[3, 4:] == -1).all() and (rids[0] == np.arange(5)).all()


def test_infinite_logits():
    """+inf takes all the probability, shared by its holders; the choice puts them first."""
    router = _router()
    z = torch.zeros((2, 8))
    z[0, 5] = math.inf
    z[1, 2] = z[1, 6] = math.inf
    w, ids = router.choose_experts(z.cuda(), 3)
    assert ids.tolist() == [[5, 0, 1], [2, 6, 0]]
    assert w.tolist() == [[1, 0, 0], [0.5, 0.5, 0]]
    w, ids = router.choose_experts(z.cuda(), 3, scoring="sigmoid", renormalize=False)
    assert w.tolist() == [[1, 0.5, 0.5], [1, 1, 0.5]]


def test_rows_apart_and_unaligned():
    """Logits that are a slice of a wider tensor, at any offset; columns apart; no tokens."""
    router = _router()
    wide = _logits(20, 90, torch.bfloat16, 3).cuda()
    for view in (wide[:, 5:65], wide[::2, 1:65], wide[:, 7:67:3], wide.t()[:40], wide[3:4, 2:40]):
        w, ids = router.choose_experts(view, 4)
        rw, rids = _choose_ref(view.double().cpu().numpy(), 4)
        assert np.array_equal(ids.cpu().numpy(), rids)
        _check_weights(w, rw, view.double().cpu().numpy())
    w, ids = router.choose_experts(wide[:0], 4)
    assert tuple(w.shape) == (0, 4) and tuple(ids.shape) == (0, 4)


def _balance_ref(z, ids, k, scoring, on, cuts):
    E = z.shape[1]
    _, p = _score(z, scoring)
    slope = np.ones_like(p)
    if scoring == "sigmoid":
        slope = 1 - _score(z, scoring)[0]
    B = len(cuts) - 1
    counts, losses, grad = np.zeros((B, E), np.int64), [], np.zeros_like(p)
    for b in range(B):
        t = np.arange(cuts[b], cuts[b + 1])
        t = t[on[t]]
        if not t.size:
            continue
        chosen = ids[t].ravel()
        counts[b] = np.bincount(chosen[(chosen >= 0) & (chosen < E)], minlength=E)
        f = counts[b] * E / (k * t.size)
        losses.append((f * p[t].mean(0)).sum())
        grad[t] = p[t] * slope[t] * (f - (p[t] * f).sum(1, keepdims=True)) / t.size
    used = max(len(losses), 1)
    return sum(losses) / used, counts, grad / used


def _grad_bound(grad, p, reach, E, dtype):
    """Half a step of the type, and the sums' error p * reach * (128 + E) U."""
    return HALF[dtype] * np.abs(grad) * 1.01 + p * reach * (128 + E) * U + 2.0**-133 + (
        2.0**-25 if dtype == torch.float16 else 0)


BALANCES = [
    # T, E, k, dtype, scoring, sequences, padded
    (1, 1, 1, torch.float32, "softmax", None, False),
    (1, 64, 2, torch.float32, "softmax", None, False),
    (100, 60, 4, torch.bfloat16, "softmax", None, True),
    (333, 128, 8, torch.float32, "sigmoid", None, False),
    (200, 61, 3, torch.float32, "softmax", [0, 0, 17, 18, 18, 190], False),
    (200, 64, 3, torch.float16, "sigmoid", [5, 60, 130, 200], True),
    (3000, 256, 8, torch.float32, "softmax", None, False),
    (40, 2048, 4, torch.float32, "softmax", [0, 20, 40], False),
    (64, 16, 1, torch.float32, "softmax", list(range(65)), True),
]


@pytest.mark.parametrize("T, E, k, dtype, scoring, cuts, padded", BALANCES)
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_balance(T, E, k, dtype, scoring, cuts, padded, wide):
    router = _router()
    logits = _logits(T, E, dtype, 7 * T + E)
    g = np.random.default_rng(T)
    ids = np.stack([g.permutation(E)[:k] for _ in range(T)])
    ids[g.random((T, k)) < 0.05] = -1
    ids[g.random((T, k)) < 0.02] = E + 3
    if T > 2:
        ids[2] = 1 % E  # the same expert several times
    on = g.random(T) < 0.8 if padded else np.ones(T, bool)
    at = [0, T] if cuts is None else cuts
    on_ref = on.copy()
    on_ref[: at[0]] = False
    on_ref[at[-1] :] = False
    leaf = logits.cuda().requires_grad_(True)
    loss, counts = router.balance_loss(
        leaf, torch.from_numpy(ids).to(wide).cuda(), scoring=scoring, mask=torch.from_numpy(on).cuda() if padded else None,
        seq_offsets=None if cuts is None else torch.tensor(cuts, dtype=wide, device="cuda"))
    (grad,) = torch.autograd.grad(loss, leaf, torch.tensor(512.0, device="cuda"))
    z = logits.double().numpy()
    rl, rc, rg = _balance_ref(z, ids, k, scoring, on_ref, at)
    assert counts.dtype == torch.int32 and tuple(counts.shape) == ((E,) if cuts is None else (len(cuts) - 1, E))
    assert np.array_equal(counts.cpu().numpy().reshape(rc.shape), rc)
    assert abs(loss.item() - rl) <= rl * (T + 64 + _span(z).max()) * U
    assert grad.dtype == dtype
    p = _score(z, scoring)[1]
    used = max(sum(on_ref[a:b].any() for a, b in zip(at, at[1:])), 1)
    reach = np.zeros((T, 1))
    for b, (a, z1) in enumerate(zip(at, at[1:])):
        n = max(on_ref[a:z1].sum(), 1)
        reach[a:z1] = 512 * rc[b].max(initial=0) * E / (k * n * n * used)
    err = np.abs(grad.double().cpu().numpy() - 512 * rg)
    bound = _grad_bound(512 * rg, p, reach, E, dtype)
    assert (err <= bound).all(), float((err / bound).max())
    assert (grad.cpu()[~torch.from_numpy(on_ref)] == 0).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T, E, k, dtype, how", [
    (50, 60, 4, torch.float32, {}), (9, 256, 8, torch.bfloat16, {"scale": 2.5}), (1, 8, 8, torch.float32, {}),
    (33, 64, 6, torch.float16, {"groups": 8, "topk_groups": 3, "bias": True}), (20, 2000, 10, torch.float32, {}),
])
def test_choice_gradient(T, E, k, dtype, how, scoring, renorm):
    """The gradient through the weights, against the formula in 64 bits."""
    router = _router()
    how = dict(how)
    scale = how.get("scale", 1.0)
    logits = _logits(T, E, dtype, E + k)
    leaf = logits.cuda().requires_grad_(True)
    bias = 0.1 * torch.randn((E,), generator=torch.Generator().manual_seed(1)).cuda() if how.pop("bias", 0) else None
    w, ids = router.choose_experts(leaf, k, scoring=scoring, renormalize=renorm, bias=bias, **how)
    gw = torch.randn((T, k), generator=torch.Generator().manual_seed(2))
    (grad,) = torch.autograd.grad(w, leaf, gw.cuda())
    z, at = logits.double().numpy(), ids.cpu().numpy().astype(np.int64)
    score, p = _score(z, scoring)
    rows = np.arange(T)[:, None]
    slope = 1 - score[rows, at] if scoring == "sigmoid" else np.ones((T, k))
    g = gw.double().numpy() * scale
    ref = np.zeros((T, E))
    own = score[rows, at]
    if renorm:
        own = own / own.sum(1, keepdims=True)
        ref[rows, at] = own * slope * (g - (g * own).sum(1, keepdims=True))
    elif scoring == "sigmoid":
        ref[rows, at] = g * own * slope
    else:
        full = np.zeros((T, E))
        full[rows, at] = g
        ref = p * (full - (full * p).sum(1, keepdims=True))
    near = p.copy()
    near[rows, at] = np.maximum(near[rows, at], own)
    err = np.abs(grad.double().cpu().numpy() - ref)
    bound = _grad_bound(ref, near, np.abs(g).max(), E, dtype)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("scoring, renorm", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                             ("sigmoid", False)])
def test_gradient_against_differences(scoring, renorm):
    """Central differences of the plain function around the same choice (64 bits, step 1e-5: errors of 1e-9)."""
    router = _router()
    T, E, k = 6, 12, 3
    logits = _logits(T, E, torch.float32, 5)
    gw, gl = torch.randn((T, k), generator=torch.Generator().manual_seed(3)), 0.7
    leaf = logits.cuda().requires_grad_(True)
    w, ids, loss, counts = router.choose_and_balance(leaf, k, scoring=scoring, renormalize=renorm)
    (grad,) = torch.autograd.grad([w, loss], leaf, [gw.cuda(), torch.tensor(gl, device="cuda")])
    at = ids.cpu().numpy().astype(np.int64)
    f = counts.cpu().numpy() * E / (k * T)

    def value(z):
        score, p = _score(z, scoring)
        own = score[np.arange(T)[:, None], at]
        if renorm:
            own = own / own.sum(1, keepdims=True)
        return (own * gw.double().numpy()).sum() + gl * (f * p.mean(0)).sum()

    z = logits.double().numpy()
    ref = np.zeros((T, E))
    for t in range(T):
        for e in range(E):
            step = np.zeros_like(z)
            step[t, e] = 1e-5
            ref[t, e] = (value(z + step) - value(z - step)) / 2e-5
    assert np.abs(grad.double().cpu().numpy() - ref).max() <= 1e-8 + 300 * U * 4


@pytest.mark.parametrize("T, E, k, cuts, padded, how", [
    (100, 64, 4, None, True, {}), (300, 256, 8, [3, 100, 100, 290], True, {"scoring": "sigmoid", "groups": 8,
                                                                          "topk_groups": 4, "bias": True}),
    (50, 60, 4, [0, 20, 45], False, {"renormalize": False, "scale": 2.0}), (5000, 16, 2, None, False, {}),
    (0, 16, 2, None, False, {}), (7, 1500, 3, [0, 7], False, {"bias": True}),
])
def test_one_pass_is_the_two_calls(T, E, k, cuts, padded, how):
    router = _router()
    how = dict(how)
    if how.pop("bias", False):
        how["bias"] = 0.1 * torch.randn((E,), generator=torch.Generator().manual_seed(1)).cuda()
    leaf = _logits(T, E, torch.float32, 11).cuda().requires_grad_(True)
    mask = torch.rand((T,), generator=torch.Generator().manual_seed(4)).cuda() < 0.8 if padded else None
    offs = None if cuts is None else torch.tensor(cuts, dtype=torch.int32, device="cuda")
    gw = torch.randn((T, k), generator=torch.Generator().manual_seed(2)).cuda()
    gl = torch.tensor(3.0, device="cuda")
    w, ids, loss, counts = router.choose_and_balance(leaf, k, mask=mask, seq_offsets=offs, **how)
    (grad,) = torch.autograd.grad([w, loss], leaf, [gw, gl])
    inside = mask
    if cuts is not None:
        t = torch.arange(T, device="cuda")
        inside = (t >= cuts[0]) & (t < cuts[-1]) & (mask if mask is not None else True)
    w2, ids2 = router.choose_experts(leaf, k, mask=inside, **how)
    loss2, counts2 = router.balance_loss(leaf, ids2, scoring=how.get("scoring", "softmax"), mask=mask, seq_offsets=offs)
    assert torch.equal(ids, ids2) and torch.equal(counts, counts2)
    assert torch.equal(w, w2) and torch.equal(loss, loss2)
    (g1,) = torch.autograd.grad(w2, leaf, gw)
    (g2,) = torch.autograd.grad(loss2, leaf, gl)
    # Both round sums of the magnitude of the largest G (see the gradient's bound above).
    per_seq = counts.double().reshape(-1, E)
    n = (per_seq.sum(1) / k).clamp(min=1)
    reach = (3.0 * per_seq.amax(1) * E / (k * n * n)).max().item() + how.get("scale", 1.0) * (
        gw.abs().max().item() if T else 0)
    err = (grad.double() - g1.double() - g2.double()).abs()
    assert (err <= 2 * (E + 128) * U * reach).all()


def test_repeatable():
    """The same call twice gives the same bits (no atomics on floating-point sums)."""
    router = _router()
    leaf = _logits(4099, 256, torch.bfloat16, 1).cuda().requires_grad_(True)
    one = router.choose_and_balance(leaf, 8)
    two = router.choose_and_balance(leaf, 8)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_streams_and_graphs():
    """A call on a side stream, and forward and backward captured and replayed on changed logits."""
    router = _router()
    T, E, k = 300, 128, 4
    fresh = [_logits(T, E, torch.float32, s).cuda() for s in range(4)]
    want = []
    for z in fresh:
        leaf = z.clone().requires_grad_(True)
        w, ids, loss, counts = router.choose_and_balance(leaf, k)
        want.append((w.detach(), ids, loss.detach(), counts, *torch.autograd.grad([w.sum() * 2 + loss], leaf)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w, ids = router.choose_experts(fresh[1], k)
    side.synchronize()
    assert torch.equal(ids, want[1][1]) and torch.equal(w, want[1][0])
    buf = fresh[0].clone().requires_grad_(True)
    gw, gl = torch.full((T, k), 2.0, device="cuda"), torch.ones((), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, ids, loss, counts = router.choose_and_balance(buf, k)
        (grad,) = torch.autograd.grad([w, loss], buf, [gw, gl])
    for i in (2, 0, 3, 1):
        with torch.no_grad():
            buf.copy_(fresh[i])
        graph.replay()
        torch.cuda.synchronize()
        got = (w, ids, loss, counts, grad)
        assert all(torch.equal(a, b) for a, b in zip(got[:4], want[i][:4]))
        assert torch.allclose(got[4], want[i][4], rtol=1e-5, atol=1e-7)
        (fresh[i] * 2).sum().item()  # the program's own work between the replays


def test_refusals():
    router = _router()
    z = torch.zeros((4, 16), device="cuda")
    bad = [
        lambda: router.choose_experts(z, 0),
        lambda: router.choose_experts(z, 17),
        lambda: router.choose_experts(z.double(), 2),
        lambda: router.choose_experts(z[0], 2),
        lambda: router.choose_experts(z, 2, scoring="tanh"),
        lambda: router.choose_experts(z, 2, groups=3),
        lambda: router.choose_experts(z, 5, groups=4, topk_groups=1),
        lambda: router.choose_experts(z, 2, groups=4, topk_groups=5),
        lambda: router.choose_experts(z, 2, bias=torch.zeros((15,), device="cuda")),
        lambda: router.choose_experts(z, 2, bias=torch.zeros((16,))),
        lambda: router.choose_experts(z, 2, mask=torch.ones((4,), device="cuda")),
        lambda: router.choose_experts(z, 2, mask=torch.ones((5,), dtype=torch.bool, device="cuda")),
        lambda: router.choose_experts(z, 2, scale=float("nan")),
        lambda: router.choose_experts(torch.zeros((4, 3000), device="cuda"), 2),
        lambda: router.choose_experts(torch.zeros((4, 2048), device="cuda"), 2, groups=2, topk_groups=1),
        lambda: router.balance_loss(z, torch.zeros((3, 2), dtype=torch.int32, device="cuda")),
        lambda: router.balance_loss(z, torch.zeros((4, 2), device="cuda")),
        lambda: router.balance_loss(z, torch.zeros((4, 2), dtype=torch.int32)),
        lambda: router.balance_loss(z, torch.zeros((4, 65), dtype=torch.int32, device="cuda")),
        lambda: router.balance_loss(z, torch.zeros((4, 2), dtype=torch.int32, device="cuda"),
                                    seq_offsets=torch.zeros((1,), dtype=torch.int32, device="cuda")),
        lambda: router.balance_loss(z, torch.zeros((4, 2), dtype=torch.int32, device="cuda"),
                                    seq_offsets=torch.zeros((3,), device="cuda")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_offsets_past_32_bits():
    """More than 2^31 logits: the last rows get what a call of their own gives."""
    router = _router()
    T, E, k, tail = (1 << 22) + 300, 520, 4, 300
    z = torch.zeros((T, E), dtype=torch.bfloat16, device="cuda")
    z[-tail:] = _logits(tail, E, torch.bfloat16, 1).cuda()
    assert z.numel() > 1 << 31
    own = z[-tail:].clone().requires_grad_(True)
    w, ids = router.choose_experts(z, k)
    w2, ids2 = router.choose_experts(own, k)
    assert torch.equal(ids[-tail:], ids2) and torch.equal(w[-tail:], w2.detach())
    small = z[:, :500]  # the form for up to 512 experts, rows apart
    w, ids = router.choose_experts(small, k)
    w2, ids2 = router.choose_experts(own.detach()[:, :500], k)
    assert torch.equal(ids[-tail:], ids2) and torch.equal(w[-tail:], w2)
    leaf = z.requires_grad_(True)
    offs = torch.tensor([T - tail, T], dtype=torch.int32, device="cuda")
    loss, counts = router.balance_loss(leaf, torch.zeros((T, 1), dtype=torch.int32, device="cuda"), seq_offsets=offs)
    (grad,) = torch.autograd.grad(loss, leaf)
    loss2, counts2 = router.balance_loss(own, torch.zeros((tail, 1), dtype=torch.int32, device="cuda"))
    (grad2,) = torch.autograd.grad(loss2, own)
    assert torch.equal(counts[0], counts2) and torch.equal(grad[-tail:], grad2) and grad[: T - tail].abs().max() == 0


def test_a_few_calls_at_once():
    """Calls on several streams at the same time, each with a workspace of its own."""
    router = _router()
    zs = [_logits(2000 + 100 * i, 64, torch.float32, i).cuda() for i in range(4)]
    want = [router.choose_and_balance(z, 4) for z in zs]
    streams = [torch.cuda.Stream() for _ in zs]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        got.clear()
        for z, st in zip(zs, streams):
            with torch.cuda.stream(st):
                got.append(router.choose_and_balance(z, 4))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_bias_and_groups_in_one_pass_of_many_experts():
    """The form of a wave per row in choose_and_balance: bias, groups, more than 512 experts or 16 choices."""
    router = _router()
    for E, k, how in ((600, 8, {}), (96, 20, {}), (1024, 4, {"bias": True, "groups": 4, "topk_groups": 2})):
        how = dict(how)
        if how.pop("bias", False):
            how["bias"] = 0.1 * torch.randn((E,), generator=torch.Generator().manual_seed(1)).cuda()
        leaf = _logits(150, E, torch.bfloat16, E).cuda().requires_grad_(True)
        w, ids, loss, counts = router.choose_and_balance(leaf, k, **how)
        w2, ids2 = router.choose_experts(leaf, k, **how)
        loss2, counts2 = router.balance_loss(leaf, ids2)
        assert torch.equal(w, w2) and torch.equal(ids, ids2) and torch.equal(loss, loss2)
        assert torch.equal(counts, counts2) and int(counts.sum()) == 150 * k


def test_offsets_of_64_bits():
    """int64 offsets that 32 bits do not hold are behind (or before) every row."""
    router = _router()
    z = _logits(50, 16, torch.float32, 11).cuda()
    near = torch.tensor([-1, 10, 50], device="cuda")
    far = torch.tensor([-(2**33) + 7, 10, 2**32 + 3], device="cuda")
    want = router.choose_and_balance(z, 2, seq_offsets=near)
    got = router.choose_and_balance(z, 2, seq_offsets=far)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert int(got[3].sum()) == 100


# The forms that no case above selects: 9 to 16 chosen of up to 512 experts (lists of 16), 257 to 512 experts (32 a lane of
# 16), and a wave per row with the sigmoid's loss and with more than 16 chosen.
FORMS = [
    # T, E, k, dtype, options
    (70, 60, 9, torch.bfloat16, {}),
    (70, 256, 16, torch.float32, {}),
    (65, 16, 16, torch.float16, {"renorm": False}),
    (40, 200, 12, torch.float32, {"scoring": "sigmoid", "scale": 2.5}),
    (33, 384, 10, torch.float32, {}),
    (33, 512, 8, torch.float16, {"renorm": False}),
    (129, 512, 10, torch.bfloat16, {}),
    (5, 300, 16, torch.float32, {"scoring": "sigmoid"}),
    (37, 511, 16, torch.bfloat16, {"scoring": "sigmoid", "renorm": False}),
    (1, 257, 1, torch.float32, {}),
    (30, 512, 17, torch.float32, {"scoring": "sigmoid"}),
    (21, 700, 33, torch.bfloat16, {}),
]
FORM_CALLS = [(*f, cuts) for f, cuts in zip(FORMS, [None, [0, 1, 30, 30, 70], None, [2, 40], [5, 5, 33], None,
                                                    [0, 100, 129], None, [0, 37], None, None, [3, 10, 21]])]


@pytest.mark.parametrize("T, E, k, dtype, how", FORMS)
def test_choice_of_every_form(T, E, k, dtype, how):
    """As test_choice, with ties, masked logits and padding among the rows."""
    logits = _logits(T, E, dtype, 3 * T + E)
    logits[T // 2] = torch.arange(E).remainder(3).to(dtype)
    logits[T // 3, ::2] = NEG
    logits[T // 4, 5:] = math.nan
    mask = np.random.default_rng(T).random(T) < 0.9
    how = {"renorm": True, **how}
    renorm = how.pop("renorm")
    w, ids = _router().choose_experts(logits.cuda(), k, renormalize=renorm, mask=torch.from_numpy(mask).cuda(), **how)
    z = logits.double().numpy()
    rw, rids = _choose_ref(z, k, renorm=renorm, mask=mask, **how)
    assert np.array_equal(ids.cpu().numpy(), rids)
    _check_weights(w, rw, z)


@pytest.mark.parametrize("T, E, k, dtype, how, cuts", FORM_CALLS)
def test_balance_of_every_form(T, E, k, dtype, how, cuts):
    """Choice, loss and counts in one pass, and the gradient through both, with masked logits and padding; then the
    loss of the same choice as a given one. Bounds as in test_balance and test_choice_gradient, added."""
    router = _router()
    how = {"renorm": True, "scoring": "softmax", "scale": 1.0, **how}
    renorm, scoring, scale = how["renorm"], how["scoring"], how["scale"]
    logits = _logits(T, E, dtype, 5 * T + E)
    logits[T // 3, ::2] = NEG
    logits[T // 4, 5:] = math.nan
    on = np.random.default_rng(E).random(T) < 0.85
    at = [0, T] if cuts is None else cuts
    live_rows = on.copy()
    live_rows[: at[0]] = False
    live_rows[at[-1] :] = False
    leaf = logits.cuda().requires_grad_(True)
    offs = None if cuts is None else torch.tensor(cuts, dtype=torch.int32, device="cuda")
    mask = torch.from_numpy(on).cuda()
    gw, gl = torch.randn((T, k), generator=torch.Generator().manual_seed(2)), 64.0
    w, ids, loss, counts = router.choose_and_balance(leaf, k, scoring=scoring, renormalize=renorm, scale=scale, mask=mask,
                                                     seq_offsets=offs)
    (grad,) = torch.autograd.grad([w, loss], leaf, [gw.cuda(), torch.tensor(gl, device="cuda")])
    z = logits.double().numpy()
    rw, rids = _choose_ref(z, k, scoring, renorm, scale=scale, mask=live_rows)
    assert np.array_equal(ids.cpu().numpy(), rids)
    _check_weights(w, rw, z)
    rl, rc, spread = _balance_ref(z, rids, k, scoring, live_rows, at)
    assert np.array_equal(counts.cpu().numpy().reshape(rc.shape), rc)
    assert abs(loss.item() - rl) <= rl * (T + 64 + _span(z).max()) * U
    loss2, counts2 = router.balance_loss(leaf, ids, scoring=scoring, mask=mask, seq_offsets=offs)
    assert torch.equal(loss, loss2) and torch.equal(counts, counts2)
    score, p = _score(z, scoring)
    rows, has = np.arange(T)[:, None], rids >= 0
    pick = np.where(has, rids, 0)
    own = np.where(has, score[rows, pick], 0.0)
    slope = 1 - score[rows, pick] if scoring == "sigmoid" else np.ones((T, k))
    g = np.where(has, gw.double().numpy() * scale, 0.0)
    if renorm:
        own = own / np.maximum(own.sum(1, keepdims=True), 1e-300)
        term = own * slope * (g - (g * own).sum(1, keepdims=True))
    else:
        term = g * own * slope
    ref, near, full = gl * spread, p.copy(), np.zeros((T, E))
    for t in range(T):
        for j in np.flatnonzero(has[t]):
            near[t, pick[t, j]] = max(near[t, pick[t, j]], own[t, j])
            if renorm or scoring == "sigmoid":
                ref[t, pick[t, j]] += term[t, j]
            else:
                full[t, pick[t, j]] += g[t, j]
    if not renorm and scoring == "softmax":
        ref = ref + p * (full - (full * p).sum(1, keepdims=True))
    used = max(sum(live_rows[a:b].any() for a, b in zip(at, at[1:])), 1)
    reach = np.full((T, 1), np.abs(g).max())
    for b, (a, z1) in enumerate(zip(at, at[1:])):
        n = max(live_rows[a:z1].sum(), 1)
        reach[a:z1] += gl * rc[b].max(initial=0) * E / (k * n * n * used)
    err = np.abs(grad.double().cpu().numpy() - ref)
    bound = _grad_bound(ref, near, reach, E, dtype)
    assert (err <= bound).all(), float((err / bound).max())
    assert (grad.cpu()[~torch.from_numpy(live_rows)] == 0).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("E, k, dtype", [(60, 4, torch.float32), (256, 16, torch.bfloat16), (12, 8, torch.float16),
                                         (600, 5, torch.float32), (40, 20, torch.float32)])
def test_gradient_of_repeated_ids(E, k, dtype, scoring, renorm):
    """The C entry point takes any choice: an expert that stands in a row several times gets the sum of its terms,
    through the weights and the loss together, in both forms of the rows."""
    from vllm_expert_pager import _native as nat

    T, scale, gl = 70, 2.5, 512.0
    g = np.random.default_rng(E + k)
    logits = _logits(T, E, dtype, E - k)
    ids = np.stack([g.permutation(E)[np.arange(k) % (E // 2 + 1)] for _ in range(T)])
    ids[:, k - 1] = ids[:, 0]  # the first and the last place of every row
    ids[3] = ids[3, 0]
    ids[4, 1:] = -1
    ids[5] = -1
    if k > 4:
        ids[6::5, 1:4] = ids[6::5, 2:3]
    ids = ids.astype(np.int32)
    gw = torch.randn((T, k), generator=torch.Generator().manual_seed(3))
    z = logits.double().numpy()
    on = np.ones(T, bool)
    _, counts, spread = _balance_ref(z, ids, k, scoring, on, [0, T])
    dev = [torch.from_numpy(ids).cuda(), gw.cuda(), torch.from_numpy(counts.astype(np.int32)).cuda(),
           torch.tensor([T, 1], dtype=torch.int32, device="cuda"), torch.tensor(gl, device="cuda")]
    leaf = logits.cuda()
    grad = torch.full((T, E), 7.0, dtype=dtype, device="cuda")
    _router()  # (the library's path)
    nat.call_on(leaf, "xp_router_backward", leaf.data_ptr(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype],
                T, E, E, k, 1 if scoring == "sigmoid" else 0, renorm, scale, None, None, 1, dev[0].data_ptr(), 4,
                dev[1].data_ptr(), dev[2].data_ptr(), dev[3].data_ptr(), dev[4].data_ptr(), grad.data_ptr())
    score, p = _score(z, scoring)
    rows = np.arange(T)[:, None]
    live = ids >= 0
    at = np.where(live, ids, 0)
    own = np.where(live, score[rows, at], 0.0)
    g64 = np.where(live, gw.double().numpy() * scale, 0.0)
    slope = 1 - score[rows, at] if scoring == "sigmoid" else np.ones((T, k))
    if renorm:
        own = own / np.maximum(own.sum(1, keepdims=True), 1e-300)
        term = own * slope * (g64 - (g64 * own).sum(1, keepdims=True))
    elif scoring == "sigmoid":
        term = g64 * own * slope
    ref, near, full = gl * spread, p.copy(), np.zeros((T, E))
    for t in range(T):
        for j in range(k):
            if not live[t, j]:
                continue
            near[t, at[t, j]] += own[t, j]
            if renorm or scoring == "sigmoid":
                ref[t, at[t, j]] += term[t, j]
            else:
                full[t, at[t, j]] += g64[t, j]
    if not renorm and scoring == "softmax":
        ref = ref + p * (full - (full * p).sum(1, keepdims=True))
    # _grad_bound with every place's terms in the reach: k of them add up where an expert repeats.
    reach = np.abs(g64).sum(1, keepdims=True) + gl * counts.max() * E / (k * T * T)
    err = np.abs(grad.double().cpu().numpy() - ref)
    bound = _grad_bound(ref, near, reach, E, dtype)
    assert (err <= bound).all(), float((err / bound).max())


def test_forward_mode_is_refused():
    """A dual tensor's tangent is never dropped in silence: the calls have no forward mode and say so."""
    router = _router()
    fw = torch.autograd.forward_ad
    z = _logits(6, 16, torch.float32, 2).cuda()
    want = router.choose_experts(z, 2)
    with fw.dual_level():
        dual = fw.make_dual(z, torch.ones_like(z))
        for call in (lambda: router.choose_experts(dual, 2), lambda: router.choose_and_balance(dual, 2),
                     lambda: router.balance_loss(dual, want[1])):
            with pytest.raises(NotImplementedError):
                call()
        got = router.choose_experts(z, 2)  # a tensor without a tangent
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
