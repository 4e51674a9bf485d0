"""The router where logits are masked, no numbers or far apart: against 64-bit restatements written from the definition."""

from __future__ import annotations

import math

import pytest
import torch
from test_experts import BF16, DEV, F16, F32, device_word, normal  # noqa: F401
from test_router import INF, assert_weights, scores_of, weights_of

from blackhole_b200 import router


# ------------------------------------------------------------------ masked experts in groups
def masked_choice(logits, k, scoring, bias, groups, topk_groups, group_top):
    """ids [T, k] from the definition: a group's value is the sum of its group_top largest s + b, where a masked expert's s
    is 0; in the open groups masked experts come after all others.  And the smallest distance a decision rested on."""
    T, E = logits.shape
    per, scores = E // groups, scores_of(logits, scoring)
    biased = scores + (0.0 if bias is None else bias.double())
    ids, gap = [], INF
    for t in range(T):
        values = [sum(sorted(biased[t, g * per:(g + 1) * per].tolist())[-group_top:]) for g in range(groups)]
        order = sorted(range(groups), key=lambda g: (-values[g], g))
        rank = [(float(logits[t, e]) == -INF, -float(logits[t, e] if bias is None else biased[t, e]), e)
                for g in order[:topk_groups] for e in range(g * per, (g + 1) * per)]
        rank = sorted((m, 0.0 if m else v, e) for m, v, e in rank)
        steps = [values[order[topk_groups - 1]] - values[order[topk_groups]]] if topk_groups < groups else []
        if bias is not None:
            steps += [b[1] - a[1] for a, b in zip(rank[:k], rank[1:k + 1]) if not b[0]]
        gap = min([gap] + [s for s in steps if s])
        ids.append([e for _, _, e in rank[:k]])
    return torch.tensor(ids), gap


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [None, "zeros", "some", "large"])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("E,k,groups,open_groups", [(4, 1, 2, 1), (24, 3, 2, 1), (40, 4, 4, 2), (96, 8, 8, 4), (256, 8, 8, 4), (500, 16, 20, 7)])
def test_masked_experts_in_groups(E, k, groups, open_groups, group_top, bias, scoring):
    """Seven of ten experts masked, groups with one expert left, groups with none, and rows with next to none."""
    g = torch.Generator().manual_seed(E + k)
    logits = normal((40, E), F32, E, 1.5)
    logits[torch.rand(40, E, generator=g) < 0.7] = -INF
    logits[1:6, :E // groups] = -INF
    logits[2] = -INF
    logits[3] = -INF
    logits[3, E - 1] = 5.0
    logits[4, E // groups:] = -INF
    b = None if bias is None else torch.zeros(E) if bias == "zeros" else normal((E,), F32, 3, 0.1 if bias == "some" else 3.0)
    how = dict(scoring=scoring, groups=groups, topk_groups=open_groups, group_top=group_top)
    want, gap = masked_choice(logits, k, bias=b, **how)
    assert gap > 1e-13
    for renormalize in (True, False):
        weights, ids = router.route(logits.to(DEV), k, bias=None if b is None else b.to(DEV), renormalize=renormalize, **how)
        assert torch.equal(ids.cpu().long(), want)
        assert_weights(weights, weights_of(logits, want, scoring, renormalize), logits[:1], 1.0)
    if bias == "zeros":   # a bias of nothing changes nothing
        assert torch.equal(router.route(logits.to(DEV), k, **how)[1].cpu().long()[3], want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_experts_in_groups_nearer_than_f32_tells(scoring):
    """Groups' values that only 64 bits tell apart, with masked experts in every group, and more equal ones than lanes."""
    E, k, how = 64, 6, dict(scoring=scoring, groups=8, topk_groups=3, group_top=2)
    logits = normal((1, E), F32, 5, 1.0) + normal((200, E), F32, 6, 1e-7)
    logits[:, ::3] = -INF
    logits[7, 1::8], logits[7, 2::8] = -INF, -INF
    bias = (0.9 - scores_of(logits[:1], scoring)[0]).float()
    want, gap = masked_choice(logits, k, bias=bias, **how)
    assert gap > 2e-15
    assert torch.equal(router.route(logits.to(DEV), k, bias=bias.to(DEV), **how)[1].cpu().long(), want)
    flat = torch.zeros(3, 512)
    flat[0, ::2], flat[1, 5:], flat[2, 40:90] = -INF, -INF, -INF
    for bias in (None, torch.zeros(512), torch.full((512,), 0.25)):
        want, _ = masked_choice(flat, 20, scoring, bias, 4, 2, 2)
        got = router.route(flat.to(DEV), 20, scoring=scoring, bias=None if bias is None else bias.to(DEV), groups=4, topk_groups=2)[1]
        assert torch.equal(got.cpu().long(), want)


# ------------------------------------------------------------------ logits that are no numbers
@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("E,groups", [(20, 1), (20, 4), (96, 1), (256, 8), (1000, 10)])
def test_one_logit_that_is_no_number(E, groups, renormalize, scoring):
    """A row with a NaN, or under a softmax with +inf, whose scores are not defined: weights are all NaN, wherever it stands,
    ids valid and distinct; other rows are not touched."""
    logits = normal((12, E), F32, 12).index_fill(0, torch.tensor([3]), 2.0)
    bad = {1: (E - 1, math.nan), 3: (E // 2, math.nan), 4: (0, math.nan), 8: (E - 2, INF), 9: (1, INF)}
    clean = logits.clone()
    for t, (e, v) in bad.items():
        logits[t, e] = v
    logits[4, 1:5] = -INF
    rows = torch.tensor([t for t, (_, v) in bad.items() if v != INF or scoring == "softmax"])
    rest = torch.tensor([t for t in range(12) if t not in bad])
    for bias in (None, torch.zeros(E, device=DEV), normal((E,), F32, 13, 0.1).to(DEV)):
        how = dict(scoring=scoring, bias=bias, groups=groups, topk_groups=min(2, groups), renormalize=renormalize)
        weights, ids = router.route(logits.to(DEV), 5, **how)
        assert weights.cpu()[rows].isnan().all() and 0 <= int(ids.min()) and int(ids.max()) < E
        assert all(len(set(row)) == 5 for row in ids.tolist())
        want, want_ids = router.route(clean.to(DEV), 5, **how)
        assert torch.equal(weights.cpu()[rest], want.cpu()[rest]) and torch.equal(ids.cpu()[rest], want_ids.cpu()[rest])
        if scoring == "sigmoid":   # +inf is a score of 1
            top = (ids.cpu()[8] == E - 2).nonzero()
            assert weights[8:10].isfinite().all() and (bias is not None or groups > 1 or top.tolist() == [[0]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("E", [20, 96, 256, 1000])
def test_gradient_of_a_row_with_one_logit_that_is_no_number(E, renormalize, dtype):
    """Softmax: the whole row's gradient is NaN, as the formula's, also where the NaN (or +inf) was not chosen."""
    logits = normal((9, E), dtype, 14)
    ids = torch.arange(3).expand(9, 3) + torch.arange(9)[:, None]
    d = normal((9, 3), F32, 15).to(DEV)
    want = router.route_backward(d, logits.to(DEV), ids.to(DEV), renormalize=renormalize)
    logits[2, E - 1], logits[5, 18], logits[6, 6] = math.nan, INF, math.nan
    got = router.route_backward(d, logits.to(DEV), ids.to(DEV), renormalize=renormalize)
    bad = torch.tensor([2, 5, 6])
    rest = torch.tensor([0, 1, 3, 4, 7, 8])
    assert got.cpu()[bad].isnan().all() and torch.equal(got.cpu()[rest], want.cpu()[rest])


# ------------------------------------------------------------------ gradients next to a score of 1
def gradient_and_mass(logits, ids, d, scale):
    """The plain softmax's gradient in 64 bits without a difference of near values, dl_e = s_e sum_i s_i (a_e - a_i) with a
    the sum of an expert's places (0 where not chosen), and the sum of the magnitudes of its terms."""
    s = torch.softmax(logits.double(), 1)
    a = torch.zeros_like(s).scatter_add_(1, ids, d.double() * scale)
    away = s[:, None, :] * (a[:, :, None] - a[:, None, :])
    return s * away.sum(2), s * away.abs().sum(2)


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [0, 5, 10, 15, 17, 20, 30, 60])
@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (8, 1), (8, 2), (33, 4), (96, 8), (256, 1), (1000, 32)])
def test_softmax_gradient_next_to_a_score_of_one(E, k, gap):
    """One expert ahead of all others, among the chosen ones or not, and ids that stand twice.  A term s_e s_i (a_e - a_i) is
    off by its two scores (exponents rounded, |l - m| 2^-24; exponentials and sums, E / 32 + 24 units) and its sum of k + E / 32
    + 5 additions; twice over."""
    T = 9
    logits, d = normal((T, E), F32, E + k), normal((T, k), F32, 21)
    ids = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(t))[:k] for t in range(T)])
    logits.scatter_add_(1, ids[:, :1], torch.full((T, 1), float(gap)))
    ids[3] = ids[3, 0]                 # one expert in every place
    ids[4] = ids[4].flip(0)
    if k > 1:
        ids[5, 0] = ids[5, 1]          # the one ahead is not chosen
        ids[6, 1] = ids[6, 0]
    want, mass = gradient_and_mass(logits, ids, d, 1.5)
    got = router.route_backward(d.to(DEV), logits.to(DEV), ids.to(DEV), renormalize=False, scale=1.5).double().cpu()
    span = float(logits.max() - logits.min())
    bound = 2 * (2 * (span + E / 32 + 24) + k + E / 32 + 5) * 2.0 ** -24 * mass + 2.0 ** -120
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / mass.clamp(min=1e-300)).max())
    ref = logits.double().requires_grad_()
    (torch.softmax(ref, 1).gather(1, ids) * 1.5 * d.double()).sum().backward()
    assert ((want - ref.grad).abs() <= 2.0 ** -48 * d.double().abs().sum(1, keepdim=True)).all()


# ------------------------------------------------------------------ weights of scores far below others
@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups", [(20, 7, 1), (96, 8, 8), (500, 16, 20), (1000, 32, 1)])
def test_weights_of_scores_far_below_others(E, k, groups, scoring):
    """Experts that a bias picks although their scores are f32's smallest, and scores that are all small: renormalised weights
    are as near as any others (what is below 2^-126 may be off by that)."""
    logits = normal((60, E), F32, E, 30.0)
    if scoring == "sigmoid":
        logits = -logits.abs() - torch.arange(60)[:, None]
    bias = normal((E,), F32, 3, 3.0)
    how = dict(scoring=scoring, groups=groups, topk_groups=max(1, groups // 2), group_top=1)
    for b in (None, bias):
        want, gap = masked_choice(logits, k, bias=b, **how)
        assert b is None or gap > 1e-13   # without: decisions between numbers of any size, as near as their own size
        weights, ids = router.route(logits.to(DEV), k, bias=None if b is None else b.to(DEV), **how)
        assert torch.equal(ids.cpu().long(), want)
        assert_weights(weights, weights_of(logits, want, scoring), logits, 1.0)
