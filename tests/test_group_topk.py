"""Grouped routing (inferno_moe_router_group_topk) against its definition in
64 bits, evaluated on the host by sorting.

Bars. Ids: equal, ties to the lower group and the lower id (64-bit values of
fp32 logits are equal only where the inputs are). Weights: a score is off by at
most 4 roundings of 2^-24 (the exponential's argument l - max rounds to 2^-24
of itself, which moves the score by |l - max| 2^-24 more), the sum of k or 256
scores adds at most k + 10 roundings, quotient and scale one each."""
import math

import numpy as np
import pytest
import torch

from inferno_amd import GROUP_MAX, GROUP_TOP2, SCORE_SIGMOID, SCORE_SOFTMAX, lib, ops


def _definition(logits, bias, k, score_fn, norm, scale, n_group, topk_group, rule):
    T, E = logits.shape
    l = logits.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        if score_fn == SCORE_SIGMOID:
            score = 1.0 / (1.0 + np.exp(-l))
            value = score
        else:
            top = l.max(1, keepdims=True)
            score = np.where(np.isneginf(top), 0.0, np.exp(l - np.where(np.isneginf(top), 0, top)))
            value = l
    value = value + (0.0 if bias is None else bias.astype(np.float64))
    size = E // n_group
    ids = np.empty((T, k), np.int64)
    for t in range(T):
        v = value[t].tolist()
        best = []
        for g in range(n_group):
            m = sorted(v[g * size:(g + 1) * size], reverse=True)
            best.append(m[0] if rule == GROUP_MAX or size == 1 else m[0] + m[1])
        kept = sorted(range(n_group), key=lambda g: (-best[g], g))[:topk_group]
        live = [e for e in range(E) if e // size in kept]
        ids[t] = sorted(live, key=lambda e: (-v[e], e))[:k]
    w = np.take_along_axis(score, ids, 1)
    total = w.sum(1, keepdims=True) if norm else score.sum(1, keepdims=True)
    if norm or score_fn == SCORE_SOFTMAX:
        w = np.where(total > 0, w / np.where(total > 0, total, 1.0), w)
    return ids, w * scale


def _check(logits, bias, k, score_fn, norm, scale, n_group, topk_group, rule):
    ids, w, tok = ops.router_group_topk(logits, bias, k, score_fn, norm, scale, n_group,
                                        topk_group, rule)
    T = logits.shape[0]
    l = logits.cpu().numpy()
    want, ww = _definition(l, None if bias is None else bias.cpu().numpy(), k, score_fn, norm,
                           scale, n_group, topk_group, rule)
    got = ids.view(T, k).cpu().numpy()
    assert np.array_equal(got, want), np.nonzero((got != want).any(1))[0][:5]
    finite = l[np.isfinite(l)]
    far = float(finite.max() - finite.min()) if score_fn == SCORE_SOFTMAX and finite.size else 0.0
    bar = (4 + 2 * far + k + 10 + 2) * 2.0 ** -24
    np.testing.assert_allclose(w.view(T, k).cpu().numpy(), ww, rtol=bar, atol=1e-38)
    assert torch.equal(tok.view(T, k).cpu(), torch.arange(T, dtype=torch.int32).repeat_interleave(k)
                       .view(T, k))
    return ids, w


SHAPES = [  # E, groups, kept groups, k
    (256, 8, 4, 8), (256, 8, 3, 16), (64, 4, 2, 6), (160, 8, 3, 6), (256, 1, 1, 8), (60, 5, 2, 4),
    (255, 15, 7, 9), (7, 7, 3, 3), (1, 1, 1, 1), (256, 256, 16, 16), (132, 3, 1, 16), (48, 16, 1, 3),
    (256, 2, 1, 10), (100, 50, 20, 16), (65, 13, 13, 1), (250, 125, 3, 5), (128, 8, 8, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("E,groups,kept,k", SHAPES)
@pytest.mark.parametrize("score_fn", [SCORE_SIGMOID, SCORE_SOFTMAX])
@pytest.mark.parametrize("rule", [GROUP_MAX, GROUP_TOP2])
def test_against_the_definition(cuda, E, groups, kept, k, score_fn, rule):
    g = torch.Generator().manual_seed(E * 7 + groups)
    for T, norm, with_bias in ((1, True, True), (5, False, True), (33, True, False),
                               (130, False, False)):
        logits = (2.0 * torch.randn(T, E, generator=g)).to(cuda)
        bias = (0.2 * torch.randn(E, generator=g)).to(cuda) if with_bias else None
        _check(logits, bias, k, score_fn, norm, 2.5, groups, kept, rule)


@pytest.mark.gpu
@pytest.mark.parametrize("score_fn", [SCORE_SIGMOID, SCORE_SOFTMAX])
@pytest.mark.parametrize("rule", [GROUP_MAX, GROUP_TOP2])
def test_ties_and_neighbours(cuda, score_fn, rule):
    # a few distinct values (ties of experts and of groups), then values one
    # fp32 step apart, whose sigmoids are equal in fp32 but not in 64 bits
    g = torch.Generator().manual_seed(3)
    few = torch.randint(0, 3, (40, 96), generator=g).float()
    _check(few.to(cuda), None, 7, score_fn, True, 1.0, 12, 5, rule)
    _check(torch.zeros(3, 96, device=cuda), None, 7, score_fn, True, 1.0, 12, 5, rule)
    near = torch.full((40, 96), 5.0) + torch.randint(0, 40, (40, 96), generator=g) * 2.0 ** -21
    _check(near.to(cuda), None, 7, score_fn, True, 1.0, 12, 5, rule)
    bias = torch.randint(0, 3, (96,), generator=g).float() * 0.25
    _check(near.to(cuda), bias.to(cuda), 7, score_fn, False, 1.0, 12, 5, rule)
    # sums of a value and a bias that round to one fp32 number
    wide = torch.randint(0, 9, (40, 96), generator=g) * 2.0 ** -30
    _check(wide.to(cuda), torch.ones(96, device=cuda), 7, score_fn, True, 1.0, 12, 5, rule)


@pytest.mark.gpu
@pytest.mark.parametrize("E", [24, 64, 70, 256])
@pytest.mark.parametrize("score_fn", [SCORE_SIGMOID, SCORE_SOFTMAX])
def test_few_and_many_near_ties(cuda, E, score_fn):
    # a handful of values next to each other among many, up to all of them
    g = torch.Generator().manual_seed(E)
    for many in (2, 9, 30, 64, 65, E):
        logits = torch.randn(50, E, generator=g) - 4.0
        for t in range(50):
            at = torch.randperm(E, generator=g)[:many]
            logits[t, at] = 3.0 + torch.randint(0, 3, (len(at),), generator=g) * 2.0 ** -22
        bias = torch.zeros(E)
        bias[::3] = 2.0 ** -24
        for b in (None, bias.to(cuda)):
            _check(logits.to(cuda), b, min(8, E), score_fn, True, 1.0, 1, 1, GROUP_MAX)
            _check(logits.to(cuda), b, 4, score_fn, False, 1.0, 2, 1, GROUP_TOP2)


@pytest.mark.gpu
def test_many_tokens(cuda):
    g = torch.Generator().manual_seed(6)
    _check(torch.randn(70001, 8, generator=g).to(cuda), None, 2, SCORE_SIGMOID, True, 1.0, 4, 2,
           GROUP_MAX)


@pytest.mark.gpu
@pytest.mark.parametrize("score_fn", [SCORE_SIGMOID, SCORE_SOFTMAX])
def test_closed_and_empty_rows(cuda, score_fn):
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(6, 32, generator=g)
    inf = float("inf")
    logits[0, 4:] = -inf      # fewer experts than are chosen
    logits[1] = -inf          # nothing
    logits[2, ::2] = -3e38    # the lowest finite values
    logits[3] = 200.0
    logits[4, 5] = 90.0       # the others' softmax scores vanish
    for rule in (GROUP_MAX, GROUP_TOP2):
        ids, w = _check(logits.to(cuda), None, 6, score_fn, True, 1.0, 8, 3, rule)
        assert w.isfinite().all() and not w.view(6, 6)[1].any()


@pytest.mark.gpu
def test_nan_rows_keep_valid_ids(cuda):
    logits = torch.randn(8, 64, generator=torch.Generator().manual_seed(5)).to(cuda)
    clean = ops.router_group_topk(logits, None, 5, 0, True, 1.0, 8, 2, GROUP_TOP2)
    bad = logits.clone()
    bad[3, 17] = float("nan")
    bad[5] = float("nan")
    ids, w, _ = ops.router_group_topk(bad, None, 5, 0, True, 1.0, 8, 2, GROUP_TOP2)
    ids, w = ids.view(8, 5), w.view(8, 5)
    assert ids[3, 0] == 17  # above +infinity
    assert ids[5].tolist() == [0, 1, 2, 3, 4]
    for t in range(8):
        assert len(set(ids[t].tolist())) == 5 and 0 <= int(ids[t].min()) <= int(ids[t].max()) < 64
        if t not in (3, 5):
            assert torch.equal(ids[t], clean[0].view(8, 5)[t]) and torch.equal(w[t], clean[1].view(8, 5)[t])


@pytest.mark.gpu
@pytest.mark.parametrize("score_fn", [SCORE_SIGMOID, SCORE_SOFTMAX])
def test_one_group_is_the_plain_top_k(cuda, score_fn):
    logits = torch.randn(50, 128, generator=torch.Generator().manual_seed(6)).to(cuda)
    a = ops.router_topk(logits, None, 8, score_fn, True, 1.5)
    b = ops.router_group_topk(logits, None, 8, score_fn, True, 1.5, 1, 1, GROUP_MAX)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    assert torch.allclose(a[1], b[1], rtol=32 * 2.0 ** -24, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("score_fn", [SCORE_SIGMOID, SCORE_SOFTMAX])
def test_groups_of_both_infinities(cuda, score_fn):
    # the two largest values of a group are +infinity and -infinity: their sum is
    # a NaN, which lies above every other group and does not open one more
    inf = float("inf")

    def route(v, k, n_group, kept):
        # as logits, or as biases of equal scores
        l, b = (v, None) if score_fn == SCORE_SOFTMAX else (torch.zeros_like(v), v[0].to(cuda))
        ids, _, _ = ops.router_group_topk(l.to(cuda), b, k, score_fn, True, 1.0, n_group, kept,
                                          GROUP_TOP2)
        return ids.view(-1, k).tolist()

    v = torch.tensor([[3.0, 2.0, inf, -inf, 2.9, 0.1, 0.5, 0.5]])
    assert route(v, 3, 4, 2) == [[2, 0, 1]]
    assert route(v, 2, 4, 1) == [[2, 3]]
    g = torch.Generator().manual_seed(11)
    for n_group in (16, 8):  # groups of 2, and of 4 with one value and -infinity
        for _ in range(20):
            v = torch.randn(1, 32, generator=g)
            of = v.view(n_group, -1)
            bad = int(torch.randint(0, n_group, (1,), generator=g))
            of[bad] = -inf
            of[bad, 0] = inf
            best = of.topk(2, 1).values.double().sum(1)
            best[bad] = inf
            size = 32 // n_group
            kept = torch.sort(best, descending=True, stable=True).indices[:3].tolist()
            live = [e for e in range(32) if e // size in kept]
            want = sorted(live, key=lambda e: (-v[0, e].item(), e))[:4]
            assert route(v, 4, n_group, 3) == [want]


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [20.0, 86.0, 95.0, 104.0, 1e4, 3e38])
def test_weights_far_below_the_closed_groups(cuda, gap):
    # the row's largest logit is in a closed group: the winners' softmax scores
    # vanish in fp32, their normalised weights do not. Sums of two in 32 bits
    # decide the second half's groups, ties send the first half's to 64 bits.
    # Bar: two exponentials whose arguments are at most 3 (rounded to 3 2^-24,
    # two roundings more), four additions, a quotient and the scale
    g = torch.Generator().manual_seed(2)
    l = torch.rand(20, 16, generator=g) * 3.0
    l[:10, 5] = l[:10, 4]
    l[:10, 8:10] = l[:10, 4:6]
    l[:, 2], l[:, 3] = gap, -gap
    ids, w, _ = ops.router_group_topk(l.to(cuda), None, 4, SCORE_SOFTMAX, True, 2.5, 8, 4,
                                      GROUP_TOP2)
    want, _ = _definition(l.numpy(), None, 4, SCORE_SOFTMAX, False, 2.5, 8, 4, GROUP_TOP2)
    assert np.array_equal(ids.view(20, 4).cpu().numpy(), want) and (want // 2 != 1).all()
    e = torch.exp(l.double().gather(1, torch.from_numpy(want)))
    e = 2.5 * e / e.sum(1, keepdim=True)
    assert ((w.view(20, 4).cpu().double() - e).abs() <= (2 * (3 + 2) + 4 + 2) * 2.0 ** -24 * e).all()


@pytest.mark.gpu
@pytest.mark.parametrize("far", [-20.0, -60.0, -86.0, -95.0, -104.0, -1e4])
@pytest.mark.parametrize("ties", [False, True])
def test_normalised_weights_of_vanishing_sigmoids(cuda, far, ties):
    # the winners' scores vanish in fp32 (biases decide), their ratios do not. Bar:
    # exponentials of arguments of at most 3 and far's rounding, which is the input's;
    # four additions, a quotient and the scale; above -17 the sigmoid's own roundings
    g = torch.Generator().manual_seed(9)
    l = far + 3.0 * torch.rand(20, 16, generator=g)
    bias = torch.rand(16, generator=g)
    if ties:  # whole rows in 64 bits
        bias[:] = 0.25
        l[:, 4:8] = l[:, 0:4]
    ids, w, _ = ops.router_group_topk(l.to(cuda), bias.to(cuda), 4, SCORE_SIGMOID, True, 2.5, 4, 2,
                                      GROUP_TOP2)
    ids = ids.view(20, 4).cpu().long()
    assert all(len(set(r)) == 4 for r in ids.tolist())
    won = l.double().gather(1, ids)
    e = torch.exp(won - won.amax(1, keepdim=True)) / (1.0 + torch.exp(won))
    e = 2.5 * e / e.sum(1, keepdim=True)
    bar = (2 * (3 + 2) + 4 + 2 + 2 * (abs(far) if far > -56.0 else 0)) * 2.0 ** -24
    assert ((w.view(20, 4).cpu().double() - e).abs() <= bar * e).all()


@pytest.mark.gpu
def test_weights_of_closed_and_infinite_logits(cuda):
    # winners of -infinity alone, below a finite or an infinite closed logit
    inf = float("inf")
    l = torch.full((3, 8), -inf)
    l[0, 0], l[1, 0], l[2, 0] = 5.0, inf, 5.0
    l[2, 6] = 1.0
    bias = torch.zeros(8)
    bias[0] = -100.0
    ids, w, _ = ops.router_group_topk(l[:, 2:].contiguous().to(cuda), None, 2, SCORE_SOFTMAX, True,
                                      1.0, 3, 1, GROUP_MAX)
    assert not w.view(3, 2)[:2].any() and w.view(3, 2)[2].tolist() == [1.0, 0.0]
    ids, w, _ = ops.router_group_topk(l.to(cuda), bias.to(cuda), 1, SCORE_SOFTMAX, True, 1.0, 4, 1,
                                      GROUP_MAX)
    assert ids.tolist()[2] == 6 and w.tolist()[2] == 1.0


def _check_ids(logits, bias, k, score_fn, n_group, topk_group, rule):
    ids, _, _ = ops.router_group_topk(logits, bias, k, score_fn, True, 1.0, n_group, topk_group,
                                      rule)
    want, _ = _definition(logits.cpu().numpy(), bias.cpu().numpy(), k, score_fn, True, 1.0, n_group,
                          topk_group, rule)
    got = ids.view(-1, k).cpu().numpy()
    assert np.array_equal(got, want), np.nonzero((got != want).any(1))[0][:5]
    return got


@pytest.mark.gpu
def test_sums_of_two_that_nearly_cancel(cuda):
    # logit + bias rounds relative to itself, which may be far more than the sum of
    # a group's two largest values; the order has to be that of 64 bits
    for l, b, best in (([1.7361599206924438, -1.7361599206924438, 17.175823211669922,
                         -17.175823211669922], [0.07883994281292, -0.07883810251951,
                                                -0.17062471807003, 0.17062482237816], 0),
                       ([1000.0, -1000.0, 1.0, -0.99999], [1.5e-5, 0.0, 0.0, 0.0], 0)):
        l, b = torch.tensor([l]).to(cuda), torch.tensor(b).to(cuda)
        assert _check_ids(l, b, 2, SCORE_SOFTMAX, 2, 1, GROUP_TOP2).min() // 2 == best


@pytest.mark.gpu
@pytest.mark.parametrize("score_fn", [SCORE_SIGMOID, SCORE_SOFTMAX])
@pytest.mark.parametrize("size", [2, 3, 8])
@pytest.mark.parametrize("far", [1.0, 60.0, 1e4, 1e30])
def test_many_sums_of_two_that_nearly_cancel(cuda, score_fn, size, far):
    # groups of a value, nearly its negative, and for larger groups values far
    # below both; their sums lie within a few roundings of each other
    g = torch.Generator().manual_seed(int(size * 1000 + min(far, 1e6)))
    T, groups = 60, 12
    E = groups * size
    big = far * (0.05 + torch.rand(groups, generator=g))
    l = torch.randn(T, groups, size, generator=g)
    bias = torch.full((groups, size), -4.0 * far)
    if score_fn == SCORE_SIGMOID:  # the magnitudes are in the biases
        bias[:, 0], bias[:, 1] = big, -big
        bias[:, 1] -= 2.0 ** -24 * torch.randn(groups, generator=g) * far
    else:
        bias[:, 0] = 2.0 ** -20 * torch.randn(groups, generator=g) * far
        bias[:, 1] = 2.0 ** -20 * torch.randn(groups, generator=g) * far
        scale = big * (0.5 + torch.rand(T, groups, generator=g))
        l[:, :, 0], l[:, :, 1] = scale, -scale
    l, bias = l.view(T, E), bias.view(E)
    for kept in (1, 4, 11):
        _check_ids(l.to(cuda), bias.to(cuda), min(kept * size, 5), score_fn, groups, kept,
                   GROUP_TOP2)


@pytest.mark.gpu
def test_group_values_behind_the_range(cuda):
    # values and sums of two that leave fp32's range, next to true infinities
    inf, big = float("inf"), 3e38
    l = torch.tensor([[big, big, big, 2.5e38, -big, big, 1.0, -inf],
                      [-big, -big, -inf, -inf, -big, -2e38, -big, big],
                      [big, -big, 2e38, -big, -inf, big, -inf, 2.9e38],
                      [-inf, -inf, -inf, -inf, 1.0, -inf, 2.0, -inf]])
    for b in (torch.zeros(8), torch.tensor([big, 2e38, big, big, -big, -big, 0.0, 0.0]),
              torch.tensor([-big, -big, big, -big, 1e38, -big, 1e38, 0.0])):
        for kept in (1, 2, 3):
            for rule in (GROUP_MAX, GROUP_TOP2):
                _check_ids(l.to(cuda), b.to(cuda), 2, SCORE_SOFTMAX, 4, kept, rule)


def test_refusals():
    logits = torch.zeros(2, 32)
    ok = dict(bias=None, k=4, score_fn=0, norm=True, scale=1.0, n_group=4, topk_group=2,
              group_score=0)
    with pytest.raises(ValueError, match="GPU tensors"):
        ops.router_group_topk(logits, **ok)
    with pytest.raises(ValueError, match="bias"):
        ops.router_group_topk(logits, **dict(ok, bias=torch.zeros(31)))
    with pytest.raises(ValueError, match="logits"):
        ops.router_group_topk(logits.bfloat16(), **ok)
    with pytest.raises(ValueError, match="contiguous"):
        ops.router_group_topk(torch.zeros(32, 2).T, **ok)
    with pytest.raises(ValueError, match="negative"):
        ops.router_group_topk(logits, **dict(ok, k=-1))
    f = lib().inferno_moe_router_group_topk

    def status(T=1, E=32, k=4, score=0, scale=1.0, groups=4, kept=2, rule=0, p=16):
        return f(None, p, None, T, E, k, score, 1, scale, groups, kept, rule, 16, 16, None)

    for bad in (dict(E=0), dict(E=257, groups=1), dict(groups=0), dict(groups=5), dict(kept=0),
                dict(kept=5), dict(k=0), dict(k=17), dict(score=2), dict(rule=2),
                dict(scale=math.inf), dict(p=None), dict(T=1 << 26), dict(k=9, kept=1)):
        assert status(**bad) == -1, bad
    assert b"exceeds the 8 experts" in lib().inferno_last_error()
    assert status(T=0, p=None) == 0


def test_refuses_more_tokens_than_a_launch_takes():
    # four tokens a workgroup of 256 threads: 2^24 workgroups are 2^32 threads
    f = lib().inferno_moe_router_group_topk
    for T in ((1 << 26) - 3, (1 << 26) - 1, 1 << 40):
        assert f(None, 16, None, T, 1, 1, 0, 1, 1.0, 1, 1, 0, 16, 16, None) == -1, T
        assert b"too many tokens" in lib().inferno_last_error()
