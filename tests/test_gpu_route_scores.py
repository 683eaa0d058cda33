"""oco_route_scores against the rule in 64 bits: ids exactly, weights within
f32 roundings of the score (1), of the sum of at most 32 of them (7), of the
quotient and of the product (4)."""
import numpy as np
import pytest

from _ops import CODE, U, dev, stored
from _util import Guarded, say

pytestmark = pytest.mark.gpu


def reference(z, bias, k, sigmoid, groups, kept, top2, renormalize, scale):
    """(ids, weights) by the written rule, one token at a time."""
    tokens, experts = z.shape
    ids, weights = np.zeros((tokens, k), np.int64), np.zeros((tokens, k))
    for t in range(tokens):
        row = z[t].copy()
        bad = np.isnan(row) | (row == np.inf)
        row[bad] = -np.inf
        open_ = row > -np.inf
        if sigmoid:
            with np.errstate(over="ignore"):
                s = np.where(open_, 1 / (1 + np.exp(-np.where(open_, row, 0))), 0.0)
        else:
            e = np.where(open_, np.exp(np.where(open_, row, 0) - (row[open_].max() if open_.any() else 0)), 0.0)
            s = e / e.sum() if open_.any() else e
        c = s + (0 if bias is None else bias.astype(np.float64))
        if bias is None and not (groups > 1 and top2):
            c = row.copy()  # the order of the logits
        c = np.where(open_ & ~np.isnan(c), c, -np.inf)
        allowed = np.ones(experts, bool)
        if groups > 1 and kept < groups:
            size, rank = experts // groups, []
            for g in range(groups):
                part = np.sort(c[g * size:(g + 1) * size])[::-1]
                rank.append(part[0] + (part[1] if top2 and size > 1 and part[1] > -np.inf else 0.0))
            best = sorted(range(groups), key=lambda g: (-rank[g], g))[:kept]
            allowed = np.isin(np.arange(experts) // size, best)
        order = sorted(np.nonzero(allowed)[0], key=lambda e: (-c[e], e))[:k]
        ids[t] = order
        w = s[order]
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else w * 0
        weights[t] = np.nan if bad.any() else scale * w
    return ids, weights


def check(lib, z, k, sigmoid, groups=1, kept=1, top2=False, bias=None, renormalize=True, scale=2.5, dtype="f32"):
    tokens, experts = z.shape
    say("route_scores", tokens, experts, k, sigmoid, groups, kept, top2, bias is not None, renormalize, dtype)
    zb, z = stored(z, dtype)
    p = lib.Routing(experts=experts, k=k, score=int(sigmoid), groups=groups, groups_kept=kept, group_rank=int(top2),
                    renormalize=int(renormalize), scale=scale)
    ids, weights = Guarded(lib, tokens * k * 4), Guarded(lib, tokens * k * 4)
    lib.route_scores(dev(lib, zb), tokens, p, ids.ptr, weights.ptr, CODE[dtype], None if bias is None else dev(lib, bias))
    lib.synchronize()
    want_ids, want = reference(z, bias, k, sigmoid, groups, kept, top2, renormalize, scale)
    np.testing.assert_array_equal(ids.read(np.uint32).reshape(tokens, k), want_ids)
    got = weights.read(np.float32).reshape(tokens, k).astype(np.float64)
    np.testing.assert_allclose(got, want, rtol=12 * U, atol=2.0 ** -140)
    return want_ids, got


@pytest.mark.parametrize("experts,k", [(1, 1), (5, 5), (63, 8), (64, 8), (65, 32), (128, 8), (129, 3), (256, 8), (257, 9), (512, 8), (1000, 32), (1024, 16)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_experts_per_lane(lib, experts, k, sigmoid):
    rng = np.random.default_rng(experts)
    z = rng.normal(size=(9, experts)) * 2
    z[3:6] = rng.integers(-2, 3, (3, experts))  # ties within and across lanes
    check(lib, z, k, sigmoid)
    check(lib, z, k, sigmoid, bias=(0.1 * rng.normal(size=experts)).astype(np.float32), renormalize=False)


@pytest.mark.parametrize("experts,groups,kept,k", [(256, 8, 4, 8), (256, 8, 1, 8), (160, 8, 3, 6), (96, 4, 2, 8), (64, 64, 8, 8), (30, 10, 3, 5), (33, 3, 2, 7),
                                                   (1024, 64, 4, 32), (24, 8, 8, 4), (990, 11, 5, 20)])
@pytest.mark.parametrize("top2", [False, True])
def test_groups(lib, experts, groups, kept, k, top2):
    rng = np.random.default_rng(experts + groups)
    z = rng.normal(size=(11, experts))
    z[2:5] = rng.integers(-1, 2, (3, experts))  # groups of equal rank
    z[5] = 0
    bias = (0.05 * rng.normal(size=experts)).astype(np.float32)
    for sigmoid in (False, True):
        check(lib, z, k, sigmoid, groups, kept, top2, bias=bias)
        check(lib, z, k, sigmoid, groups, kept, top2)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens", [1, 2, 4, 5, 130])
def test_types_and_tokens(lib, dtype, tokens):
    rng = np.random.default_rng(tokens)
    z = rng.normal(size=(tokens, 128))
    check(lib, z, 8, True, 8, 4, True, bias=(0.05 * rng.normal(size=128)).astype(np.float32), dtype=dtype)
    check(lib, z, 8, False, dtype=dtype)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_masked_experts(lib, sigmoid, with_bias):
    """-Inf logits: never before an available expert, whatever the bias; a
    token with fewer than k, with one and with none left; groups likewise."""
    rng = np.random.default_rng(5)
    experts, k = 96, 6
    z = rng.normal(size=(6, experts))
    z[0, ::2] = -np.inf
    z[1, 3:] = -np.inf
    z[2, :95] = -np.inf
    z[3] = -np.inf
    z[4, :12] = -np.inf  # a whole group
    z[4, 13:24] = -np.inf  # all but one of a group
    bias = np.full(experts, 0.5, np.float32) if with_bias else None
    if with_bias:
        bias[1], bias[30] = 100.0, -100.0
    check(lib, z, k, sigmoid, bias=bias)
    for top2 in (False, True):
        ids, w = check(lib, z, k, sigmoid, 8, 3, top2, bias=bias)
        assert not w[3].any()
    check(lib, z, k, sigmoid, bias=bias, renormalize=False)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_logits_that_are_not_numbers(lib, bad):
    rng = np.random.default_rng(6)
    z = rng.normal(size=(5, 70))
    z[1, 69] = bad
    z[3, 0] = bad
    for sigmoid in (False, True):
        check(lib, z, 8, sigmoid)
        check(lib, z, 8, sigmoid, 7, 3, True, bias=np.zeros(70, np.float32))


def test_a_bias_that_is_not_a_number_ranks_last(lib):
    rng = np.random.default_rng(7)
    bias = (0.1 * rng.normal(size=40)).astype(np.float32)
    bias[[3, 20]] = np.nan
    bias[7] = np.inf
    bias[8] = -np.inf
    check(lib, rng.normal(size=(4, 40)), 8, True, bias=bias)


def test_extreme_logits(lib):
    """Scores that underflow or saturate keep the logits' order without a bias."""
    z = np.array([[500.0, 400, 300, -300, -500, 0, 1, 2], [-1000, -999, -1001, -2000, -1500, -1200, -998, -3000]])
    for sigmoid in (False, True):
        check(lib, z, 4, sigmoid)
    check(lib, z[:1], 8, True, renormalize=False)


def test_scores_under_the_range_of_f32_keep_their_ratios(lib):
    rng = np.random.default_rng(10)
    z = rng.normal(size=(5, 48)) - 120.0
    check(lib, z, 8, True)  # sigmoids of 1e-52
    bias = np.zeros(48, np.float32)
    bias[8:16] = 1.0
    z[:, 0] = 0.0  # the softmax is all on an expert that the bias leaves out
    check(lib, z, 8, False, bias=bias)
    check(lib, z, 8, True, 6, 1, True, bias=bias)
    check(lib, z, 8, False, bias=bias, renormalize=False)


def test_close_scores_are_told_apart(lib):
    """Sums of score and bias that differ by less than an f32 step."""
    z = np.zeros((1, 64))
    bias = np.zeros(64, np.float32)
    bias[40] = np.float32(2.0 ** -40)
    bias[50] = np.float32(2.0 ** -41)
    ids, _ = check(lib, z, 3, True, bias=bias)
    assert list(ids[0]) == [40, 50, 0]


def test_matches_the_library_s_selection(lib):
    """Softmax without bias, groups or scale, renormalised: oco_route_select's ids, and its probabilities up to
    their bf16 roundings (of the logits, 2^-8 of at most 4 each, and of the result)."""
    rng = np.random.default_rng(9)
    z = np.clip(rng.normal(size=(40, 128)), -4, 4).astype(np.float32)
    ids, w = check(lib, z, 8, False, scale=1.0)
    ids2, probs = lib.DeviceBuffer(40 * 8 * 4), lib.DeviceBuffer(40 * 8 * 4)
    lib.route_select(dev(lib, z), 40, 128, 8, ids2, probs)
    lib.synchronize()
    np.testing.assert_array_equal(ids2.download(np.uint32).reshape(40, 8), ids)
    np.testing.assert_allclose(probs.download(np.float32).reshape(40, 8), w, rtol=2 * 4 * 2.0 ** -8 + 2.0 ** -8 + 2.0 ** -9)


def by_logits(z, k, sigmoid, groups, kept):
    """Without a bias: groups by the sum of their two largest scores, experts by their logits."""
    ids, size = [], z.shape[1] // groups
    for row in z:
        s = 1 / (1 + np.exp(-row)) if sigmoid else np.exp(row - row.max()) / np.exp(row - row.max()).sum()
        two = -np.sort(-s.reshape(groups, size), 1)[:, :2].sum(1)
        best = sorted(range(groups), key=lambda g: (-two[g], g))[:kept]
        ids.append(sorted((e for e in range(len(row)) if e // size in best), key=lambda e: (-row[e], e))[:k])
    return np.array(ids)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("experts,groups,kept,k", [(64, 4, 2, 8), (256, 8, 4, 8), (30, 5, 2, 6), (1024, 16, 3, 20)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_without_a_bias_the_order_is_that_of_the_logits(lib, sigmoid, experts, groups, kept, k, dtype):
    """Logits whose 64-bit scores coincide (sigmoids from 37 on, what lies 700
    and more under a softmax's largest), in groups ranked by their two best."""
    say("route_scores by logits", sigmoid, experts, groups, dtype)
    rng = np.random.default_rng(experts)
    z = 100 + 100 * rng.random((7, experts)) if sigmoid else rng.normal(size=(7, experts))
    if not sigmoid:  # two large logits per group decide its rank, the rest are far under them
        z = z - 1500
        for g in range(groups):
            z[:, g * (experts // groups):g * (experts // groups) + 2] = rng.normal(size=(7, 2))
    zb, z = stored(z, dtype)
    p = lib.Routing(experts=experts, k=k, score=int(sigmoid), groups=groups, groups_kept=kept, group_rank=1, renormalize=1, scale=1.0)
    ids, weights = Guarded(lib, 7 * k * 4), Guarded(lib, 7 * k * 4)
    lib.route_scores(dev(lib, zb), 7, p, ids.ptr, weights.ptr, CODE[dtype])
    lib.synchronize()
    want = by_logits(z, k, sigmoid, groups, kept)
    np.testing.assert_array_equal(ids.read(np.uint32).reshape(7, k), want)
    w = np.ones((7, k)) if sigmoid else np.exp(np.take_along_axis(z, want, 1) - z.max(1, keepdims=True))  # sigmoids: all 1
    np.testing.assert_allclose(weights.read(np.float32).reshape(7, k), w / w.sum(1, keepdims=True), rtol=12 * U, atol=2.0 ** -140)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_extreme_logits_in_groups(lib, sigmoid):
    z = np.array([[500.0, 400, 300, -300, -500, 0, 1, 2], [-1000, -999, -1001, -2000, -1500, -1200, -998, -3000], [39, 40, 41, 38, 45, 44, 46, 43]])
    say("route_scores extremes in groups", sigmoid)
    for kept in (1, 2, 3):
        k = 2 * kept
        p = lib.Routing(experts=8, k=k, score=int(sigmoid), groups=4, groups_kept=kept, group_rank=1, renormalize=0, scale=1.0)
        ids, weights = Guarded(lib, 3 * k * 4), Guarded(lib, 3 * k * 4)
        lib.route_scores(dev(lib, stored(z, "f32")[0]), 3, p, ids.ptr, weights.ptr, 0)
        lib.synchronize()
        got = ids.read(np.uint32).reshape(3, k).astype(int)
        for row, chosen in zip(z, got):  # whole groups, in the order of their logits
            assert len({e // 2 for e in chosen}) == kept and list(chosen) == sorted(chosen, key=lambda e: (-row[e], e))
