"""oco_draft_verify against the rule in 64 bits: counts and tokens exactly,
probabilities within the roundings of f32 exponentials."""
import sys

import numpy as np
import pytest

from _ops import CODE, dev, stored
from _util import Guarded, say

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


def distribution(row, logits, temperature):
    if temperature == 0:
        if np.isnan(row).any() or (row == np.inf).any() or not (row > -np.inf).any():
            return None
        if not logits and not row.max() > 0:
            return None
        p = np.zeros_like(row)
        p[int(np.argmax(row))] = 1
        return p
    if not logits:
        return row
    if np.isnan(row).any() or (row == np.inf).any() or not (row > -np.inf).any():
        return None
    e = np.exp((row - row.max()) / np.float64(np.float32(temperature)))
    return e / e.sum()


def verify(target, draft, ids, lengths, u, t_logits, d_logits, temperature):
    S, D1, V = target.shape
    D = D1 - 1
    accepted, tokens, probs = np.zeros(S, np.int64), np.full((S, D1), NONE, np.int64), np.zeros((S, D1))
    for s in range(S):
        L = D if lengths is None else min(int(lengths[s]), D)
        n, rest, p = 0, None, None
        while True:
            p, rest = distribution(target[s, n], t_logits, temperature), None
            if n == L or p is None:
                break
            d = int(ids[s, n])
            if draft is None or temperature == 0:
                q = np.zeros(V)
                if d < V:
                    q[d] = 1
            else:
                q = distribution(draft[s, n], d_logits, temperature)
            pd, qd = (p[d] if d < V else 0.0), (1.0 if d >= V else np.nan if q is None else q[d])
            if (0 if temperature == 0 else np.float64(u[s, n])) * qd < pd < np.inf and (temperature > 0 or pd == 1):
                tokens[s, n], probs[s, n] = d, pd
                n += 1
                continue
            rest = None if q is None else np.where(np.isinf(q), np.nan, np.maximum(p - q, 0))
            if q is None or np.isnan(rest).any():
                p = None
            break
        accepted[s] = n
        if p is not None:
            rest = np.maximum(p, 0) if rest is None or rest.sum() <= 0 else rest
            sums = np.cumsum(rest)
            if not (sums[-1] > 0 and np.isfinite(sums[-1])):
                p = None
        if p is None:
            probs[s, n] = np.nan
            continue
        passed = np.nonzero((sums > (0 if temperature == 0 else np.float64(u[s, D])) * sums[-1]) & (rest > 0))[0]
        token = int(passed[0]) if len(passed) else int(np.nonzero(rest > 0)[0][-1])
        tokens[s, n], probs[s, n] = token, p[token]
    return accepted, tokens, probs


def run(lib, target, draft, ids, lengths, u, t_logits=True, d_logits=True, temperature=1.0, t_dtype="f32", d_dtype="f32", pad=(0, 0), stream=None,
        want_probs=True):
    """target [S, D+1, V], draft [S, D, V] or None as f64; the library's (accepted, tokens, probabilities) and the rule's."""
    S, D1, V = target.shape
    say("draft_verify", S, D1 - 1, V, t_logits, d_logits, temperature, t_dtype, d_dtype, draft is not None, lengths is not None)
    grown = [np.concatenate([a, np.full(a.shape[:2] + (x,), 77.0)], 2) if a is not None else None for a, x in ((target, pad[0]), (draft, pad[1]))]
    tb, tv = stored(grown[0], t_dtype)
    db, dv = stored(grown[1], d_dtype) if draft is not None else (None, None)
    p = lib.Draft(sequences=S, drafts=D1 - 1, vocabulary=V, target_values=0 if t_logits else 1, draft_values=0 if d_logits else 1,
                  target_dtype=CODE[t_dtype], draft_dtype=CODE[d_dtype], temperature=temperature, target_stride=V + pad[0] if pad[0] else 0,
                  draft_stride=V + pad[1] if pad[1] else 0)
    need = lib.draft_verify_workspace(p)
    work, acc, tok, prob = Guarded(lib, need), Guarded(lib, S * 4), Guarded(lib, S * D1 * 4), Guarded(lib, S * D1 * 4)
    u, ids = np.asarray(u, np.float32), np.asarray(ids)
    hold = [dev(lib, tb), dev(lib, db) if db is not None and db.size else None, dev(lib, np.asarray(ids, np.uint32)) if D1 > 1 else None, dev(lib, u),
            dev(lib, np.asarray(lengths, np.uint32)) if lengths is not None else None]
    lib.draft_verify(hold[0], hold[1], hold[2], hold[3], acc.ptr, tok.ptr, p, lengths=hold[4], probabilities=prob.ptr if want_probs else None,
                     workspace=work.ptr, workspace_bytes=need, stream=stream)
    lib.synchronize(stream)
    work.read(np.uint8)
    got = acc.read(np.uint32).astype(np.int64), tok.read(np.uint32).astype(np.int64).reshape(S, D1), prob.read(np.float32).reshape(S, D1)
    want = verify(tv[:, :, :V], dv[:, :, :V] if draft is not None else None, ids, lengths, u, t_logits, d_logits, temperature)
    np.testing.assert_array_equal(got[0], want[0])
    np.testing.assert_array_equal(got[1], want[1])
    if want_probs:
        # a row's sum is one of f32 exponentials 2^x, x = (v - max) log2(e) / T: each is off by a step of its own
        # (2 half steps of 2^-24) and by ln 2 |x| times the roundings of v - max and of the product with
        # log2(e) / T (1 half step each: 1.4 |x|); 4 additions in f32, the rest in 64 bits; the result's rounding.
        # Over the row |x| weighs in by p, and sum p |x| = H(p) - log2(1 / max p) <= log2(V), H the entropy in bits.
        np.testing.assert_allclose(got[2], want[2], rtol=(2 + 4 + 1 + 1.4 * np.log2(max(V, 2))) * 2.0 ** -24, atol=2.0 ** -140)
    return got


def sample(rng, S, D, V, noise=0.7, sharp=3.0):
    target = rng.normal(size=(S, D + 1, V)) * sharp
    draft = target[:, :D] + rng.normal(size=(S, D, V)) * noise
    ids = (draft + rng.gumbel(size=draft.shape)).argmax(2) if D else np.zeros((S, 0), np.int64)
    return target, draft, ids, rng.random((S, D + 1))


def softmax(z):
    e = np.exp(z - z.max(2, keepdims=True))
    return e / e.sum(2, keepdims=True)


@pytest.mark.parametrize("V", [1, 2, 7, 100, 4095, 4096, 4097, 8200, 32001])
@pytest.mark.parametrize("S,D", [(1, 1), (3, 4), (2, 0)])
def test_vocabularies(lib, S, D, V):
    rng = np.random.default_rng(V + D)
    t, d, ids, u = sample(rng, S, D, V)
    run(lib, t, d, ids, None, u)
    run(lib, t, None, ids, None, u, temperature=0.8)
    run(lib, t, d, ids, None, u, temperature=0.0)
    run(lib, softmax(t), softmax(d) if D else d, ids, None, u, False, False)


@pytest.mark.parametrize("t_dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d_dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t_logits,d_logits", [(True, True), (True, False), (False, False), (False, True)])
def test_types_and_kinds(lib, t_dtype, d_dtype, t_logits, d_logits):
    rng = np.random.default_rng(11)
    t, d, ids, u = sample(rng, 5, 3, 5000)
    run(lib, t if t_logits else softmax(t), d if d_logits else softmax(d), ids, [3, 0, 2, 1, 900], u, t_logits, d_logits, 1.0, t_dtype, d_dtype, pad=(3, 5))


@pytest.mark.parametrize("temperature", [0.01, 0.3, 1.0, 7.5])
def test_temperatures(lib, temperature):
    rng = np.random.default_rng(int(temperature * 100))
    t, d, ids, u = sample(rng, 6, 5, 9000)
    got = run(lib, t, d, ids, None, u, temperature=temperature)
    assert got[0].max() > 0 or temperature < 1


def test_accepts_everything_where_the_drafter_is_the_target(lib):
    rng = np.random.default_rng(1)
    t, _, ids, u = sample(rng, 4, 64, 300)
    got = run(lib, t, t[:, :64], ids, None, u)
    assert np.all(got[0] == 64) and np.all(got[1] != NONE)


def test_refused_with_nothing_left_draws_from_the_target(lib):
    """p == q as probabilities, but a drafted id of probability 0: refused,
    max(p - q, 0) is 0 everywhere, and the token comes from p."""
    p = np.zeros((1, 2, 10))
    p[:, :, 3], p[:, :, 7] = 0.25, 0.75
    for u, token in ((0.1, 3), (0.24, 3), (0.26, 7), (0.9999999, 7)):
        got = run(lib, p, p[:, :1], [[5]], None, [[0.0, u]], False, False)
        assert got[0][0] == 0 and got[1][0, 0] == token and got[1][0, 1] == NONE


def test_random_numbers_at_their_ends(lib):
    """u = 0 takes the first token with any probability, the largest u below
    1 the last one; acceptance is strict."""
    last = np.float32(1) - np.float32(2.0 ** -24)
    p = np.zeros((1, 2, 6000))
    p[0, :, 100], p[0, :, 5000] = 0.5, 0.5
    q = np.zeros((1, 1, 6000))
    q[0, 0, 100] = 1.0
    for u0, u1, want in ((0.0, 0.0, (1, 100, 100)), (0.5, 0.0, (0, 5000, NONE)), (0.49999997, last, (1, 100, 5000)), (last, last, (0, 5000, NONE))):
        got = run(lib, p, q, [[100]], None, [[u0, u1]], False, False)
        assert (got[0][0], got[1][0, 0], got[1][0, 1]) == want


def test_masked_tokens_and_ids_past_the_vocabulary(lib):
    rng = np.random.default_rng(3)
    t, d, ids, u = sample(rng, 6, 3, 9000)
    t[:, :, :5000] = -np.inf  # a whole chunk of 4096 and part of the next
    d[0, :, ::2] = -np.inf
    ids[1, 0], ids[2, 1], ids[3, 2] = 9000, 0x7FFFFFFF, 100  # past the vocabulary; masked in the target
    run(lib, t, d, ids, None, u)
    run(lib, t, None, ids, None, u)
    run(lib, t, None, ids, None, u, temperature=0.0)
    t[4] = -np.inf
    t[4, :, 8999] = -3.0  # one token left
    run(lib, t, d, ids, None, u)


@pytest.mark.parametrize("bad", [np.nan, np.inf, None])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_rows_without_a_distribution_end_their_sequence(lib, bad, temperature):
    rng = np.random.default_rng(4)
    t, _, ids, u = sample(rng, 5, 3, 4100)
    d = t[:, :3].copy()
    for s, i in ((0, 0), (1, 2), (2, 3)):
        if bad is None:
            t[s, i] = -np.inf
        else:
            t[s, i, 4099] = bad
    ids[:, :] = np.where(np.isfinite(d), d, -9e9).argmax(2)
    got = run(lib, t, d, ids, None, u, temperature=temperature)
    assert got[1][0, 0] == NONE and np.isnan(got[2][0, 0])
    if temperature > 0 and bad is not None:
        d2 = rng.normal(size=d.shape)
        d2[3, 1, 7] = bad
        run(lib, t, d2, ids, None, u)


def test_rows_of_probabilities_without_a_distribution(lib):
    """Infinite or missing probabilities: at a drafted id, in the row that a
    token is drawn from, in the drafter's; greedy rows of zeros."""
    rng = np.random.default_rng(14)
    t, _, ids, u = sample(rng, 5, 2, 4200)
    t = softmax(t)
    d = t[:, :2].copy()
    t[0, 0, ids[0, 0]] = np.inf
    t[1, 2, 4199] = np.inf
    t[2, 2] = 0.0
    d[3, 1, ids[3, 1]] = np.inf
    got = run(lib, t, d, ids, None, u, False, False)
    assert [list(r).index(NONE) for r in got[1][:4]] == [0, 2, 2, 1]
    t[4, 0] = 0.0
    got = run(lib, t, None, t.argmax(2)[:, :2], None, u, False, temperature=0.0)
    assert [int(x) for x in got[0]] == [0, 2, 2, 2, 0] and list(got[1][:, 2]) == [NONE, NONE, NONE, got[1][3, 2], NONE]


@pytest.mark.parametrize("temperature", [2.0 ** -126, 2.0 ** 64])
def test_the_ends_of_the_temperatures(lib, temperature):
    rng = np.random.default_rng(15)
    t, d, ids, u = sample(rng, 4, 2, 4200)
    t[:, :, 4000:] = -np.inf
    run(lib, t, d, ids, None, u, temperature=temperature)


def test_greedy_takes_the_first_of_equal_values(lib):
    t = np.zeros((1, 3, 5000))
    t[0, 0, [4500, 300]] = 2.0
    t[0, 1, [10, 11]] = -0.0
    got = run(lib, t, None, [[300, 0]], None, [[0, 0, 0]], temperature=0.0)
    assert list(got[1][0]) == [300, 0, 0] and got[0][0] == 2
    t[0, 0, 200] = 2.0
    got = run(lib, t, None, [[300, 0]], None, [[0, 0, 0]], temperature=0.0)
    assert list(got[1][0]) == [200, NONE, NONE] and got[0][0] == 0


def test_large_vocabulary_and_batch(lib):
    rng = np.random.default_rng(5)
    t, d, ids, u = sample(rng, 3, 2, 151936)
    run(lib, t, d, ids, [2, 1, 0], u)
    run(lib, t, d, ids, None, u, temperature=0.5, t_dtype="bf16", want_probs=False)
    t, d, ids, u = sample(rng, 33, 2, 150)
    run(lib, t, d, ids, None, u)


def test_more_chunks_than_lanes(lib):
    """A vocabulary of more than 64 chunks of 4096, flat, so that the drawn
    token lies anywhere."""
    rng = np.random.default_rng(6)
    V = 300001
    t = rng.normal(size=(4, 1, V)) * 0.01
    got = run(lib, t, np.zeros((4, 0, V)), np.zeros((4, 0), int), None, [[0.0], [0.3], [0.9], [0.9999999]])
    assert got[1][1, 0] > 64 * 1000 and got[1][2, 0] > 64 * 4096


def test_the_result_is_distributed_as_the_target(lib):
    """Over a grid of random numbers the emitted first token's frequencies
    are the target's probabilities, whatever the drafter: with G equal steps
    of u for each of the two draws, each of the V thresholds of either draw
    shifts a frequency by at most 1 / G."""
    rng = np.random.default_rng(7)
    V, G = 6, 40
    p, q = softmax(rng.normal(size=(1, 1, V)))[0, 0], softmax(rng.normal(size=(1, 1, V)))[0, 0]
    freq = np.zeros(V)
    grid = (np.arange(G) + 0.5) / G
    u = np.stack(np.meshgrid(grid, grid, indexing="ij"), -1).reshape(-1, 2)
    for d in range(V):  # the drafter proposes d with probability q[d]
        S = len(u)
        target = np.broadcast_to(p, (S, 2, V)).copy()
        got = run(lib, target, np.broadcast_to(q, (S, 1, V)).copy(), np.full((S, 1), d), None, u, False, False)
        freq += q[d] * np.bincount(got[1][:, 0], minlength=V)[:V] / S
    assert np.all(np.abs(freq - p) <= 2.0 / G)


@pytest.mark.parametrize("t_dtype,d_dtype", [("f32", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("S", [4, 300])
def test_values_under_zero_count_as_zero(lib, monkeypatch, S, t_dtype, d_dtype):
    """Negative probabilities on both sides, -Inf among them, at drafted ids
    and elsewhere: the rule on rows whose negative values are 0.  A token that
    the target gives nothing is neither accepted nor drawn."""
    zeroed = lambda a: None if a is None else np.where(a < 0, 0.0, a)  # noqa: E731
    plain = verify
    monkeypatch.setattr(sys.modules[__name__], "verify", lambda t, d, *rest: plain(zeroed(t), zeroed(d), *rest))
    rng = np.random.default_rng(16)
    D, V = 3, 9000
    t, d, ids, u = sample(rng, S, D, V)
    t, d = softmax(t), softmax(d)
    t[:, :, ::5] *= -1
    d[:, :, ::7] *= -1
    t[:, :, 11], d[:, :, 13] = -np.inf, -np.inf
    rows = np.arange(S)
    ids[:2, 0] = 35, 70  # negative on both sides
    ids[2, 0], ids[3, 0] = 11, 13
    u[:2, 0] = 0.0, 0.5
    run(lib, t, d, ids, None, u, False, False, t_dtype=t_dtype, d_dtype=d_dtype)
    run(lib, t, None, ids, None, u, False, t_dtype=t_dtype)
    t[:, :, ids[:, 0]] = 0.0  # refused, unless a negative q lets it in
    d[rows, 0, ids[:, 0]] = -0.25
    got = run(lib, t, d, ids, None, u, False, False, t_dtype=t_dtype, d_dtype=d_dtype)
    assert not got[0].any()
    t[:, :, :] = 0.0
    t[:, :, 17] = 1.0
    d[:, :, :] = -1.0
    d[:, :, 17] = 1.0  # nothing left but what negative values would add
    got = run(lib, t, d, np.zeros_like(ids), None, u, False, False, t_dtype=t_dtype, d_dtype=d_dtype)
    assert np.all(got[1][:, 0] == 17)


BATCH = dict(S=130, D=2, V=17001)  # 650 chunks of 4096: past the number that decide for themselves


@pytest.mark.parametrize("t_dtype,d_dtype,draft,temperature,ragged", [
    ("f32", "f32", "logits", 1.0, False), ("bf16", "f32", "logits", 0.7, True), ("bf16", "f32", None, 0.8, True), ("f16", "bf16", "probabilities", 1.0, True),
    ("f32", "f16", "logits", 1.3, True), ("f32", "f32", None, 0.0, True)])
def test_large_batches(lib, t_dtype, d_dtype, draft, temperature, ragged):
    """Decisions in a launch of their own: vocabularies of several chunks and
    of steps that are not whole, masked, absent and NaN rows."""
    rng = np.random.default_rng(17)
    t, d, ids, u = sample(rng, **BATCH)
    lengths = rng.integers(0, 4, BATCH["S"]) if ragged else None
    t[5, :, :4096] = -np.inf
    t[6, 1, 17000] = np.nan
    t[7, 0] = -np.inf
    t[8, :, 17000] = 60.0  # all of it in the last, partial step
    ids[9, 0] = 17001
    d = None if draft is None else softmax(d) if draft == "probabilities" else d
    run(lib, t, d, ids, lengths, u, True, draft != "probabilities", temperature, t_dtype, d_dtype, pad=(3, 0))


@pytest.mark.parametrize("t_logits,draft", [(True, "logits"), (True, None), (False, "probabilities")])
def test_a_batch_equals_its_sequences_in_small_calls(lib, t_logits, draft):
    rng = np.random.default_rng(18)
    t, d, ids, u = sample(rng, **BATCH)
    t = t if t_logits else softmax(t)
    d = None if draft is None else softmax(d) if draft == "probabilities" else d
    whole = run(lib, t, d, ids, None, u, t_logits, draft == "logits")
    for s in range(0, BATCH["S"], 13):
        part = run(lib, t[s:s + 13], None if d is None else d[s:s + 13], ids[s:s + 13], None, u[s:s + 13], t_logits, draft == "logits")
        for a, b in zip(whole, part):
            np.testing.assert_array_equal(a[s:s + 13], b)


@pytest.mark.parametrize("S", [1, 3])
def test_more_chunks_than_lanes_in_few_sequences(lib, S):
    """Decisions in every workgroup, on rows of more than 64 chunks."""
    rng = np.random.default_rng(19)
    t, d, ids, u = sample(rng, S, 2, 300001, sharp=1.0)
    run(lib, t, d, ids, None, u)
    run(lib, t, None, t[:, :2].argmax(2), None, u, temperature=0.2)
