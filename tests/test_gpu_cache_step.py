"""A decoding step from the q/k/v product to the chosen token: product -> append with rotation -> attention -> output
product -> head -> adjusted logits -> argmax and draft verification, eager, recorded into graphs and on two streams; then
step after step of one sequence against attention over everything that was appended."""
import numpy as np
import pytest

from _cache import Batch, dequantize, quantize
from _ops import dev, stored, values
from _util import say
from test_gpu_cache import near, turned

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, D, V, P = 256, 8, 2, 64, 4000, 32
WIDTH = (HEADS + 2 * KV) * D


class Step:
    """Sequences with a prompt chunk, single tokens and drafts."""

    def __init__(self, lib, rows, lengths, seed):
        from oco_amd import synth
        rng = np.random.default_rng(seed)
        self.lib, b = lib, Batch(rng, rows, lengths, P)
        self.b, T, S = b, b.total, len(rows)
        d, new = (lambda a: dev(lib, a)), lib.DeviceBuffer
        self.x = stored(rng.normal(size=(T, HIDDEN)), "bf16")[0]
        self.w = {n: d(synth.weights(8, o, i, seed + j)) for j, (n, o, i) in enumerate([("qkv", WIDTH, HIDDEN), ("out", HIDDEN, HEADS * D), ("head", V, HIDDEN)])}
        self.f, self.magnitude = lib.rotation_frequencies(D, 10000.0, lib.Scaling.YARN, factor=4.0, original=64.0)
        self.cache = lib.PagedCache(b.pages, D, KV, P)
        self.keep = [d(b.table), d(np.array(lengths, np.uint32)), d(b.starts), d(self.f), d(rng.normal(size=HEADS).astype(np.float32))]
        self.rotation = lib.Rotation(dim=D, layout=0, magnitude=self.magnitude, frequencies=self.keep[3].ptr)
        self.batch = self.cache.batch(self.keep[0], self.keep[1], S, T, max(rows), max(lengths), b.stride, HEADS, starts=self.keep[2])
        self.i = {"x": d(self.x), "history": d(rng.integers(0, V, (T, 40)).astype(np.uint32)),
                  "penalties": d(np.tile(np.array([1.2, 0.1, 0.2], np.float32), (T, 1))), "mask": d((rng.integers(0, 2 ** 32, (T, V // 32)) | 1).astype(np.uint32)),
                  "u": d(rng.random((T, 1)).astype(np.float32))}
        self.o = {"qkv": new(T * WIDTH * 2), "q": new(T * HEADS * D * 2), "a": new(T * HEADS * D * 2), "h": new(T * HIDDEN * 2), "z": new(T * V * 4),
                  "y": new(T * V * 4), "best": new(4), "acc": new(T * 4), "tok": new(T * 4), "cache": self.cache.buffer}
        self.draft = lib.Draft(sequences=T, drafts=0, vocabulary=V, temperature=0.8)
        self.need = lib.draft_verify_workspace(self.draft)
        self.work = [new(self.need), new(max(lib.argmax_workspace(V), 16)), new(max(self.batch.workspace_bytes(), 16)), new(1 << 22)]

    def product(self, x, y, w, n, k, y_dtype, stream):
        m = self.b.total
        p = self.lib.Matrix(k, n, m, 0, 1, 1, 0)
        if m < 32:
            self.lib.matvec(8, self.w[w], x, y, p, 1, y_dtype, stream=stream)
        else:
            self.lib.matmul(8, self.w[w], x, y, p, 1, y_dtype, stream=stream, workspace=self.work[3], workspace_bytes=self.work[3].nbytes)

    def run(self, stream=None):
        lib, i, o, T = self.lib, self.i, self.o, self.b.total
        self.product(i["x"], o["qkv"], "qkv", WIDTH, HIDDEN, 1, stream)
        at = o["qkv"].ptr
        self.batch.append(at + HEADS * D * 2, at + (HEADS + KV) * D * 2, q=at, q_out=o["q"], rotation=self.rotation, stride=WIDTH, stream=stream)
        self.batch.attention(o["q"], o["a"], sinks=self.keep[4], workspace=self.work[2], stream=stream)
        self.product(o["a"], o["h"], "out", HIDDEN, HEADS * D, 1, stream)
        self.product(o["h"], o["z"], "head", V, HIDDEN, 0, stream)
        lib.logits_adjust(o["z"], o["y"], lib.Logits(rows=T, vocabulary=V, history_stride=40), history=i["history"], penalties=i["penalties"], mask=i["mask"],
                          stream=stream)
        lib.argmax(o["z"], V, o["best"], stream=stream, workspace=self.work[1], workspace_bytes=self.work[1].nbytes)
        lib.draft_verify(o["y"], None, None, i["u"], o["acc"], o["tok"], self.draft, workspace=self.work[0], workspace_bytes=self.need, stream=stream)

    def read(self):
        return {k: v.download(np.uint8) for k, v in self.o.items()}


def attended(step, q, k, v):
    """Rows [T, HEADS, D] from queries as the device holds them, and how far off they may be (bf16: as in the attention tests)."""
    out, tol, b = np.zeros(q.shape), np.zeros(q.shape), step.b
    sinks = step.keep[4].download(np.float32).astype(np.float64)
    for s, (n, length) in enumerate(zip(b.rows, b.lengths)):
        for i in range(n):
            r, at = int(b.starts[s]) + i, length - n + i
            for h in range(HEADS):
                kk, vv = k[s][:at + 1, h // (HEADS // KV)], v[s][:at + 1, h // (HEADS // KV)]
                score = kk @ q[r, h] / np.sqrt(D)
                top = max(score.max(), sinks[h])
                e = np.exp(score - top)
                total = e.sum() + np.exp(sinks[h] - top)
                out[r, h] = e @ vv / total
                d = ((D + 2) * (np.abs(kk) @ np.abs(q[r, h])).max() / np.sqrt(D) + 4 * (np.abs(score).max() + abs(top)) + 4) * 2.0 ** -24
                tol[r, h] = e @ np.abs(vv) / total * (2.0 ** -8 + 2 * d + 2 * (len(e) + 16) * 2.0 ** -24) + 2.0 ** -8 * np.abs(out[r, h]) * 1.001 + 2.0 ** -130
    return out, tol


@pytest.mark.parametrize("rows,lengths", [([1], [1]), ([1, 5, 3], [70, 5, 33]), ([40, 1, 2], [40, 200, 64])])
def test_step(lib, rows, lengths):
    """Each operator's result follows by its rule from what the one before it wrote."""
    say("cache step", rows, lengths)
    st = Step(lib, rows, lengths, seed=len(rows))
    b, T = st.b, st.b.total
    # what the sequences held before: appended in one call of their own, all tokens as rows
    rng = np.random.default_rng(77)
    before = [int(n) - r for r, n in zip(rows, lengths)]
    keys, vals = [np.zeros((n, KV, D)) for n in lengths], [np.zeros((n, KV, D)) for n in lengths]
    if sum(before):
        raw, old = stored(rng.normal(size=(sum(before), 2 * KV, D)), "bf16")
        starts = np.concatenate([[0], np.cumsum(before)]).astype(np.uint32)
        prefix = st.cache.batch(st.keep[0], dev(lib, np.array(before, np.uint32)), len(rows), sum(before), max(before), max(lengths), b.stride, HEADS,
                                starts=dev(lib, starts))
        buf = dev(lib, raw)
        prefix.append(buf.ptr, buf.ptr + KV * D * 2, stride=2 * KV * D)
        for s in range(len(rows)):
            part = old[starts[s]:starts[s + 1]]
            keys[s][:before[s]], vals[s][:before[s]] = dequantize(*quantize(part[:, :KV])), dequantize(*quantize(part[:, KV:]))
    st.run()
    lib.synchronize()
    o = st.read()
    qkv = values(o["qkv"], "bf16", (T, HEADS + 2 * KV, D))
    at = np.array([t for _, t in b.row_positions()])
    y, off = turned(qkv[:, :HEADS + KV], at, st.f, st.magnitude, D, False)
    q = values(o["q"], "bf16", (T, HEADS, D))
    near(q, y[:, :HEADS], off[:, :HEADS], "bf16")
    new_k, new_v = dequantize(*quantize(stored(y[:, HEADS:], "bf16")[1])), dequantize(*quantize(qkv[:, HEADS + KV:]))
    for r, (s, t) in enumerate(b.row_positions()):
        keys[s][t], vals[s][t] = new_k[r], new_v[r]
    want, tol = attended(st, q, keys, vals)
    got = values(o["a"], "bf16", (T, HEADS, D))
    assert np.all(np.abs(got - want) <= tol)
    # adjusted logits: hidden words are -Inf, the token is one that is left
    z, adj = o["z"].view(np.float32).reshape(T, V), o["y"].view(np.float32).reshape(T, V)
    bits = np.unpackbits(st.i["mask"].download(np.uint8).reshape(T, -1), axis=1, bitorder="little")[:, :V].astype(bool)
    assert np.all(adj[~bits] == -np.inf) and np.all(np.isfinite(adj[bits]))
    tok = o["tok"].view(np.uint32)
    assert all(bits[r, tok[r]] for r in range(T))
    assert o["best"].view(np.uint32)[0] == np.argmax(z[0])


def test_step_in_a_graph(lib):
    """Recorded and replayed, with eager work and waits between: every replay equals the eager run on the same inputs; two graphs
    with workspaces of their own run at once, and lengths change between replays."""
    streams = [lib.Stream(), lib.Stream()]
    steps = [Step(lib, [2, 1, 4], [60, 900, 4], seed=5), Step(lib, [33, 6], [400, 70], seed=6)]
    for st, s in zip(steps, streams):
        st.run(s)  # kernels loaded before the capture
        s.sync()
    graphs = [lib.Graph(s, lambda st=st, s=s: st.run(s)) for st, s in zip(steps, streams)]
    rng = np.random.default_rng(7)
    for turn in range(4):
        say("replay", turn)
        for st in steps:
            st.i["x"].upload(stored(rng.normal(size=(st.b.total, HIDDEN)), "bf16")[0])
            shorter = [max(n, length - turn) for n, length in zip(st.b.rows, st.b.lengths)]
            st.keep[1].upload(np.array(shorter, np.uint32))
        for g in graphs:
            g.launch()
        for s in streams:
            s.sync()
        got = [st.read() for st in steps]
        for st, g in zip(steps, got):
            st.run()
            lib.synchronize()
            want = st.read()
            for k in want:
                np.testing.assert_array_equal(g[k], want[k], err_msg=k)


def test_steps_on_two_streams_at_once(lib):
    """Two caches on two streams, scratch memory of each stream's own."""
    steps = [Step(lib, [3, 1, 1], [50, 700, 20 + i], seed=60 + i) for i in range(2)]
    for st in steps:
        st.work[2] = None  # the stream's
    want = []
    for st in steps:
        st.run()
        lib.synchronize()
        want.append(st.read())
    streams = [lib.Stream() for _ in steps]
    for _ in range(3):
        for st, s in zip(steps, streams):
            st.run(s)
    for s in streams:
        s.sync()
    for st, w in zip(steps, want):
        got = st.read()
        for k in w:
            np.testing.assert_array_equal(got[k], w[k], err_msg=k)


def test_token_by_token_equals_a_prompt(lib):
    """Tokens appended one at a time leave the pages of a prompt appended at once, and the last one's attention is the prompt's last row's."""
    rng = np.random.default_rng(8)
    n = 70
    b = Batch(rng, [n], [n], P)
    raw, _ = stored(rng.normal(size=(n, WIDTH)), "bf16")
    f, _ = lib.rotation_frequencies(D)
    keep = [dev(lib, b.table), dev(lib, f), dev(lib, raw)]
    r = lib.Rotation(dim=D, layout=1, magnitude=1.0, frequencies=keep[1].ptr)
    caches = [lib.PagedCache(b.pages, D, KV, P) for _ in range(2)]
    outs = []
    for cache, chunks in zip(caches, ([(0, n)], [(i, i + 1) for i in range(n)])):
        cache.buffer.fill32(0)
        for lo, hi in chunks:
            step = cache.batch(keep[0], dev(lib, np.array([hi], np.uint32)), 1, hi - lo, hi - lo, hi, b.stride, HEADS)
            at, q, out = keep[2].ptr + lo * WIDTH * 2, lib.DeviceBuffer((hi - lo) * HEADS * D * 2), lib.DeviceBuffer((hi - lo) * HEADS * D * 2)
            step.append(at + HEADS * D * 2, at + (HEADS + KV) * D * 2, q=at, q_out=q, rotation=r, stride=WIDTH)
            step.attention(q, out)
            lib.synchronize()
        outs.append(values(out.download(np.uint8), "bf16", (hi - lo, HEADS, D))[-1])
    np.testing.assert_array_equal(caches[0].buffer.download(np.uint8), caches[1].buffer.download(np.uint8))
    # either is within the rounding of its probabilities and of its result
    np.testing.assert_allclose(outs[0], outs[1], rtol=2.0 ** -7, atol=2.0 ** -6)
