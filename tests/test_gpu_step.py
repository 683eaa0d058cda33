"""The row operators together, as a decoding step of a routed 8-bit model uses
them: block step with 8-bit rows -> product; router logits -> experts by
scores -> the expert layer; block step -> lm_head -> verification.  The whole
run recorded into a graph and replayed equals the calls one by one."""
import numpy as np
import pytest

from _ops import dev, e4m3, quantized, stored, values
from _util import say
from test_gpu_draft import verify
from test_gpu_fp8 import operands, product
from test_gpu_route_scores import reference

pytestmark = pytest.mark.gpu
HIDDEN, FFN, E, K, V, GROUPS, KEPT = 512, 256, 64, 4, 3000, 8, 3


class Step:
    """S sequences of `drafts` drafted tokens: rows = S * (drafts + 1)."""

    def __init__(self, lib, S, drafts, seed):
        from oco_amd import synth
        rng = np.random.default_rng(seed)
        self.lib, self.S, self.D, self.rows = lib, S, drafts, S * (drafts + 1)
        r = self.rows
        self.x, self.y = stored(rng.normal(size=(r, HIDDEN)), "bf16")[0], stored(rng.normal(size=(r, HIDDEN)), "bf16")[0]
        self.norms = [(1 + 0.1 * rng.normal(size=HIDDEN)).astype(np.float32) for _ in range(4)]
        self.gate = stored(rng.normal(size=(1, HIDDEN)), "bf16")[0]
        _, self.router_w, _, self.router_s = operands(rng, 1, E, HIDDEN)
        _, self.head_w, _, self.head_s = operands(rng, 1, V, HIDDEN)
        self.router_s, self.head_s = self.router_s * 0.05, self.head_s * 0.1
        self.bias = (0.02 * rng.normal(size=E)).astype(np.float32)
        self.bank_host = [synth.weights(12, E * n, k, seed + i) for i, (n, k) in enumerate([(FFN, HIDDEN), (FFN, HIDDEN), (HIDDEN, FFN)])]
        self.ids = rng.integers(0, V, (S, drafts)).astype(np.uint32)
        self.u = rng.random((S, drafts + 1)).astype(np.float32)
        d = lambda a: dev(lib, a)  # noqa: E731
        self.b = {"x": d(self.x), "y": d(self.y), "gate": d(self.gate), "rw": d(self.router_w), "rs": d(self.router_s), "hw": d(self.head_w),
                  "hs": d(self.head_s), "bias": d(self.bias), "ids": d(self.ids), "u": d(self.u), "zero": d(np.zeros((r, HIDDEN), np.uint16))}
        self.n = [d(n) for n in self.norms]
        self.bank = lib.ExpertBank(12, HIDDEN, FFN, E, K, *[d(w) for w in self.bank_host], activation=1, up_bias_one=False)
        kb = HIDDEN // 128
        new = lib.DeviceBuffer
        self.o = {"x1": new(r * HIDDEN * 2), "h": new(r * HIDDEN * 2), "codes": new(r * HIDDEN), "scales": new(kb * r * 4), "logits": new(r * E * 4),
                  "eid": new(r * K * 4), "w": new(r * K * 4), "moe": new(r * HIDDEN * 2), "x2": new(r * HIDDEN * 2), "codes2": new(r * HIDDEN),
                  "scales2": new(kb * r * 4), "vocab": new(r * V * 4), "acc": new(S * 4), "tok": new(r * 4), "prob": new(r * 4)}
        self.draft = lib.Draft(sequences=S, drafts=drafts, vocabulary=V, temperature=0.9)
        self.pr, self.ph = lib.Matrix(HIDDEN, E, r, 0, 1, 1, 0), lib.Matrix(HIDDEN, V, r, 0, 1, 1, 0)
        self.need = [lib.draft_verify_workspace(self.draft), lib.fp8_matmul_workspace(self.pr), lib.fp8_matmul_workspace(self.ph)]
        self.work = [new(max(n, 16)) for n in self.need] + [new(self.bank.workspace_bytes(r))]

    def run(self, stream=None):
        lib, o, b, r = self.lib, self.o, self.b, self.rows
        lib.block_norm(b["x"], b["y"], lib.Block(rows=r, n=HIDDEN, x_dtype=1, dtype=1, gate=2, scale=0.7, epsilon=1e-6), x_out=o["x1"], gate=b["gate"],
                       post_w=self.n[0], pre_w=self.n[1], out=o["h"], codes=o["codes"], scales=o["scales"], stream=stream)
        lib.fp8_matmul(b["rw"], b["rs"], o["codes"], o["scales"], o["logits"], self.pr, workspace=self.work[1], workspace_bytes=self.need[1], stream=stream)
        lib.route_scores(o["logits"], r, lib.Routing(experts=E, k=K, score=1, groups=GROUPS, groups_kept=KEPT, group_rank=1, renormalize=1, scale=1.5),
                         o["eid"], o["w"], bias=b["bias"], stream=stream)
        # the expert layer adds to its output rows: start from zeros
        lib._check(lib.load_library().oco_buffer_copy(o["moe"].ptr, b["zero"].ptr, r * HIDDEN * 2, lib._stream(stream)))
        self.bank.apply(o["h"], lib.DType.BF16, o["eid"], o["w"], r, o["moe"], workspace=self.work[3], stream=stream)
        lib.block_norm(o["x1"], o["moe"], lib.Block(rows=r, n=HIDDEN, x_dtype=1, dtype=1, scale=1.0, epsilon=1e-6), x_out=o["x2"], post_w=self.n[2],
                       pre_w=self.n[3], codes=o["codes2"], scales=o["scales2"], stream=stream)
        lib.fp8_matmul(b["hw"], b["hs"], o["codes2"], o["scales2"], o["vocab"], self.ph, workspace=self.work[2], workspace_bytes=self.need[2], stream=stream)
        lib.draft_verify(o["vocab"], None, b["ids"], b["u"], o["acc"], o["tok"], self.draft, probabilities=o["prob"], workspace=self.work[0],
                         workspace_bytes=self.need[0], stream=stream)

    def read(self):
        return {k: v.download(np.uint8) for k, v in self.o.items()}


@pytest.mark.parametrize("S,drafts", [(1, 0), (3, 4), (20, 3)])
def test_step(lib, S, drafts):
    """Each operator's result follows by its rule from what the one before it wrote."""
    say("step", S, drafts)
    st = Step(lib, S, drafts, seed=S)
    st.run()
    lib.synchronize()
    o, r, kb = st.read(), st.rows, HIDDEN // 128
    # 8-bit rows -> router logits
    codes, scales = o["codes"].reshape(r, HIDDEN), o["scales"].view(np.float32).reshape(kb, r)
    want, mag = product(codes, st.router_w, scales, st.router_s)
    logits = o["logits"].view(np.float32).reshape(r, E)
    assert np.all(np.abs(logits - want) <= (256 + kb + 12) * 2.0 ** -24 * mag)
    # the 8-bit rows stand for the bf16 ones: within half a code step and a bf16 rounding
    h = values(o["h"], "bf16", (r, HIDDEN))
    back = e4m3(o["codes"], (r, HIDDEN)) * np.repeat(scales.T.astype(np.float64), 128, 1)
    assert np.all(np.abs(back - h) <= np.maximum(np.abs(h) * 2.0 ** -4, np.repeat(scales.T, 128, 1) * 2.0 ** -10) * 1.01 + np.abs(h) * 2.0 ** -8)
    # experts from the logits
    ids, w = reference(logits.astype(np.float64), st.bias, K, True, GROUPS, KEPT, True, True, 1.5)
    np.testing.assert_array_equal(o["eid"].view(np.uint32).reshape(r, K), ids)
    np.testing.assert_allclose(o["w"].view(np.float32).reshape(r, K), w, rtol=12 * 2.0 ** -24)
    # the expert layer took those ids: its own call on the same inputs gives the same rows
    out = lib.DeviceBuffer.from_array(np.zeros((r, HIDDEN), np.uint16))
    st.bank.apply(st.o["h"], lib.DType.BF16, st.o["eid"], st.o["w"], r, out)
    lib.synchronize()
    np.testing.assert_array_equal(out.download(np.uint8), o["moe"])
    # lm_head and verification
    c2, s2 = o["codes2"].reshape(r, HIDDEN), o["scales2"].view(np.float32).reshape(kb, r)
    want, mag = product(c2, st.head_w, s2, st.head_s)
    vocab = o["vocab"].view(np.float32).reshape(r, V)
    assert np.all(np.abs(vocab - want) <= (256 + kb + 12) * 2.0 ** -24 * mag)
    acc, tok, _ = verify(vocab.astype(np.float64).reshape(S, drafts + 1, V), None, st.ids, None, st.u, True, True, np.float32(0.9))
    np.testing.assert_array_equal(o["acc"].view(np.uint32), acc)
    np.testing.assert_array_equal(o["tok"].view(np.uint32).reshape(S, drafts + 1), tok)


def test_step_in_a_graph(lib):
    """Recorded and replayed, with eager work and waits between: every replay
    equals the eager run on the same inputs, after the inputs change too; a
    second graph of other sizes runs between the replays."""
    stream, other = lib.Stream(), lib.Stream()
    a, b = Step(lib, 5, 3, seed=50), Step(lib, 2, 1, seed=51)
    for st, s in ((a, stream), (b, other)):
        st.run(s)  # kernels loaded before the capture
        s.sync()
    ga, gb = lib.Graph(stream, lambda: a.run(stream)), lib.Graph(other, lambda: b.run(other))
    rng = np.random.default_rng(52)
    for turn in range(4):
        say("replay", turn)
        for st in (a, b):
            st.b["x"].upload(stored(rng.normal(size=(st.rows, HIDDEN)), "bf16")[0])
            st.b["u"].upload(rng.random((st.S, st.D + 1)).astype(np.float32))
        ga.launch()
        gb.launch()
        stream.sync()
        other.sync()
        got = a.read(), b.read()
        for st, g in ((a, got[0]), (b, got[1])):
            st.run()
            lib.synchronize()
            want = st.read()
            for k in want:
                np.testing.assert_array_equal(g[k], want[k], err_msg=k)


def test_calls_on_two_streams_at_once(lib):
    """The same operators on two streams with workspaces of their own."""
    steps = [Step(lib, 4, 3, seed=60 + i) for i in range(2)]
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
