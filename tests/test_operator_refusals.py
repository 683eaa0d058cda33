"""Arguments that the row operators refuse, before any GPU work (the pointers
are never read), and their workspace sizes."""
import ctypes

import pytest

import oco_amd as oco

FAKE = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1008)


def refused(rc, word, code=1):
    message = oco.load_library().oco_last_error().decode()
    assert rc == code, (rc, message)
    assert word in message, message


def block(**over):
    d = dict(rows=4, n=256, x_dtype=1, dtype=1, gate=1, scale=1.0, epsilon=1e-6)
    d.update(over)
    return oco.Block(**d)


def call_block(p, x=FAKE, y=FAKE, x_out=FAKE, gate=FAKE, post=FAKE, pre=FAKE, out=FAKE, codes=None, scales=None):
    return oco.load_library().oco_block_norm(x, y, x_out, gate, post, pre, out, codes, scales, ctypes.byref(p), None)


def test_block_norm():
    refused(call_block(block(gate=4)), "gate 4")
    refused(call_block(block(), gate=None), "without gate rows")
    for missing in ("x", "y", "x_out"):
        refused(call_block(block(), **{missing: None}), "null pointer")
    refused(call_block(block(), pre=None), "second norm")
    refused(call_block(block(), out=None), "second norm")
    refused(call_block(block(), codes=FAKE), "come together")
    refused(call_block(block(n=250), codes=FAKE, scales=FAKE), "n % 16")
    refused(call_block(block(), codes=ODD, scales=FAKE), "16-byte")
    for stride in ("x_stride", "y_stride", "gate_stride", "out_stride"):
        refused(call_block(block(**{stride: 255})), "stride of 255")
    refused(call_block(block(x_dtype=1, dtype=2)), "residual type", 2)
    refused(call_block(block(x_dtype=1, dtype=0)), "residual type", 2)
    refused(call_block(block(x_dtype=7, dtype=7)), "residual type", 2)
    refused(oco.load_library().oco_block_norm(*[FAKE] * 7, None, None, None, None), "null description")
    assert call_block(block(rows=0), x=None) == 0 and call_block(block(n=0), y=None) == 0


def test_fp8():
    L = oco.load_library()
    quant = lambda x=FAKE, dt=1, rows=4, k=256, stride=0, codes=FAKE, scales=FAKE: L.oco_fp8_quantize(x, dt, rows, k, stride, codes, scales, None)  # noqa: E731
    refused(quant(k=250), "k % 16")
    refused(quant(codes=ODD), "16-byte")
    refused(quant(stride=255), "stride")
    refused(quant(x=None), "null pointer")
    refused(quant(scales=None), "null pointer")
    refused(quant(dt=5), "type 5", 2)
    refused(quant(rows=0x7FFFFFFF, k=0x7FFFFF0), "rows of")
    assert quant(rows=0, x=None) == 0

    def product(w=FAKE, ws=FAKE, codes=FAKE, scales=FAKE, y=FAKE, dt=0, bias=None, k=256, n=64, m=4, experts=1, has_bias=0, work=None, bytes_=0):
        p = oco.Matrix(k, n, m, 0, 1, experts, has_bias)
        return L.oco_fp8_matmul(w, ws, codes, scales, y, dt, bias, ctypes.byref(p), work, bytes_, None)
    refused(product(k=250), "groups of 16")
    refused(product(k=0), "groups of 16")
    for missing in ("w", "ws", "codes", "scales", "y"):
        refused(product(**{missing: None}), "null pointer")
    refused(product(has_bias=1), "null pointer")
    refused(product(has_bias=2, bias=FAKE), "has_bias 2", 2)
    refused(product(experts=4), "dense", 2)
    refused(product(dt=3), "type 3", 2)
    refused(product(w=ODD), "16-byte")
    refused(product(codes=ODD), "16-byte")
    refused(product(k=0x400010), "x 4194320")
    refused(L.oco_fp8_matmul(FAKE, FAKE, FAKE, FAKE, FAKE, 0, None, None, None, 0, None), "null matrix")
    assert product(m=0, w=None) == 0 and product(n=0, w=None) == 0
    with pytest.raises(ValueError):
        oco.Fp8Matrix(None, None, 100, 64)


def routing(**over):
    d = dict(experts=64, k=8, score=0, groups=1, groups_kept=1, group_rank=0, renormalize=1, scale=1.0)
    d.update(over)
    return oco.Routing(**d)


def test_route_scores():
    L = oco.load_library()
    call = lambda p, logits=FAKE, dt=0, tokens=4, ids=FAKE, w=FAKE: L.oco_route_scores(logits, dt, None, tokens, ctypes.byref(p), ids, w, None)  # noqa: E731
    refused(call(routing(experts=1025)), "of 1025 experts")
    refused(call(routing(experts=0)), "of 0 experts")
    refused(call(routing(k=0)), "0 of 64")
    refused(call(routing(k=33)), "33 of 64")
    refused(call(routing(experts=4, k=5)), "5 of 4")
    refused(call(routing(score=2)), "score 2")
    refused(call(routing(group_rank=2)), "rank 2")
    refused(call(routing(groups=7)), "7 groups")
    refused(call(routing(experts=130, groups=65)), "65 groups")
    refused(call(routing(groups=8, groups_kept=0)), "from 0 of 8")
    refused(call(routing(groups=8, groups_kept=9)), "from 9 of 8")
    refused(call(routing(groups=16, groups_kept=1)), "from 1 of 16")  # 8 of a group of 4
    refused(call(routing(), logits=None), "null pointer")
    refused(call(routing(), ids=None), "null pointer")
    refused(call(routing(), w=None), "null pointer")
    refused(call(routing(), dt=3), "type 3", 2)
    refused(L.oco_route_scores(FAKE, 0, None, 4, None, FAKE, FAKE, None), "null description")
    assert call(routing(), tokens=0, logits=None) == 0


def draft(**over):
    d = dict(sequences=2, drafts=3, vocabulary=1000, temperature=1.0)
    d.update(over)
    return oco.Draft(**d)


def test_draft_verify():
    L = oco.load_library()

    def call(p, target=FAKE, rows=FAKE, ids=FAKE, u=FAKE, acc=0x2000, tok=0x3000, work=FAKE, bytes_=1 << 30):
        return L.oco_draft_verify(target, rows, ids, None, u, acc, tok, None, ctypes.byref(p), work, bytes_, None)
    bad = [(dict(drafts=65), "too many drafts"), (dict(vocabulary=0), "vocabulary"), (dict(vocabulary=1 << 31), "vocabulary"),
           (dict(target_values=2), "kind"), (dict(draft_values=2), "kind"), (dict(target_dtype=3), "type"), (dict(draft_dtype=9), "type"),
           (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
           (dict(target_stride=999), "stride"), (dict(draft_stride=1), "stride"), (dict(sequences=1 << 31, vocabulary=1 << 30), "too many rows")]
    for over, word in bad:
        refused(call(draft(**over)), word)
        assert oco.draft_verify_workspace(draft(**over)) == 0
    for missing in ("target", "ids", "u", "acc", "tok"):
        refused(call(draft(), **{missing: None}), "null pointer")
    need = oco.draft_verify_workspace(draft())
    assert need > 0 and need % 16 == 0
    refused(call(draft(), bytes_=need - 1), "workspace")
    refused(call(draft(), work=None), "workspace")
    refused(call(draft(), work=ODD), "workspace")
    refused(L.oco_draft_verify(*[FAKE] * 8, None, FAKE, 1 << 30, None), "null description")
    assert call(draft(sequences=0), target=None) == 0


def test_draft_verify_apart():
    """Outputs over the ids, the lengths or the random numbers; temperatures whose exponents f32 cannot hold."""
    L = oco.load_library()

    def call(acc, tok, prob, p=None):  # 2 sequences of 3: ids 24 bytes, lengths 8, random numbers 32
        return L.oco_draft_verify(FAKE, FAKE, 0x10000, 0x20000, 0x30000, acc, tok, prob, ctypes.byref(p or draft()), FAKE, 0, None)
    for acc, tok, prob in ((0x20000, 0x50000, 0x60000), (0x20004, 0x50000, None), (0x40000, 0x10000, None), (0x40000, 0x10000 - 28, None),
                           (0x40000, 0x50000, 0x30000), (0x30000 + 28, 0x50000, None), (0x40000, 0x20000, None)):
        refused(call(acc, tok, prob), "lies over")
    for acc, tok, prob in ((0x20008, 0x50000, 0x60000), (0x40000, 0x10000 - 32, 0x30020), (0x20000 - 8, 0x10018, None)):
        refused(call(acc, tok, prob), "workspace")
    refused(call(0x40000, 0x50000, 0x30000, draft(temperature=0.0)), "workspace")  # greedy reads no random numbers
    for t in (2.0 ** -127, 2.0 ** 65, 1e-45):
        refused(call(0x40000, 0x50000, None, draft(temperature=t)), "temperature")
