"""oco_logits_adjust against its rule in 64 bits."""
import numpy as np
import pytest

from _ops import CODE, HALF, LEAST, SIZE, U, dev, stored, values
from _util import Guarded, say

pytestmark = pytest.mark.gpu


def adjusted(x, history, penalties, biases, mask, group, mask_group):
    """(values, tolerance in f32 steps' magnitude); history and biases: lists per group, of ids and (id, bias)."""
    y, mag = x.copy(), np.abs(x)
    V = x.shape[1]
    for r in range(len(x)):
        g = r // group
        if history is not None:
            ids, count = np.unique([i for i in history[g] if i < V], return_counts=True)
            ids = ids.astype(int)
            rep, freq, pres = penalties[g].astype(np.float64)
            with np.errstate(all="ignore"):
                v = np.where(y[r, ids] > 0, y[r, ids] / rep, y[r, ids] * rep)
                y[r, ids] = v - (freq * count + pres)
                mag[r, ids] = np.abs(v) + np.abs(freq) * count + np.abs(pres)
        if biases is not None:
            for i, b in {i: b for i, b in biases[g] if i < V}.items():
                y[r, i] += np.float64(b)
                mag[r, i] += abs(np.float64(b))
        if mask is not None:
            y[r, ~mask[r // mask_group]] = -np.inf
    return y, mag


def bits(mask, stride):
    raw = np.zeros((len(mask), stride * 4), np.uint8)
    packed = np.packbits(mask, axis=1, bitorder="little")
    raw[:, :packed.shape[1]] = packed
    raw[:, packed.shape[1]:] = 0xFF  # words behind the row are not looked at
    return raw.view(np.uint32)


def run(lib, rng, rows, V, dtype="f32", H=0, B=0, masked=False, lengths=True, group=1, mask_group=1, pad=(0, 0), in_place=False, x=None, mask_pad=0,
        history=None, biases=None, stream=None):
    groups, mgroups = -(-rows // group), -(-rows // mask_group)
    say("logits", rows, V, dtype, H, B, masked, group, mask_group, pad, in_place)
    raw, full = stored(rng.normal(size=(rows, V + pad[0])) * 4 if x is None else x, dtype)
    v = full[:, :V]
    hist = ids = bias = mask = None
    keep = {}
    if H:
        hist = history if history is not None else (rng.random((groups, H)) ** 3 * V * 1.02).astype(np.uint32)
        n = rng.integers(0, H + 3, groups) if lengths else np.full(groups, H)
        pen = np.stack([rng.uniform(0.5, 2, groups), rng.uniform(-1, 1, groups), rng.uniform(-1, 1, groups)], 1).astype(np.float32)
        keep.update(history=dev(lib, hist), penalties=dev(lib, pen), history_lengths=dev(lib, n.astype(np.uint32)) if lengths else None)
        hist = [h[:min(int(k), H)] for h, k in zip(hist, n)]
    if B:
        ids = biases if biases is not None else rng.integers(0, V + 5, (groups, B)).astype(np.uint32)
        bias = (rng.normal(size=(groups, B)) * 5).astype(np.float32)
        n = rng.integers(0, B + 3, groups) if lengths else np.full(groups, B)
        keep.update(bias_ids=dev(lib, ids), biases=dev(lib, bias), bias_lengths=dev(lib, n.astype(np.uint32)) if lengths else None)
        ids = [list(zip(i[:min(int(k), B)].tolist(), b.tolist())) for i, b, k in zip(ids, bias, n)]
    words = (V + 31) // 32 + mask_pad
    if masked:
        mask = rng.random((mgroups, V)) < 0.4
        mask[0] = False  # a grammar with no way on
        keep.update(mask=dev(lib, bits(mask, words)))
    p = lib.Logits(rows=rows, vocabulary=V, dtype=CODE[dtype], history_stride=H, bias_stride=B, mask_stride=words if mask_pad else 0,
                   group=0 if group == 1 else group, mask_group=0 if mask_group == 1 else mask_group, stride=V + pad[0] if pad[0] else 0,
                   out_stride=(V + pad[0] if in_place else V + pad[1]) if (pad[0] if in_place else pad[1]) else 0)
    buf = dev(lib, raw)
    if in_place:
        lib.logits_adjust(buf, buf, p, stream=stream, **keep)
        lib.synchronize(stream)
        got = values(buf.download(np.uint8), dtype, full.shape)
        np.testing.assert_array_equal(got[:, V:], full[:, V:])
        got = got[:, :V]
    else:
        out = Guarded(lib, rows * (V + pad[1]) * SIZE[dtype])
        lib.logits_adjust(buf, out.ptr, p, stream=stream, **keep)
        lib.synchronize(stream)
        got = values(out.read(np.uint8)[:rows * (V + pad[1]) * SIZE[dtype]], dtype, (rows, V + pad[1]))[:, :V]
    want, mag = adjusted(v, hist, pen if H else None, ids, mask, group, mask_group)
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite])
    # five roundings in f32 (the quotient or product, the count's product, two differences, the bias), then the type's
    with np.errstate(all="ignore"):
        tol = 5 * U * 1.01 * mag + HALF[dtype] * np.abs(want) * (1 + 2.0 ** -10) + LEAST[dtype]
        bad = finite & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])
    touched = np.zeros(want.shape, bool)
    touched |= want != v
    np.testing.assert_array_equal(got[~touched & finite], v[~touched & finite])
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [1, 7, 8, 31, 33, 4095, 4096, 4097, 16385, 50001])
def test_vocabularies(lib, dtype, V):
    rng = np.random.default_rng(V)
    run(lib, rng, 3, V, dtype, H=50, B=9, masked=True)
    run(lib, rng, 2, V, dtype, H=50)
    run(lib, rng, 2, V, dtype, B=4)
    run(lib, rng, 2, V, dtype, masked=True)
    run(lib, rng, 1, V, dtype)


@pytest.mark.parametrize("H", [1, 64, 1000, 5000, 40000])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_histories(lib, H, rows):
    if rows * H > 400000:
        rows = 9
    rng = np.random.default_rng(H + rows)
    run(lib, rng, rows, 30011, "f32", H=H, B=3, lengths=rows != 3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_groups_strides_in_place(lib, dtype):
    rng = np.random.default_rng(5)
    run(lib, rng, 10, 9001, dtype, H=33, B=5, masked=True, group=4, mask_group=3, pad=(3, 5), mask_pad=2)
    run(lib, rng, 10, 9001, dtype, H=33, B=5, masked=True, group=20, mask_group=1, pad=(7, 0), in_place=True)
    run(lib, rng, 6, 9001, dtype, H=33, B=5, masked=True, group=1, mask_group=6, in_place=True)


def test_one_word_again_and_again(lib):
    """The same id all over the history and the biases: the count, and the last bias."""
    rng = np.random.default_rng(6)
    H, B = 0xFFFFF // 64, 4095
    run(lib, rng, 2, 5000, H=H, B=B, lengths=False, history=np.full((2, H), 4321, np.uint32), biases=np.full((2, B), 4321, np.uint32))
    run(lib, rng, 1, 200, H=0xFFFFF, lengths=False, history=np.full((1, 0xFFFFF), 199, np.uint32))


def test_ids_past_the_vocabulary(lib):
    rng = np.random.default_rng(7)
    for V in (4096, 4100, 10):
        far = np.array([[V, V + 1, 0xFFFFFFFF, 0x80000000, V - 1, 4096 + V]], np.uint32)
        run(lib, rng, 1, V, H=6, B=6, lengths=False, history=far, biases=far)


def test_not_finite(lib):
    """A NaN stays unless the mask hides it, infinities stay infinities, hidden words are -Inf whatever they were."""
    rng = np.random.default_rng(8)
    for dtype in ("f32", "bf16", "f16"):
        x = rng.normal(size=(2, 1000))
        x[:, 0:1000:7], x[:, 1:1000:7], x[:, 2:1000:7] = np.nan, np.inf, -np.inf
        every = np.tile(np.arange(1000, dtype=np.uint32), (2, 1))
        run(lib, rng, 2, 1000, dtype, H=1000, B=20, masked=True, lengths=False, x=x, history=every)


def test_hidden_then_chosen(lib):
    """The token that argmax_f32 and draft_verify take from an adjusted row is one that the mask leaves."""
    rng = np.random.default_rng(9)
    V = 20000
    x = rng.normal(size=(1, V)).astype(np.float32)
    x[0, 77] = 50.0
    mask = np.zeros((1, V), bool)
    mask[0, [5, 600, 19999]] = True
    buf, m, out = dev(lib, x), dev(lib, bits(mask, (V + 31) // 32)), lib.DeviceBuffer(V * 4)
    lib.logits_adjust(buf, out, lib.Logits(rows=1, vocabulary=V), mask=m)
    tok, acc, prob = lib.DeviceBuffer(4), lib.DeviceBuffer(4), lib.DeviceBuffer(4)
    p = lib.Draft(sequences=1, drafts=0, vocabulary=V, temperature=0.0)
    need = lib.draft_verify_workspace(p)
    lib.draft_verify(out, None, None, None, acc, tok, p, probabilities=prob, workspace=lib.DeviceBuffer(need), workspace_bytes=need)
    lib.synchronize()
    best = [5, 600, 19999][int(np.argmax(x[0, [5, 600, 19999]]))]
    assert tok.download(np.uint32)[0] == best
