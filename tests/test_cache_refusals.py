"""Arguments that the rotation, the paged cache, its attention and the adjustment of logits refuse, before any GPU work (the
pointers are never read); page and workspace sizes; frequencies, which the host computes."""
import ctypes

import numpy as np
import pytest

import oco_amd as oco

FAKE = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1008)


def refused(rc, word, code=1):
    message = oco.load_library().oco_last_error().decode()
    assert rc == code, (rc, message)
    assert word in message, message


def cache(**over):
    d = dict(head_dim=128, heads=8, kv_heads=2, page_size=64, pages=10, sequences=2, rows=4, max_rows=2, max_length=500, table_stride=8, dtype=1)
    d.update(over)
    return oco.Cache(**d)


BAD = [(dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(heads=7), "multiple of kv_heads"), (dict(kv_heads=0), "kv_heads"),
       (dict(heads=65536 * 2), "under 65536"), (dict(page_size=0), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=65552), "page_size"),
       (dict(pages=0), "no pages"), (dict(max_length=513), "max_length"), (dict(max_length=1 << 30, table_stride=1 << 30), "max_length"),
       (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q_stride=1023), "stride"),
       (dict(out_stride=5), "stride"), (dict(k_stride=255), "stride"), (dict(v_stride=255), "stride")]


def rotation(**over):
    d = dict(dim=128, layout=0, magnitude=1.0, frequencies=0x1000)
    d.update(over)
    return oco.Rotation(**d)


def append(p, pages=FAKE, table=FAKE, starts=FAKE, lengths=FAKE, q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, r=None):
    return oco.load_library().oco_cache_append(pages, table, starts, lengths, None, q, k, v, q_out, ctypes.byref(r) if r else None,
                                               ctypes.byref(p) if p else None, None)


def read(p, pages=FAKE, table=FAKE, starts=FAKE, lengths=FAKE, k=FAKE, v=FAKE):
    return oco.load_library().oco_cache_read(pages, table, starts, lengths, k, v, ctypes.byref(p) if p else None, None)


def attention(p, q=FAKE, pages=FAKE, table=FAKE, starts=FAKE, lengths=FAKE, out=FAKE, work=FAKE, bytes_=1 << 40):
    return oco.load_library().oco_cache_attention(q, pages, table, starts, lengths, None, out, ctypes.byref(p) if p else None, work, bytes_, None)


@pytest.mark.parametrize("call", [append, read, attention])
def test_cache(call):
    for over, word in BAD:
        refused(call(cache(**over)), word)
        assert oco.cache_attention_workspace(cache(**over)) == 0
        if set(over) & {"head_dim", "kv_heads", "page_size"}:
            assert oco.cache_page_bytes(cache(**over)) == 0
    refused(call(None), "null description")
    for missing in ("pages", "table", "lengths") + (("q", "out") if call is attention else ("k", "v")):
        refused(call(cache(), **{missing: None}), "null pointer")
    refused(call(cache(), pages=ODD), "16-byte")
    refused(call(cache(dtype=3)), "type 3", 2)
    refused(call(cache(rows=5), starts=None), "5 rows of 2")
    for over in (dict(rows=0), dict(sequences=0), dict(max_rows=0)):
        assert call(cache(**over), pages=None) == 0
    assert oco.cache_page_bytes(cache()) == 2 * 64 * (128 + 8)
    assert oco.cache_page_bytes(cache(head_dim=64, page_size=16)) == 2 * 16 * (64 + 4)


def test_append():
    refused(append(cache(), q_out=None), "null pointer")
    refused(append(cache(q_stride=2000)), "in place")
    for over, word in ((dict(dim=63), "odd"), (dict(dim=130), "past the head"), (dict(layout=2), "layout"), (dict(frequencies=None), "frequencies")):
        refused(append(cache(), r=rotation(**over)), word)


def test_attention():
    refused(attention(cache(dtype=0)), "type 0", 2)
    refused(attention(cache(heads=0)), "no heads")
    refused(attention(cache(rows=1 << 30)), "too many rows")
    refused(attention(cache(sequences=1 << 31)), "too many rows")
    refused(attention(cache(q_stride=2000)), "in place")
    refused(attention(cache(out_stride=1032)), "in place")
    p = cache(sequences=1, rows=1, max_rows=1, max_length=100000, table_stride=2000)
    need = oco.cache_attention_workspace(p)
    assert need > 0 and need % 16 == 0
    refused(attention(p, bytes_=need - 1), "workspace")
    refused(attention(p, work=None), "workspace")
    refused(attention(p, work=ODD), "workspace")
    assert oco.cache_attention_workspace(cache(max_length=10)) == 0


def test_pool_in_a_buffer_that_is_too_small():
    class Small:
        nbytes = 10 * 2 * 64 * (128 + 8) - 1
    with pytest.raises(ValueError, match="for 10 pages"):
        oco.PagedCache(10, 128, 2, 64, buffer=Small())
    with pytest.raises(ValueError, match="no cache"):
        oco.PagedCache(10, 96, 2, 64, buffer=Small())


def test_rotate():
    L = oco.load_library()

    def call(x=FAKE, dt=1, rows=4, heads=2, d=128, xs=0, pos=FAKE, out=ODD, os=0, r=None):
        return L.oco_rotate(x, dt, rows, heads, d, xs, pos, out, os, ctypes.byref(r or rotation()), None)
    refused(L.oco_rotate(FAKE, 1, 4, 2, 128, 0, FAKE, FAKE, 0, None, None), "null rotation")
    for over, word in ((dict(dim=63), "odd"), (dict(dim=130), "past the head"), (dict(layout=2), "layout"), (dict(frequencies=None), "frequencies")):
        refused(call(r=rotation(**over)), word)
    refused(call(d=2048, r=rotation(dim=1026)), "dim")
    for missing in ("x", "pos", "out"):
        refused(call(**{missing: None}), "null pointer")
    refused(call(xs=255), "stride")
    refused(call(os=255), "stride")
    refused(call(out=FAKE, xs=300), "in place")
    refused(call(dt=3), "type 3", 2)
    refused(call(heads=1 << 30), "rows of")
    assert call(rows=0, x=None) == 0 and call(heads=0, x=None) == 0


def test_logits():
    L = oco.load_library()

    def call(x=FAKE, out=ODD, history=FAKE, penalties=FAKE, ids=FAKE, biases=FAKE, mask=FAKE, **over):
        d = dict(rows=2, vocabulary=1000, dtype=0, history_stride=10, bias_stride=3)
        d.update(over)
        return L.oco_logits_adjust(x, out, history, None, penalties, ids, biases, None, mask, ctypes.byref(oco.Logits(**d)), None)
    refused(call(vocabulary=1 << 31), "vocabulary")
    refused(call(history_stride=1 << 20), "history")
    refused(call(bias_stride=4096), "biases")
    refused(call(mask_stride=31), "mask stride")
    refused(call(stride=999), "stride")
    refused(call(out_stride=999), "stride")
    refused(call(dtype=3), "type 3", 2)
    for missing in ("x", "out", "penalties", "biases"):
        refused(call(**{missing: None}), "null pointer")
    refused(call(out=FAKE, stride=1001), "in place")
    refused(call(rows=1 << 31, vocabulary=1 << 20), "rows")
    refused(L.oco_logits_adjust(*[FAKE] * 9, None, None), "null description")
    assert call(rows=0, x=None) == 0 and call(vocabulary=0, x=None) == 0


def test_frequencies():
    """Each scaling by its definition, written out pair by pair."""
    dim, base = 64, 500000.0
    plain = np.array([base ** (-2.0 * j / dim) for j in range(dim // 2)])
    f, m = oco.rotation_frequencies(dim, base)
    np.testing.assert_allclose(f, plain, rtol=1e-14)
    assert m == 1.0
    f, m = oco.rotation_frequencies(dim, base, oco.Scaling.LINEAR, factor=4.0)
    np.testing.assert_allclose(f, plain / 4, rtol=1e-14)
    extra = np.linspace(1, 9, dim // 2).astype(np.float32)
    np.testing.assert_allclose(oco.rotation_frequencies(dim, base, factors=extra)[0], plain / extra.astype(np.float64), rtol=1e-14)
    # by the number of turns over the original context: untouched from `fast` on, divided up to `slow`
    f, m = oco.rotation_frequencies(dim, base, oco.Scaling.BANDS, factor=8.0, original=8192.0, fast=4.0, slow=1.0)
    for j, g in enumerate(f):
        turns = 8192.0 * plain[j] / (2 * np.pi)
        keep = min(max((turns - 1.0) / 3.0, 0.0), 1.0)
        assert abs(g - plain[j] * (keep + (1 - keep) / 8)) <= 1e-14 * plain[j]
    assert m == 1.0
    # by the pair's index between the pairs that turn 32 times and once
    f, m = oco.rotation_frequencies(dim, base, oco.Scaling.YARN, factor=8.0, original=4096.0)
    low = np.floor(dim * np.log(4096.0 / (32 * 2 * np.pi)) / (2 * np.log(base)))
    high = np.ceil(dim * np.log(4096.0 / (2 * np.pi)) / (2 * np.log(base)))
    for j, g in enumerate(f):
        divided = min(max((j - low) / (high - low), 0.0), 1.0)
        assert abs(g - plain[j] * (divided / 8 + 1 - divided)) <= 1e-14 * plain[j]
    assert abs(m - (0.1 * np.log(8.0) + 1)) < 1e-15
    assert oco.rotation_frequencies(0)[0].size == 0


def test_frequencies_refused():
    for args, word in ((dict(dim=63), "odd"), (dict(dim=1026), "odd or past"), (dict(dim=64, scaling=4), "scaling 4"), (dict(dim=64, base=1.0), "base"),
                       (dict(dim=64, base=float("nan")), "base"), (dict(dim=64, scaling=1, factor=0.5), "factor"),
                       (dict(dim=64, scaling=2, factor=2.0), "original"), (dict(dim=64, scaling=3, factor=2.0, original=10.0, fast=1.0, slow=1.0), "fast"),
                       (dict(dim=64, factors=np.zeros(32)), "factor of pair 0")):
        with pytest.raises(oco.OcoError, match=word):
            oco.rotation_frequencies(**args)
    with pytest.raises(ValueError):
        oco.rotation_frequencies(64, factors=np.ones(31))
