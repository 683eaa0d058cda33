"""oco_cache_attention against softmax attention in 64 bits over the values that the pages stand for."""
import numpy as np
import pytest

from _cache import Batch, Pool, dequantize, quantize
from _ops import CODE, HALF, LEAST, SIZE, dev, stored, values
from _util import Guarded, say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(params=[0, 8, 16], ids=["", "prompt", "long"])
def kernel(request, lib):
    """The kernel that the rule takes, and the two of prompts (which heads of 256 do not have)."""
    with lib.overridden(lib.Knob.ATTENTION, (request.param,)):
        yield request.param


class Case:
    def __init__(self, lib, rng, rows, lengths, heads, kv, d, P, dtype, window=0, sinks=False, extra_rows=0, pad=(0, 0), q_scale=2.0, scale=0.0,
                 holes=0, max_rows=None, v_scale=1.0):
        self.lib, self.dtype, self.heads, self.kv, self.d, self.window = lib, dtype, heads, kv, d, window
        b = self.b = Batch(rng, rows, lengths, P, extra_rows=extra_rows)
        self.scale = scale or 1 / np.sqrt(d)
        self.k, self.v, pool = [], [], Pool(b.pages, kv, P, d)
        for s, n in enumerate(lengths):
            k, v = rng.normal(size=(n, kv, d)), rng.normal(size=(n, kv, d)) * v_scale + 0.3
            for _ in range(holes if n else 0):  # blocks of NaN among the tokens
                (k if rng.random() < 0.5 else v)[rng.integers(0, n), rng.integers(0, kv), rng.integers(0, d)] = np.nan
            ck, cv = quantize(k), quantize(v)
            for t in range(n):
                page, slot = b.place(s, t)
                for j in range(kv):
                    pool.put(page, slot, j, (ck[0][t, j], ck[1][t, j]), (cv[0][t, j], cv[1][t, j]))
            self.k.append(dequantize(*ck))
            self.v.append(dequantize(*cv))
        self.pool = pool
        self.q_stride, self.out_stride = heads * d + pad[0], heads * d + pad[1]
        raw, q = stored(rng.normal(size=(b.total, self.q_stride)) * q_scale, dtype)
        self.q = q[:, :heads * d].reshape(b.total, heads, d)
        self.sinks = (rng.normal(size=heads) * 2).astype(np.float32) if sinks else None
        self.p = b.describe(lib, heads, kv, d, CODE[dtype], window=window, scale=scale, q_stride=self.q_stride if pad[0] else 0,
                            out_stride=self.out_stride if pad[1] else 0, **({} if max_rows is None else {"max_rows": max_rows}))
        self.dev = [dev(lib, raw), dev(lib, pool.bytes), dev(lib, b.table), dev(lib, np.array(lengths, np.uint32)), dev(lib, b.starts),
                    dev(lib, self.sinks) if sinks else None]
        self.out = Guarded(lib, b.total * self.out_stride * SIZE[dtype])
        self.need = lib.cache_attention_workspace(self.p)
        self.work = Guarded(lib, self.need)

    def call(self, stream=None, starts=True):
        q, cache, table, lengths, st, sinks = self.dev
        self.lib.cache_attention(q, cache, table, lengths, self.out.ptr, self.p, starts=st if starts else None, sinks=sinks,
                                 workspace=self.work.ptr if self.need else None, workspace_bytes=self.need, stream=stream)

    def want(self, b=None):
        """The rows, and how far off they may be."""
        b = b or self.b
        out, tol = np.zeros(self.q.shape), np.zeros(self.q.shape)
        g = self.heads // self.kv
        for s, (n, length) in enumerate(zip(b.rows, b.lengths)):
            for i in range(n):
                r, at = int(b.starts[s]) + i, length - n + i
                lo = max(0, at + 1 - self.window) if self.window else 0
                for h in range(self.heads):
                    if at < 0:
                        continue
                    q, k, v = self.q[r, h], self.k[s][lo:at + 1, h // g], self.v[s][lo:at + 1, h // g]
                    with np.errstate(all="ignore"):
                        score, mag = k @ q * self.scale, np.abs(k) @ np.abs(q) * self.scale
                        top = score.max() if self.sinks is None else max(score.max(), float(self.sinks[h]))
                        e = np.exp(score - top)
                        total = e.sum() + (0.0 if self.sinks is None else np.exp(float(self.sinks[h]) - top))
                        out[r, h], a = e @ v / total, e @ np.abs(v) / total
                        # scores: products are exact, d sums in f32, then the factor, the maximum's subtraction and the exponential
                        # (a step each, of numbers up to |score| log2 e and |top| log2 e): a relative error of each e of
                        d = ((self.d + 2) * mag.max() + 4 * (np.abs(score).max() + abs(top)) + 4) * U
                        # of the products' sum and of the total: d each, a step per f32 sum; e rounds to the 16-bit type (its
                        # subnormal numbers in f16: half of 2^-24 each, where the largest e is 1 or more); the result rounds
                        m = len(score) + 16
                        tol[r, h] = a * (HALF[self.dtype] + 2 * d + 2 * m * U) + HALF[self.dtype] * np.abs(out[r, h]) * (1 + U) + LEAST[self.dtype]
                        if self.dtype == "f16":
                            tol[r, h] += 2.0 ** -25 * np.abs(v).sum(0) / total
        return out, tol

    def check(self, b=None):
        want, tol = self.want(b)
        z = SIZE[self.dtype]
        raw = self.out.read(np.uint8)[:self.b.total * self.out_stride * z]
        self.work.read(np.uint8)
        n = int(self.b.starts[-1])
        got = values(raw, self.dtype, (self.b.total, self.out_stride))[:n, :self.heads * self.d].reshape(n, self.heads, self.d)
        want, tol = want[:n], tol[:n]
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        fine = ~np.isnan(want)
        bad = np.abs(got - want)[fine] > tol[fine]
        assert not bad.any(), (int(bad.sum()), got[fine][bad][:4], want[fine][bad][:4])
        return got


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,lengths", [([1], [1]), ([1], [2]), ([1, 1, 1, 1], [15, 16, 17, 33]), ([1, 1], [500, 1300]), ([3, 0, 5], [40, 7, 300]),
                                          ([4], [4]), ([40, 1], [90, 260])])
def test_lengths(kernel, lib, dtype, d, rows, lengths):
    rng = np.random.default_rng(d + sum(lengths))
    say("attention", dtype, d, rows, lengths)
    c = Case(lib, rng, rows, lengths, 4, 2, d, 16, dtype)
    c.call()
    lib.synchronize()
    c.check()


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (14, 2), (16, 1), (17, 1), (32, 1), (40, 8), (72, 2)])
@pytest.mark.parametrize("rows", [1, 3])
def test_heads(kernel, lib, heads, kv, rows):
    """Groups of one head to more than a tile of rows."""
    rng = np.random.default_rng(heads * 10 + rows)
    say("attention", heads, kv, rows)
    c = Case(lib, rng, [rows, rows], [70, 133], heads, kv, 64, 48, "bf16")
    c.call()
    lib.synchronize()
    c.check()


@pytest.mark.parametrize("P", [16, 32, 48, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 16, 31, 100, 5000])
def test_windows_and_pages(kernel, lib, P, window):
    rng = np.random.default_rng(P + window)
    say("attention", P, window)
    for rows, lengths in (([1, 4, 2], [333, 64, 1]), ([65, 20], [200, 20])):
        c = Case(lib, rng, rows, lengths, 8, 2, 64, P, "bf16", window=window)
        c.call()
        lib.synchronize()
        c.check()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,lengths", [([1, 1], [50, 2100]), ([6, 3], [6, 700]), ([80], [160])])
def test_sinks(kernel, lib, dtype, rows, lengths):
    rng = np.random.default_rng(7)
    say("sinks", dtype, rows)
    c = Case(lib, rng, rows, lengths, 6, 2, 128, 64, dtype, sinks=True, q_scale=0.5)
    c.sinks[0], c.sinks[1] = -np.inf, 60.0
    c.dev[5].upload(c.sinks)
    c.call()
    lib.synchronize()
    c.check()


@pytest.mark.parametrize("sinks", [False, True])
def test_rows_that_see_nothing(kernel, lib, sinks):
    """Sequences without tokens, and with fewer tokens than rows: zeros; rows behind the last sequence stay."""
    rng = np.random.default_rng(2)
    for rows, lengths in (([1, 2, 5], [0, 0, 3]), ([90, 40], [30, 0])):
        c = Case(lib, rng, rows, lengths, 4, 2, 128, 16, "bf16", sinks=sinks, extra_rows=4)
        say("nothing seen", rows, lengths)
        c.call()
        lib.synchronize()
        got = c.check()
        assert not got[0].any()
        tail = c.out.read(np.uint8).reshape(c.b.total, -1)[sum(rows):]
        assert np.all(np.ascontiguousarray(tail).reshape(-1).view(np.uint32) == 0x7FC12345)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,lengths,window", [([1, 8], [300, 40], 0), ([4, 3], [60, 200], 24), ([70, 33], [140, 33], 0), ([100], [150], 40)])
def test_blocks_of_nan(kernel, lib, dtype, d, rows, lengths, window):
    """A NaN reaches the rows that see it, a value's in its own 32 columns, and no other row: not those before it, not those
    whose window has passed it."""
    rng = np.random.default_rng(d + sum(rows))
    say("nan", dtype, d, rows, lengths, window)
    c = Case(lib, rng, rows, lengths, 4, 2, d, 32, dtype, window=window, holes=3)
    c.call()
    lib.synchronize()
    c.check()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [5, 60])
def test_nan_in_the_last_token(kernel, lib, d, rows):
    """Only the last row sees it: a value's NaN its block of columns, a key's all of them."""
    rng = np.random.default_rng(d)
    for in_key in (False, True):
        c = Case(lib, rng, [rows], [200], 4, 2, d, 16, "bf16")
        page, slot = c.b.place(0, 199)
        at = 16 * d + (slot * (d // 32) + 1 if in_key else 16 * (d // 32) + slot // 4 * (d // 8) + 4 + slot % 4)
        c.pool.bytes[page, 1, at] = 255  # block 1 of the second head
        (c.k if in_key else c.v)[0][199, 1, 32:64] = np.nan
        c.dev[1].upload(c.pool.bytes)
        say("last token", d, rows, in_key)
        c.call()
        lib.synchronize()
        got = np.isnan(c.check())
        want = np.zeros(got.shape, bool)
        want[-1, 2:, slice(None) if in_key else slice(32, 64)] = True
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_pages_of_anything(kernel, lib, dtype):
    """Memory that no token was written to, behind the last token and in pages of nobody, whatever it holds."""
    rng = np.random.default_rng(21)
    for rows, lengths in (([1, 3], [37, 70]), ([45], [75])):
        for fill in (0xFD, 0xFE, 0x8D, 0xC8, 0x00, None):
            c = Case(lib, rng, rows, lengths, 4, 2, 128, 32, dtype, window=50)
            empty = np.ones(c.pool.bytes.shape, bool)
            for s, n in enumerate(lengths):  # a pool that marks what the tokens take
                for t in range(n):
                    page, slot = c.b.place(s, t)
                    mark = Pool(1, 1, 32, 128)
                    mark.bytes[:] = 0
                    one = (np.full(128, 15, np.uint8), np.full(4, 255, np.uint8))
                    mark.put(0, slot, 0, one, one)
                    empty[page] &= mark.bytes[0] == 0
            noise = rng.integers(0, 256, empty.shape).astype(np.uint8) if fill is None else np.full(empty.shape, fill, np.uint8)
            c.dev[1].upload(np.where(empty, noise, c.pool.bytes))
            say("anything", dtype, rows, fill)
            c.call()
            lib.synchronize()
            got = c.check()
            assert not np.isnan(got).any()


def test_blocks_past_f16(kernel, lib):
    """In f16 a block that the type cannot hold is NaN to the rows that see it, and to no other."""
    rng = np.random.default_rng(22)
    for rows in ([3], [45]):
        c = Case(lib, rng, rows, [90], 4, 2, 64, 16, "f16")
        for at, (what, t, scale) in enumerate((("v", 89, 141), ("k", 89, 200), ("v", 88, 252))):
            if what == "k" and rows == [3]:
                continue
            page, slot = c.b.place(0, t)
            c.pool.bytes[page, at % 2, 16 * 64 + (slot * 2 if what == "k" else 32 + slot // 4 * 8 + slot % 4)] = scale
            (c.k if what == "k" else c.v)[0][t, at % 2, :32] = np.nan
        c.dev[1].upload(c.pool.bytes)
        say("past f16", rows)
        c.call()
        lib.synchronize()
        got = c.check()
        assert np.isnan(got[-1]).any() and not np.isnan(got[-3]).any()


def test_sinks_that_are_nan(kernel, lib):
    rng = np.random.default_rng(23)
    for rows, lengths in (([1], [3000]), ([40], [60])):
        c = Case(lib, rng, rows, lengths, 4, 2, 64, 16, "bf16", sinks=True)
        c.sinks[2] = np.nan
        c.dev[5].upload(c.sinks)
        say("nan sink", rows)
        c.call()
        lib.synchronize()
        c.sinks[2] = 0.0
        raw = values(c.out.read(np.uint8), "bf16", c.q.shape)
        assert np.isnan(raw[:, 2]).all() and not np.isnan(raw[:, [0, 1, 3]]).any()


@pytest.mark.parametrize("rows,lengths", [([1, 2], [2000, 30]), ([60], [100]), ([6], [1500])])
def test_in_the_place_of_the_queries(kernel, lib, rows, lengths):
    rng = np.random.default_rng(24)
    c = Case(lib, rng, rows, lengths, 8, 2, 128, 32, "bf16", sinks=True)
    c.call()
    q, cache, table, lens, starts, sinks = c.dev
    say("in place", rows)
    lib.cache_attention(q, cache, table, lens, q, c.p, starts=starts, sinks=sinks, workspace=c.work.ptr if c.need else None, workspace_bytes=c.need)
    lib.synchronize()
    np.testing.assert_array_equal(q.download(np.uint8), c.out.read(np.uint8))


def test_pages_outside_the_pool(kernel, lib):
    """They read as NaN where a row sees them, and nothing is read there."""
    rng = np.random.default_rng(12)
    for rows, lengths in (([1, 1], [100, 60]), ([40, 3], [100, 60])):
        c = Case(lib, rng, rows, lengths, 4, 2, 128, 16, "bf16", window=30)
        c.b.table[0, 1], c.b.table[0, 5], c.b.table[1, 3] = 0xFFFFFFFF, c.b.pages, 0x7FFFFFFF
        c.dev[2].upload(c.b.table)
        for s, page in ((0, 1), (0, 5), (1, 3)):
            c.k[s][page * 16:page * 16 + 16] = np.nan
        say("bad pages", rows)
        c.call()
        lib.synchronize()
        c.check()


@pytest.mark.parametrize("rows,lengths", [([2, 2, 2], [90, 5, 400]), ([30, 30], [30, 77])])
def test_strides_and_no_starts(kernel, lib, rows, lengths):
    rng = np.random.default_rng(5)
    c = Case(lib, rng, rows, lengths, 6, 2, 64, 32, "f16", pad=(6, 10), scale=0.2)
    say("strides", rows)
    c.call(starts=False)
    lib.synchronize()
    c.check()
    raw = c.out.read(np.uint8)[:c.b.total * c.out_stride * 2].view(np.uint16).reshape(c.b.total, c.out_stride)
    guard = np.tile(np.array([0x2345, 0x7FC1], np.uint16), c.out_stride * c.b.total // 2 + 1)[:raw.size].reshape(raw.shape)
    np.testing.assert_array_equal(raw[:, 6 * 64:], guard[:, 6 * 64:])


@pytest.mark.parametrize("rows", [[1], [130]])
def test_scores_that_rise_and_fall(kernel, lib, rows):
    """Maxima that come early, late and in between, scores over a range of hundreds."""
    rng = np.random.default_rng(6)
    for order in (1, -1, 0):
        c = Case(lib, rng, rows, [2000], 4, 1, 128, 64, "bf16", q_scale=30.0)
        pool = Pool(c.b.pages, 1, 64, 128)
        ramp = np.linspace(0.01, 1, 2000)[::order] if order else rng.random(2000)
        k = rng.normal(size=(1, 128)) * 0.1 + ramp[:, None] * np.sign(c.q[0, 0])[None]
        k, v = quantize(k), quantize(rng.normal(size=(2000, 128)))
        for t in range(2000):
            page, slot = c.b.place(0, t)
            pool.put(page, slot, 0, (k[0][t], k[1][t]), (v[0][t], v[1][t]))
        c.k[0], c.v[0] = dequantize(*k)[:, None], dequantize(*v)[:, None]
        c.dev[1].upload(pool.bytes)
        say("ramp", rows, order)
        c.call()
        lib.synchronize()
        c.check()


def test_infinite_queries(kernel, lib):
    """An infinity or a NaN in a query makes its own row NaN and no other."""
    rng = np.random.default_rng(15)
    for rows in ([3], [50]):
        c = Case(lib, rng, rows, [120], 4, 2, 64, 16, "bf16")
        raw = c.dev[0].download(np.uint16).reshape(c.b.total, 4, 64)
        raw[0, 1, 5], raw[1, 3, 2] = 0x7F80, 0x7FC0
        c.dev[0].upload(raw)
        c.q[0, 1, 5], c.q[1, 3, 2] = np.inf, np.nan
        say("infinite", rows)
        c.call()
        lib.synchronize()
        got = c.check()
        bad = np.isnan(got).any(-1)
        assert bad.sum() == 2 and bad[0, 1] and bad[1, 3]


@pytest.mark.parametrize("dtype,v_scale", [("bf16", 2.0 ** 100), ("bf16", 2.0 ** -100), ("f16", 2.0 ** 11), ("f16", 2.0 ** -11)])
def test_large_and_small_values(kernel, lib, dtype, v_scale):
    rng = np.random.default_rng(16)
    for rows in ([2], [40]):
        c = Case(lib, rng, rows, [150], 4, 2, 128, 32, dtype, v_scale=v_scale)
        say("range", dtype, v_scale, rows)
        c.call()
        lib.synchronize()
        c.check()


def test_shorter_bounds(kernel, lib):
    """Lengths past max_length count as max_length; rows past max_rows stay."""
    rng = np.random.default_rng(17)
    c = Case(lib, rng, [3, 6], [50, 80], 4, 2, 64, 16, "bf16", max_rows=4)
    c.p.max_length = 64
    c.need = lib.cache_attention_workspace(c.p)
    say("bounds")
    c.call()
    lib.synchronize()
    raw = c.out.read(np.uint8).reshape(c.b.total, -1)
    assert np.all(np.ascontiguousarray(raw[7:]).reshape(-1).view(np.uint32) == 0x7FC12345)
    c.b.rows[1], c.b.lengths[1] = 4, 64
    want, tol = c.want()
    got = values(raw[:7], "bf16", (7, 4, 64))
    assert np.all(np.abs(got - want[:7]) <= tol[:7])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tile", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("chunk", [0, 128, 384])
def test_every_kernel_and_chunk(lib, d, tile, chunk):
    """Each kernel on few and many rows, whole and in chunks, with windows that begin inside a step."""
    rng = np.random.default_rng(d + tile + chunk)
    with lib.overridden(lib.Knob.ATTENTION, (tile, chunk)):
        for rows, lengths, window in (([1, 3], [5, 700], 0), ([45, 7], [900, 450], 0), ([45, 70], [900, 450], 333), ([30], [30], 0)):
            say("kernel", d, tile, chunk, rows, lengths, window)
            c = Case(lib, rng, rows, lengths, 8, 2, d, 48, "bf16", window=window, sinks=True, holes=1)
            c.call()
            lib.synchronize()
            c.check()


def test_same_result_every_time(kernel, lib):
    rng = np.random.default_rng(18)
    for rows, lengths in (([1, 1], [3000, 10]), ([200], [700])):
        c = Case(lib, rng, rows, lengths, 8, 2, 128, 64, "bf16")
        first = None
        for _ in range(3):
            c.call()
            lib.synchronize()
            raw = c.out.read(np.uint8).copy()
            first = raw if first is None else first
            np.testing.assert_array_equal(raw, first)


def test_a_cache_past_32_bits(kernel, lib):
    """Pages whose byte offsets pass 2^32."""
    rng = np.random.default_rng(19)
    for rows in ([1], [40]):
        c = Case(lib, rng, rows, [100], 4, 2, 128, 16, "bf16")
        page = int(lib.cache_page_bytes(c.p))
        far = (1 << 32) // page + 5
        big = lib.DeviceBuffer((far + c.b.pages) * page)
        big.upload(c.pool.bytes, far * page)
        c.p.pages = far + c.b.pages
        c.b.table[0, :7] += far
        c.dev[1] = big
        c.dev[2].upload(c.b.table)
        say("far pages", rows, far)
        c.call()
        lib.synchronize()
        c.check()
        big.free()


@pytest.mark.parametrize("d,rows,window", [(64, 8, 0), (64, 1, 700), (128, 16, 0), (256, 3, 0), (64, 2, 1500), (128, 24, 0)])
@pytest.mark.parametrize("sequences", [1, 3, 20, 64, 65, 200])
def test_chunks_by_the_lengths(lib, d, rows, window, sequences):
    """Bounds far past the lengths, as a captured step has them: chunks follow the lengths, of sequences without rows or tokens too."""
    rng = np.random.default_rng(d + sequences)
    n = [int(i) for i in rng.integers(0 if sequences > 3 else 1, rows + 1, sequences)]
    lengths = [int(i) for i in rng.integers(0, 1500 if sequences < 20 else 300, sequences)]
    c = Case(lib, rng, n, lengths, 4, 2, d, 16, "bf16", window=window, sinks=True, holes=sequences % 2, max_rows=rows)
    c.p.max_length = 100000 // sequences
    stride = c.p.max_length // 16 + 1
    c.p.table_stride = stride
    c.dev[2] = dev(lib, np.ascontiguousarray(np.pad(c.b.table, ((0, 0), (0, stride - c.b.table.shape[1])))))
    c.need = lib.cache_attention_workspace(c.p)
    c.work = Guarded(lib, c.need)
    say("chunks", d, n[:8], lengths[:8])
    c.call()
    lib.synchronize()
    c.check()


@pytest.mark.parametrize("d,rows,heads,kv", [(64, 1, 16, 8), (128, 1, 16, 4), (128, 8, 16, 4), (256, 1, 8, 8), (64, 12, 16, 4), (128, 9, 16, 4)])
@pytest.mark.parametrize("even", [False, True])
def test_long_sequences_in_chunks(lib, d, rows, heads, kv, even):
    """As in chunks of 4096 tokens, each within the roundings of its probabilities and of its result."""
    rng = np.random.default_rng(d + rows + even)
    S, P, longest = 12, 64, 20000
    lengths = np.full(S, longest) if even else rng.integers(rows, longest, S)
    p = lib.Cache(head_dim=d, heads=heads, kv_heads=kv, page_size=P, pages=40, sequences=S, rows=S * rows, max_rows=rows, max_length=longest,
                  table_stride=longest // P + 1, dtype=1)
    pool = rng.integers(0, 256, (40, kv, P * d + P * d // 16), dtype=np.uint8)
    pool[:, :, P * d:] = rng.integers(124, 128, pool[:, :, P * d:].shape)
    buffers = [dev(lib, stored(rng.normal(size=(S * rows, heads * d)), "bf16")[0]), dev(lib, pool), dev(lib, rng.integers(0, 40, (S, p.table_stride)).astype(np.uint32)),
               dev(lib, lengths.astype(np.uint32))]
    got = []
    for knob in ((0, 4096), (0,)):
        with lib.overridden(lib.Knob.ATTENTION, knob):
            need = lib.cache_attention_workspace(p)
            work, out = Guarded(lib, need), Guarded(lib, S * rows * heads * d * 2)
            say("long", d, rows, even, knob)
            lib.cache_attention(buffers[0], buffers[1], buffers[2], buffers[3], out.ptr, p, workspace=work.ptr, workspace_bytes=need)
            lib.synchronize()
            work.read(np.uint8)
            got.append(values(out.read(np.uint8), "bf16", (S * rows, heads, d)))
    # values up to 6 * 2: each side's probabilities round by half a step of bf16, of weights that add up to 1, and its result
    # by half a step of itself; f32 sums of 20000 terms, 2 * 2^-24 a term, and of scores up to about 500
    assert np.isfinite(got[0]).all()
    bound = 12 * (2.0 ** -8 + 20000 * 2.0 ** -23 + 4 * 500 * 2.0 ** -23)
    assert np.abs(got[0] - got[1]).max() <= 2 * bound + 2.0 ** -8 * (np.abs(got[0]).max() + np.abs(got[1]).max())


@pytest.mark.parametrize("d,window", [(64, 0), (128, 50), (256, 0)])
@pytest.mark.parametrize("sequences,most", [(2, 200), (5, 200), (64, 30), (65, 30)])
def test_tiles_of_uneven_batches(kernel, lib, d, window, sequences, most):
    """Some sequences with many tiles, some with one and some with none; rows behind the last one stay."""
    rng = np.random.default_rng(d + sequences)
    rows = [int(most * r ** 3) for r in rng.random(sequences)]
    rows[int(rng.integers(sequences))] = most
    rows[-1] = 0
    lengths = [n + int(rng.integers(0, 90)) for n in rows]
    lengths[0] = max(rows[0] - 3, 0)  # its first rows have no token
    say("uneven", d, rows[:10])
    c = Case(lib, rng, rows, lengths, 4, 1, d, 16, "bf16", window=window, sinks=True, extra_rows=3, holes=1)
    c.call()
    lib.synchronize()
    c.check()
    assert np.all(np.ascontiguousarray(c.out.read(np.uint8)[sum(rows) * 4 * d * 2:]).view(np.uint32) == 0x7FC12345)


@pytest.mark.parametrize("d,heads,rows", [(64, 20, 5), (128, 16, 6), (128, 4, 40), (256, 4, 17)])
@pytest.mark.parametrize("sequences", [2, 7, 40])
def test_chunks_and_tiles_by_the_lengths(lib, d, heads, rows, sequences):
    """As test_chunks_by_the_lengths, where sequences have up to four tiles."""
    rng = np.random.default_rng(d + heads + sequences)
    n = [int(i) for i in rng.integers(0, rows + 1, sequences)]
    n[int(rng.integers(sequences))] = rows
    lengths = [int(i) for i in rng.integers(0, 1500 if sequences < 20 else 200, sequences)]
    c = Case(lib, rng, n, lengths, heads, 2, d, 16, "bf16", sinks=True, holes=sequences % 2, max_rows=rows, extra_rows=1)
    c.p.max_length = 100000 // sequences
    stride = c.p.max_length // 16 + 1
    c.p.table_stride = stride
    c.dev[2] = dev(lib, np.ascontiguousarray(np.pad(c.b.table, ((0, 0), (0, stride - c.b.table.shape[1])))))
    c.need = lib.cache_attention_workspace(c.p)
    c.work = Guarded(lib, c.need)
    say("chunks and tiles", d, heads, n[:8], lengths[:8])
    c.call()
    lib.synchronize()
    c.check()


def test_chunks_in_a_graph(lib):
    """A captured call follows lengths that change between its replays, with eager calls in between."""
    rng = np.random.default_rng(23)
    c = Case(lib, rng, [1, 3, 2, 1, 4], [900, 40, 1400, 7, 300], 4, 2, 64, 16, "bf16", sinks=True)
    c.p.max_length, c.p.table_stride = 40000, 2500
    c.dev[2] = dev(lib, np.ascontiguousarray(np.pad(c.b.table, ((0, 0), (0, 2500 - c.b.table.shape[1])))))
    c.need = lib.cache_attention_workspace(c.p)
    c.work = Guarded(lib, c.need)
    assert c.need
    stream, longest = lib.Stream(), list(c.b.lengths)
    c.call(stream)
    stream.sync()
    graph = lib.Graph(stream, lambda: c.call(stream))
    for turn in range(4):
        say("replay", turn)
        c.b.lengths = [int(rng.integers(n, most + 1)) for n, most in zip(c.b.rows, longest)]
        c.dev[3].upload(np.array(c.b.lengths, np.uint32))
        graph.launch()
        stream.sync()
        got = c.out.read(np.uint8).copy()
        c.check()
        c.call()
        lib.synchronize()
        np.testing.assert_array_equal(got, c.out.read(np.uint8))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,lengths,window", [([40], [6500], 0), ([70, 0, 33], [3500, 10, 3300], 0), ([35], [6000], 4000)])
def test_prompt_chunks_after_long_contexts(lib, d, rows, lengths, window):
    """A chunk of a prompt after a long context, which is split along its tokens."""
    rng = np.random.default_rng(d + sum(rows))
    say("prompt chunks", d, rows, lengths, window)
    c = Case(lib, rng, rows, lengths, 4, 1, d, 32, "bf16", window=window, sinks=True, extra_rows=1)
    assert c.need
    c.call()
    lib.synchronize()
    c.check()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,lengths,window,chunk", [([200], [460], 0, 0), ([130, 0, 150], [330, 5, 500], 0, 0), ([150], [900], 300, 0), ([140], [1500], 0, 256)])
def test_first_step_of_every_wavefront(lib, d, rows, lengths, window, chunk):
    """Tiles of 128 rows, where the third step's keys take the place of the first one's: of a tile's or chunk's tokens the
    first 64 have other keys than all others, so that a wavefront that met them late would give them other weights."""
    rng = np.random.default_rng(d + sum(rows))
    with lib.overridden(lib.Knob.ATTENTION, (8, chunk)):
        c = Case(lib, rng, rows, lengths, 32, 4, d, 16, "bf16", window=window, q_scale=4.0)
        side = np.sign(rng.normal(size=d))
        for s, n in enumerate(lengths):
            k = rng.normal(size=(n, 4, d)) * 0.5 + np.where(np.arange(n) % 256 < 64, 1.0, -1.0)[:, None, None] * side
            v = rng.normal(size=(n, 4, d)) + np.where(np.arange(n) % 256 < 64, 4.0, -4.0)[:, None, None]
            k, v = quantize(k), quantize(v)
            for t in range(n):
                page, slot = c.b.place(s, t)
                for j in range(4):
                    c.pool.put(page, slot, j, (k[0][t, j], k[1][t, j]), (v[0][t, j], v[1][t, j]))
            c.k[s], c.v[s] = dequantize(*k), dequantize(*v)
        c.dev[1].upload(c.pool.bytes)
        first = None
        for _ in range(3):
            say("first step", d, rows, lengths, window, chunk)
            c.call()
            lib.synchronize()
            got = c.check()
            first = got if first is None else first
            np.testing.assert_array_equal(got, first)


@pytest.mark.parametrize("tile,d,rows", [(1, 64, 20), (2, 64, 40), (2, 256, 40), (3, 128, 52), (8, 64, 132), (8, 128, 132), (16, 128, 260)])
def test_rows_of_a_tile_that_is_not_full(lib, tile, d, rows):
    """The lanes without a row take nothing from other rows, which may be written meanwhile where the result takes the queries'
    place: whatever a sequence's first query is, the rows of its last tile have the same bits."""
    rng = np.random.default_rng(d + rows)
    with lib.overridden(lib.Knob.ATTENTION, (tile,)):
        c = Case(lib, rng, [rows], [1200], 2, 2, d, 16, "bf16")
        raw, last, got = c.dev[0].download(np.uint16).reshape(rows, 2 * d), rows // (16 * tile) * 16 * tile, []
        for scale in (0.0, 50.0):
            first = stored(np.random.default_rng(1).normal(size=2 * d) * scale, "bf16")
            raw[0], c.q[0] = first[0].view(np.uint16), first[1].reshape(2, d)
            c.dev[0].upload(raw)
            say("first query", tile, d, scale)
            c.call()
            lib.synchronize()
            got.append(c.check()[last:])
        np.testing.assert_array_equal(*got)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,lengths", [([1, 2], [3000, 2]), ([45, 3], [50, 1]), ([300], [300])])
@pytest.mark.parametrize("sinks", [False, True])
def test_scores_that_are_all_minus_infinity(kernel, lib, d, rows, lengths, sinks):
    """Such a row has no softmax and is NaN, or 0 where a sink takes all the weight; a row that sees nothing is 0 either way."""
    rng = np.random.default_rng(d + sum(rows))
    c = Case(lib, rng, rows, lengths, 4, 2, d, 16, "bf16", sinks=sinks)
    for s, n in enumerate(lengths):  # keys that are positive in column 3
        k = np.abs(c.k[s])
        k[:, :, 3] = 1.0 + (k[:, :, 3] > 1)
        ck, cv = quantize(k), quantize(c.v[s])
        for t in range(n):
            page, slot = c.b.place(s, t)
            for j in range(2):
                c.pool.put(page, slot, j, (ck[0][t, j], ck[1][t, j]), (cv[0][t, j], cv[1][t, j]))
        c.k[s], c.v[s] = dequantize(*ck), dequantize(*cv)
        assert (c.k[s][:, :, 3] > 0).all()
    c.dev[1].upload(c.pool.bytes)
    raw = c.dev[0].download(np.uint16).reshape(c.b.total, 4, d)
    for r in (0, sum(rows) - 1):
        raw[r, 1], raw[r, 1, 3] = 0, 0xFF80
        c.q[r, 1], c.q[r, 1, 3] = 0.0, -np.inf
    c.dev[0].upload(raw)
    say("minus infinity", d, rows, sinks)
    c.call()
    lib.synchronize()
    got = c.check()
    want = np.zeros(got.shape[:2], bool)
    want[0, 1] = want[-1, 1] = not sinks
    np.testing.assert_array_equal(np.isnan(got).all(-1), want)
    if sinks:
        assert not got[0, 1].any() and not got[-1, 1].any()


@pytest.mark.parametrize("sequences,d,group,kv,rows,longest,window",
                         [(2, 64, 8, 2, 2, 45000, 0), (40, 128, 4, 2, 1, 8000, 2100), (20, 128, 8, 2, 3, 5000, 0), (64, 256, 4, 2, 2, 8000, 0), (64, 128, 8, 1, 5, 13000, 0),
                          (65, 64, 8, 1, 2, 4000, 0), (65, 64, 8, 1, 5, 4000, 1500), (200, 128, 4, 1, 1, 8000, 0),  # tiles of 16 rows, four sequences per lane
                          (100, 128, 8, 2, 3, 4096, 0), (130, 256, 8, 1, 3, 6000, 0), (200, 64, 8, 1, 3, 8000, 0), (65, 64, 8, 2, 9, 4000, 0),  # of 32
                          (130, 128, 8, 1, 5, 6000, 0), (200, 64, 8, 2, 5, 8000, 0), (256, 64, 8, 1, 5, 8000, 0)])  # of 48
def test_chunks_are_by_the_lengths(lib, sequences, d, group, kv, rows, longest, window):
    """As the two tests above, at bounds where the tokens are split for certain: the workspace says so, and says that the kernel
    sized the chunks itself. Sequences without rows and without tokens lie among a lane's four."""
    rng = np.random.default_rng(d + sequences + rows)
    n, lengths = rng.integers(1, rows + 1, sequences), rng.integers(rows, 90, sequences)
    for i in rng.integers(0, sequences, min(sequences, 3)):
        n[i], lengths[i] = rows, min(3000, longest - 3)
    if sequences > 4:
        n[1], n[-2], lengths[sequences // 2] = 0, 0, 0
        n[5:13] = [0, rows, 0, 0, 0, 0, 0, rows]
    c = Case(lib, rng, [int(i) for i in n], [int(i) for i in lengths], group * kv, kv, d, 16, "bf16", window=window, sinks=True, holes=sequences % 2, max_rows=rows,
             extra_rows=2)
    c.p.max_length = longest
    stride = c.p.max_length // 16 + 1
    c.p.table_stride = stride
    c.dev[2] = dev(lib, np.ascontiguousarray(np.pad(c.b.table, ((0, 0), (0, stride - c.b.table.shape[1])))))
    c.need = lib.cache_attention_workspace(c.p)
    c.work = Guarded(lib, c.need)
    say("by the lengths", sequences, d, group, rows)
    assert c.need
    c.call()
    lib.synchronize()
    size = int(c.work.read(np.uint8)[-16:].view(np.uint32)[0])  # where the join finds it
    assert 0 < size < max(lengths) and size % 128 == 0
    c.check()
    assert np.all(np.ascontiguousarray(c.out.read(np.uint8)[int(n.sum()) * group * kv * d * 2:]).view(np.uint32) == 0x7FC12345)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("rows,lengths,first", [([50, 1, 1, 2], [120, 900, 0, 1400], 1), ([1, 3, 140], [2000, 3, 200], 2), ([1] * 70 + [30], [90] * 70 + [700], 70)])
def test_a_batch_in_two_calls(lib, d, rows, lengths, first):
    """A prompt's rows and single tokens apart: each call has the whole batch's rows and its own sequences' starts, lengths and
    tables, and leaves the other's rows as they were."""
    rng = np.random.default_rng(d + len(rows))
    c = Case(lib, rng, rows, lengths, 8, 2, d, 16, "bf16", sinks=True, extra_rows=2)
    q, cache, table, lens, starts, sinks = c.dev
    total, z = int(c.b.starts[-1]), 8 * d * 2
    for at, n in ((0, first), (first, len(rows) - first)):
        p = lib.Cache.from_buffer_copy(c.p)
        p.sequences, p.max_rows, p.max_length = n, max(rows[at:at + n]), max(lengths[at:at + n])
        need = lib.cache_attention_workspace(p)
        work = Guarded(lib, need)
        say("in two", d, rows[:5], at, n)
        before = c.out.read(np.uint8).copy()
        lib.cache_attention(q, cache, table.ptr + 4 * at * c.b.stride, lens.ptr + 4 * at, c.out.ptr, p, starts=starts.ptr + 4 * at, sinks=sinks,
                            workspace=work.ptr if need else None, workspace_bytes=need)
        lib.synchronize()
        work.read(np.uint8)
        after, mine = c.out.read(np.uint8), slice(int(c.b.starts[at]) * z, int(c.b.starts[at + n]) * z)
        before[mine] = after[mine]
        np.testing.assert_array_equal(after, before)
    c.check()
    assert np.all(np.ascontiguousarray(c.out.read(np.uint8)[total * z:]).view(np.uint32) == 0x7FC12345)
