"""oco_rotate, oco_cache_append and oco_cache_read against their rules in 64 bits: rotations within one rounding,
pages byte for byte."""
import numpy as np
import pytest

from _cache import Batch, Pool, dequantize, quantize
from _ops import CODE, HALF, LEAST, SIZE, dev, stored, values
from _util import Guarded, say

pytestmark = pytest.mark.gpu


def turned(x, positions, f, magnitude, dim, interleaved):
    """Rows [r, h, d] in 64 bits, and what a rounding of products and sums can be off by at most."""
    y, a = x.copy(), positions.astype(np.float64)[:, None] * f
    c, s = (np.cos(a) * magnitude)[:, None], (np.sin(a) * magnitude)[:, None]
    first = slice(0, dim, 2) if interleaved else slice(0, dim // 2)
    second = slice(1, dim, 2) if interleaved else slice(dim // 2, dim)
    u, v = x[..., first], x[..., second]
    y[..., first], y[..., second] = u * c - v * s, v * c + u * s
    off = np.zeros_like(x)
    off[..., first] = off[..., second] = (np.abs(u) + np.abs(v)) * 2.0 ** -50 * abs(magnitude)
    return y, off


def rotation(lib, f, magnitude, dim, interleaved, keep):
    keep.append(dev(lib, np.asarray(f, np.float64)) if dim else None)
    return lib.Rotation(dim=dim, layout=int(interleaved), magnitude=magnitude, frequencies=keep[-1].ptr if dim else None)


def near(got, want, off, dtype):
    # f64 -> f32 -> the type: half a step of each
    tol = np.abs(want) * HALF[dtype] * (1 + 2.0 ** -10) + np.abs(want) * 2.0 ** -24 + LEAST[dtype] + off
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,d,dim", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 80, 32), (7, 3, 96, 70), (130, 4, 64, 64), (2, 1, 5, 4), (200, 3, 256, 0),
                                              (5, 2, 1024, 1024)])
def test_rotate(lib, dtype, interleaved, rows, heads, d, dim):
    rng = np.random.default_rng(rows * 1000 + d + dim)
    keep, f = [], 10000.0 ** (-np.arange(dim // 2) * 2.0 / max(dim, 1))
    r = rotation(lib, f, 1.25, dim, interleaved, keep)
    pos = rng.integers(0, 2 ** 32 - 1, rows) if rows > 4 else rng.integers(0, 200000, rows)
    raw, x = stored(rng.normal(size=(rows, heads, d)) * 3, dtype)
    say("rotate", dtype, interleaved, rows, heads, d, dim)
    out = Guarded(lib, raw.nbytes)
    lib.rotate(dev(lib, raw), rows, heads, d, out.ptr, r, dev(lib, pos.astype(np.uint32)), CODE[dtype])
    lib.synchronize()
    want, off = turned(x, pos, f, 1.25, dim, interleaved)
    got = values(out.read(np.uint8), dtype, x.shape)
    near(got, want, off, dtype)
    np.testing.assert_array_equal(got[..., dim:], x[..., dim:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotate_strided_and_in_place(lib, interleaved):
    """Queries inside wider rows at an odd offset: what lies between them stays; in place as elsewhere."""
    rng = np.random.default_rng(4)
    rows, heads, d, dim, stride, keep = 9, 3, 40, 24, 3 * 40 + 7, []
    f = 500.0 ** (-np.arange(dim // 2) * 2.0 / dim)
    r = rotation(lib, f, 1.0, dim, interleaved, keep)
    raw, x = stored(rng.normal(size=(rows, stride)), "bf16")
    pos = rng.integers(0, 5000, rows)
    buf, p = dev(lib, raw), dev(lib, pos.astype(np.uint32))
    want, off = turned(x[:, 3:3 + heads * d].reshape(rows, heads, d), pos, f, 1.0, dim, interleaved)
    out = Guarded(lib, rows * heads * d * 2)
    lib.rotate(buf.ptr + 6, rows, heads, d, out.ptr, r, p, 1, x_stride=stride)
    lib.rotate(buf.ptr + 6, rows - 1, heads, d, buf.ptr + 6, r, p, 1, x_stride=stride, out_stride=stride)
    lib.synchronize()
    got = values(out.read(np.uint8), "bf16", want.shape)
    near(got, want, off, "bf16")
    after = values(buf.download(np.uint8), "bf16", x.shape)
    mine = np.zeros(x.shape, bool)
    mine[:rows - 1, 3:3 + heads * d] = True
    np.testing.assert_array_equal(after[~mine], x[~mine])
    np.testing.assert_array_equal(after[:rows - 1, 3:3 + heads * d].reshape(rows - 1, heads, d), got[:rows - 1])


def test_rotate_not_finite(lib):
    """A NaN or an infinity reaches its own pair and no other value."""
    x = np.ones((1, 2, 16))
    x[0, 0, 3], x[0, 1, 9] = np.nan, np.inf
    raw, _ = stored(x, "f16")
    keep = []
    out = Guarded(lib, raw.nbytes)
    lib.rotate(dev(lib, raw), 1, 2, 16, out.ptr, rotation(lib, np.full(8, 0.5), 1.0, 16, False, keep), dev(lib, np.array([1], np.uint32)), 2)
    lib.synchronize()
    got = np.isfinite(values(out.read(np.uint8), "f16", x.shape))
    want = np.ones(x.shape, bool)
    want[0, 0, [3, 11]] = want[0, 1, [1, 9]] = False
    np.testing.assert_array_equal(got, want)


class Case:
    """An append of a batch into a pool of NaN pages, with and without its queries."""

    def __init__(self, lib, rng, rows, lengths, heads, kv, d, P, dtype, dim, interleaved=False, extra_rows=0, packed=False, own_positions=False,
                 queries=True, scale=1.0, with_starts=True):
        self.lib, self.b, self.dtype = lib, Batch(rng, rows, lengths, P, extra_rows=extra_rows), dtype
        b, T = self.b, self.b.total
        width = (heads + 2 * kv) * d + (5 if packed else 0)
        self.raw, x = stored(rng.normal(size=(T, width)) * scale, dtype)
        self.x = x[:, :(heads + 2 * kv) * d].reshape(T, heads + 2 * kv, d)
        self.f = 10000.0 ** (-np.arange(dim // 2) * 2.0 / max(dim, 1))
        self.heads, self.kv, self.d, self.dim, self.interleaved = heads, kv, d, dim, interleaved
        self.positions = rng.integers(0, 90000, T) if own_positions else None
        self.p = b.describe(lib, heads, kv, d, CODE[dtype], q_stride=width, k_stride=width, v_stride=width)
        self.pool = Pool(b.pages, kv, P, d)
        self.keep = [dev(lib, self.raw), dev(lib, b.table), dev(lib, np.array(lengths, np.uint32)), dev(lib, b.starts),
                     dev(lib, self.positions.astype(np.uint32)) if own_positions else None]
        self.r = rotation(lib, self.f, 1.0, dim, interleaved, self.keep)
        assert lib.cache_page_bytes(self.p) * b.pages == self.pool.bytes.nbytes
        self.cache, self.queries, self.with_starts = Guarded(lib, self.pool.bytes.nbytes), queries, with_starts
        lib._check(lib.load_library().oco_buffer_fill32(self.cache.ptr, 0xFFFFFFFF, self.pool.bytes.nbytes // 4, None))
        self.out = Guarded(lib, T * heads * d * SIZE[dtype])

    def call(self, stream=None):
        z, x = SIZE[self.dtype], self.keep[0].ptr
        k, v = x + self.heads * self.d * z, x + (self.heads + self.kv) * self.d * z
        self.lib.cache_append(self.cache.ptr, self.keep[1], self.keep[2], k, v, self.p, starts=self.keep[3] if self.with_starts else None,
                              q=x if self.queries else None, q_out=self.out.ptr if self.queries else None, positions=self.keep[4],
                              rotation=self.r if self.dim else None, stream=stream)

    def check(self):
        b, h, kv = self.b, self.heads, self.kv
        live = list(b.row_positions())
        at = np.array([max(t, 0) for _, t in live])
        turn = self.positions[:len(live)] if self.positions is not None else at
        y, off = turned(self.x[:len(live), :h + kv], turn, self.f, 1.0, self.dim, self.interleaved)
        keys = quantize(stored(y[:, h:], self.dtype)[1])
        vals = quantize(self.x[:len(live), h + kv:])
        for r, (s, t) in enumerate(live):
            if t < 0:
                continue
            page, slot = b.place(s, t)
            if page >= b.pages:
                continue
            for j in range(kv):
                self.pool.put(page, slot, j, (keys[0][r, j], keys[1][r, j]), (vals[0][r, j], vals[1][r, j]))
        got = self.cache.read(np.uint8).reshape(self.pool.bytes.shape)
        np.testing.assert_array_equal(got, self.pool.bytes)
        out = self.out.read(np.uint8)
        if self.queries:
            got = values(out, self.dtype, (b.total, h, self.d))
            near(got[:len(live)], y[:, :h], off[:, :h], self.dtype)
            out = out.reshape(b.total, -1)[len(live):]
        words = np.ascontiguousarray(out).reshape(-1).view(np.uint32)
        assert np.all(words == 0x7FC12345)  # queries that nobody asked for, and rows behind the last sequence
        return dequantize(*keys), dequantize(*vals)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,lengths,P", [([1], [1], 16), ([1, 1, 1], [17, 64, 200], 16), ([5, 0, 33, 1], [5, 9, 100, 48], 48), ([7, 3], [4, 0], 32),
                                            ([70], [70], 256)])
def test_append(lib, dtype, d, rows, lengths, P):
    """Pages that start and end inside a sequence, empty sequences, rows without a token (more rows than tokens)."""
    rng = np.random.default_rng(d + sum(rows))
    say("append", dtype, d, rows, lengths, P)
    c = Case(lib, rng, rows, lengths, 6, 2, d, P, dtype, d)
    c.call()
    lib.synchronize()
    c.check()


@pytest.mark.parametrize("over", [dict(dim=0), dict(dim=32), dict(dim=50, interleaved=True), dict(dim=64, interleaved=True, packed=True),
                                  dict(dim=128, own_positions=True), dict(dim=128, extra_rows=9), dict(dim=128, queries=False), dict(dim=30, packed=True)])
@pytest.mark.parametrize("heads,kv", [(1, 1), (24, 24), (40, 8)])
def test_append_forms(lib, over, heads, kv):
    """Partial and interleaved rotations, packed rows at odd strides, given positions, rows behind the last sequence, no
    queries, more heads than one workgroup takes."""
    rng = np.random.default_rng(heads)
    say("append", over, heads, kv)
    c = Case(lib, rng, [9, 2, 1], [40, 2, 65], heads, kv, 128, 32, "bf16", **over)
    c.call()
    lib.synchronize()
    c.check()


def test_append_without_starts_and_many_sequences(lib):
    """The same number of rows of each; with starts, sequences enough for several rounds of the search."""
    rng = np.random.default_rng(8)
    for rows, starts in (([2] * 70, False), ([1] * 300, True), ([int(n) for n in rng.integers(0, 3, 5000)], True)):
        lengths = [n + int(k) for n, k in zip(rows, rng.integers(0, 20, len(rows)))]
        say("append", len(rows), starts)
        c = Case(lib, rng, rows, lengths, 2, 1, 64, 16, "bf16", 64, with_starts=starts)
        c.call()
        lib.synchronize()
        c.check()


def test_append_to_pages_outside_the_pool(lib):
    rng = np.random.default_rng(9)
    c = Case(lib, rng, [40, 3], [40, 20], 4, 2, 128, 16, "bf16", 128)
    c.b.table[0, 1], c.b.table[1, 1] = c.b.pages, 0xFFFFFFFF
    c.keep[1].upload(c.b.table)
    c.call()
    lib.synchronize()
    c.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_blocks_at_their_borders(lib, dtype):
    """Values on and next to the borders between two codes at every scale, blocks of zeros, of subnormal numbers, with NaN
    and infinities in them."""
    rng = np.random.default_rng(3)
    e = np.concatenate([np.arange(-149, 126, 3), np.arange(-30, 16)])
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    n = len(e)
    v = rng.choice(np.concatenate([borders, borders * (1 + 2.0 ** -7), borders * (1 - 2.0 ** -8), LEVELS_AND_MORE]), (n, 4, 32)) * rng.choice([-1, 1], (n, 4, 32))
    v[:, :, 0] = rng.choice([4.0, 7.96875, 5.0, 6.0], (n, 4))
    v = v * np.ldexp(1.0, e)[:, None, None]
    v[5, 0], v[6, 1, 7], v[7, 2, 3], v[8, 3, 31], v[9, 0] = 0, np.nan, np.inf, -np.inf, -0.0
    rows = v.reshape(n, 1, 128)
    raw, x = stored(np.concatenate([np.zeros((n, 1, 128)), rows, rows[::-1]], 1), dtype)
    b = Batch(rng, [n], [n], 64)
    p = b.describe(lib, 1, 1, 128, CODE[dtype], k_stride=384, v_stride=384)
    pool, z = Pool(b.pages, 1, 64, 128), SIZE[dtype]
    cache, buf = dev(lib, pool.bytes), dev(lib, raw)
    table, lengths = dev(lib, b.table), dev(lib, np.array([n], np.uint32))
    say("borders", dtype)
    lib.cache_append(cache, table, lengths, buf.ptr + 128 * z, buf.ptr + 256 * z, p)
    k, w = Guarded(lib, n * 128 * z), Guarded(lib, n * 128 * z)
    back = b.describe(lib, 1, 1, 128, CODE[dtype])
    lib.cache_read(cache, table, lengths, k.ptr, w.ptr, back)
    lib.synchronize()
    keys, vals = quantize(x[:, 1]), quantize(x[:, 2])
    for t in range(n):
        page, slot = b.place(0, t)
        pool.put(page, slot, 0, (keys[0][t], keys[1][t]), (vals[0][t], vals[1][t]))
    np.testing.assert_array_equal(cache.download(np.uint8).reshape(pool.bytes.shape), pool.bytes)
    for got, (codes, scales) in ((k, keys), (w, vals)):
        np.testing.assert_array_equal(values(got.read(np.uint8), dtype, (n, 128)), stored(dequantize(codes, scales), dtype)[1])


LEVELS_AND_MORE = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.1, 2.2, 6.9])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_read(lib, dtype, d):
    """What was appended comes back as the values it stands for; rows without a token are 0, pages outside the pool NaN, rows
    behind the last sequence stay."""
    rng = np.random.default_rng(d)
    c = Case(lib, rng, [37, 0, 6, 2], [50, 3, 4, 90], 4, 2, d, 16, dtype, d, extra_rows=3)
    c.call()
    lib.synchronize()
    keys, vals = c.check()
    live = list(c.b.row_positions())
    for r, (s, t) in enumerate(live):
        if t < 0:
            keys[r] = vals[r] = 0
    broken = c.b.table.copy()
    broken[3, 89 // 16] = c.b.pages + 1
    for r, (s, t) in enumerate(live):
        if s == 3 and t // 16 == 89 // 16:
            keys[r] = vals[r] = np.nan
    p = c.b.describe(lib, 4, 2, d, CODE[dtype], k_stride=2 * d + 3)
    z = SIZE[dtype]
    k, v = Guarded(lib, c.b.total * (2 * d + 3) * z), Guarded(lib, c.b.total * 2 * d * z)
    say("read", dtype, d)
    lib.cache_read(c.cache.ptr, dev(lib, broken), c.keep[2], k.ptr, v.ptr, p, starts=c.keep[3])
    lib.synchronize()
    got_k = values(k.read(np.uint8)[:c.b.total * (2 * d + 3) * z], dtype, (c.b.total, 2 * d + 3))[:len(live), :2 * d]
    got_v = values(v.read(np.uint8), dtype, (c.b.total, 2 * d))[:len(live)]
    np.testing.assert_array_equal(got_k.reshape(keys.shape), stored(keys, dtype)[1])
    np.testing.assert_array_equal(got_v.reshape(vals.shape), stored(vals, dtype)[1])
    tail = v.read(np.uint8).reshape(c.b.total, -1)[len(live):]
    assert np.all(np.ascontiguousarray(tail).reshape(-1).view(np.uint32) == 0x7FC12345)


@pytest.mark.parametrize("named", [False, True])
def test_append_packed_queries_in_place(lib, named):
    """Queries turned where they lie, between the keys and values of one product's rows, through PagedCache: those turned into
    rows of their own, and nothing else of the product changes; the attention reads them there, and may leave its rows there."""
    rng = np.random.default_rng(3)
    heads, kv, d, P, rows, lengths = 6, 2, 64, 16, [3, 1], [3, 1]
    b, width = Batch(rng, rows, lengths, P), (heads + 2 * kv) * d + 6
    raw, _ = stored(rng.normal(size=(b.total, width)), "bf16")
    keep = []
    r = rotation(lib, 100.0 ** (-np.arange(d // 2) * 2.0 / d), 1.0, d, False, keep)
    table, lens, starts, apart = dev(lib, b.table), dev(lib, np.array(lengths, np.uint32)), dev(lib, b.starts), Guarded(lib, b.total * heads * d * 2)
    pages, product = [], dev(lib, raw)
    for place in (apart.ptr, product.ptr if named else None):
        cache = lib.PagedCache(b.pages, d, kv, P)
        cache.buffer.fill32(0)
        batch = cache.batch(table, lens, len(rows), b.total, max(rows), max(lengths), b.stride, heads, starts=starts)
        say("packed", named, place is None)
        batch.append(product.ptr + heads * d * 2, product.ptr + (heads + kv) * d * 2, q=product.ptr, q_out=place, rotation=r, stride=width)
        lib.synchronize()
        pages.append(cache.buffer.download(np.uint8))
    np.testing.assert_array_equal(*pages)
    after = product.download(np.uint16).reshape(b.total, width)
    np.testing.assert_array_equal(after[:, :heads * d], apart.read(np.uint16).reshape(b.total, heads * d))
    np.testing.assert_array_equal(after[:, heads * d:], raw.view(np.uint16).reshape(b.total, width)[:, heads * d:])
    out = [Guarded(lib, b.total * heads * d * 2) for _ in range(2)]
    say("packed attention", named)
    batch.attention(apart.ptr, out[0].ptr)
    batch.attention(product, out[1].ptr, stride=width)
    batch.attention(product.ptr, product, stride=width)
    lib.synchronize()
    want = out[0].read(np.uint16).reshape(b.total, heads * d)
    np.testing.assert_array_equal(out[1].read(np.uint16).reshape(b.total, heads * d), want)
    again = product.download(np.uint16).reshape(b.total, width)
    np.testing.assert_array_equal(again[:, :heads * d], want)
    np.testing.assert_array_equal(again[:, heads * d:], after[:, heads * d:])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim", [64, 50])
def test_roundings_by_way_of_f32(lib, dtype, interleaved, dim):
    """Products next to the middle between two numbers of the type, nearer to it than f32 tells apart, go where the middle goes: to
    the even number. In f32 itself they go to the nearer one."""
    half, tiny, d = HALF[dtype], 2.0 ** -45, 64
    raw, x = stored(np.ldexp(1.0, np.arange(d) % 24 - 12) * np.where(np.arange(d) % 3, 1, -1), dtype)
    once = dtype == "f32"
    for factor, want in ((1 + half + tiny, 1 + 2 * half if once else 1.0), (1 + half - tiny, 1.0), (1 + 3 * half - tiny, 1 + 2 * half if once else 1 + 4 * half),
                         (1 + 3 * half + tiny, 1 + 4 * half)):
        keep, out = [], Guarded(lib, raw.nbytes)
        say("roundings", dtype, interleaved, factor)
        lib.rotate(dev(lib, raw), 1, 1, d, out.ptr, rotation(lib, np.zeros(dim // 2), factor, dim, interleaved, keep), dev(lib, np.array([7], np.uint32)),
                   CODE[dtype])
        lib.synchronize()
        np.testing.assert_array_equal(values(out.read(np.uint8), dtype, (d,)), np.where(np.arange(d) < dim, x * want, x))
