"""oco_block_norm against the formula in 64 bits.

Error counted in u = 2^-24 (half a step of f32, relative): the sum of squares
of a row is at most 32 terms per thread (P = 0: n / 1024 terms), 6 steps
within a wavefront and 16 between them; the inverse root halves its error and
adds 4; the products with weight and gate add 4, the gate's own value 8.  Then
the residual's rounding, half a step of its type.  The second norm is held to
the formula of the rounded x_out that the call returned.
"""
import numpy as np
import pytest

from _ops import CODE, HALF, LEAST, SIZE, U, dev, e4m3, stored, values
from _util import Guarded, say

pytestmark = pytest.mark.gpu
EPS = 1e-6


def norm_u(n):
    return ((56 + n / 1024) / 2 + 4) * U


def gates(kind, g):
    return {0: np.ones_like(g), 1: g, 2: 1 / (1 + np.exp(-g)), 3: np.tanh(g)}[kind]


def check(lib, rows, n, x_dtype, dtype, kind=1, gate_rows=0, post=True, pre=True, codes=False, pad=(0, 0, 0, 0), offset=0.0,
          scale=0.5, seed=0, inplace=False, spread=1.0, skip=0):
    say("block_norm", rows, n, x_dtype, dtype, kind, gate_rows, post, pre, codes, pad, offset, inplace)
    rng = np.random.default_rng(seed + rows * 7 + n)
    xs, ys, gs, os_ = (n + p for p in pad)
    ngate = 1 if gate_rows == 0 else -(-rows // gate_rows)
    xb, x = stored(4 * spread * rng.normal(size=(rows, xs)), x_dtype)
    yb, y = stored(spread * rng.normal(size=(rows, ys)), dtype)
    gb, g = stored(2 * rng.normal(size=(ngate, gs)), dtype)
    post_w, pre_w = (1 + 0.3 * rng.normal(size=n)).astype(np.float32), (1 + 0.3 * rng.normal(size=n)).astype(np.float32)
    x_out = Guarded(lib, rows * xs * SIZE[x_dtype])
    out = Guarded(lib, rows * os_ * SIZE[dtype])
    code_out, scale_out = Guarded(lib, rows * n), Guarded(lib, -(-n // 128) * rows * 4)
    if inplace:
        x_out.buf.upload(xb, 128)  # behind the guard
    # operands `skip` bytes into their buffers: a type's own alignment, no more
    xd, yd, gd = (dev(lib, np.concatenate([np.zeros(skip * SIZE[t] // 1, np.uint8), np.ravel(b)])) for b, t in ((xb, x_dtype), (yb, dtype), (gb, dtype)))
    p = lib.Block(rows=rows, n=n, x_dtype=CODE[x_dtype], dtype=CODE[dtype], gate=kind, gate_rows=gate_rows, x_stride=xs if pad[0] else 0,
                  y_stride=ys if pad[1] else 0, gate_stride=gs if pad[2] else 0, out_stride=os_ if pad[3] else 0, scale=scale,
                  epsilon=EPS, weight_offset=offset)
    post_d, pre_d = dev(lib, post_w), dev(lib, pre_w)
    lib.block_norm(x_out.ptr if inplace else xd.ptr + skip * SIZE[x_dtype], yd.ptr + skip * SIZE[dtype], p, x_out=x_out.ptr,
                   gate=gd.ptr + skip * SIZE[dtype] if kind else None,
                   post_w=post_d if post else None, pre_w=pre_d if pre else None, out=out.ptr if pre else None,
                   codes=code_out.ptr if codes else None, scales=scale_out.ptr if codes else None)
    lib.synchronize()
    x, y, g = x[:, :n], y[:, :n], g[:, :n]
    v = y / np.sqrt((y * y).mean(1, keepdims=True) + EPS) * (post_w.astype(np.float64) + offset) if post else y
    v = v * gates(kind, g)[np.arange(rows) // gate_rows if gate_rows else np.zeros(rows, int)] * scale
    want = x + v
    got = values(x_out.read(np.uint8), x_dtype, (rows, xs))
    bound = np.abs(v) * (norm_u(n) + 16 * U) + (2 * U + HALF[x_dtype]) * np.abs(want) * 1.01 + LEAST[x_dtype]
    assert np.all(np.abs(got[:, :n] - want) <= bound)
    if pad[0] and not inplace:  # columns between rows are left as they were
        raw = x_out.read(np.uint8).reshape(rows, xs * SIZE[x_dtype])[:, n * SIZE[x_dtype]:]
        assert np.array_equal(raw, np.resize(np.frombuffer(np.uint32(0x7FC12345).tobytes() * (x_out.words + 1), np.uint8),
                                             rows * xs * SIZE[x_dtype]).reshape(rows, -1)[:, n * SIZE[x_dtype]:])
    if not pre:
        assert np.all(out.read(np.uint8).view(np.uint8)[:4] == np.frombuffer(np.uint32(0x7FC12345).tobytes(), np.uint8)[:4])
        return got
    kept = got[:, :n]
    exact = kept / np.sqrt((kept * kept).mean(1, keepdims=True) + EPS) * (pre_w.astype(np.float64) + offset)
    norm = values(out.read(np.uint8), dtype, (rows, os_))[:, :n]
    assert np.all(np.abs(norm - exact) <= (norm_u(n) + 4 * U + HALF[dtype]) * 1.01 * np.abs(exact) + LEAST[dtype])
    if codes:
        scales = scale_out.read(np.float32).astype(np.float64).reshape(-1, rows)
        c = e4m3(code_out.read(np.uint8), (rows, n))
        err = norm_u(n) + 8 * U
        for b in range(len(scales)):
            part = exact[:, 128 * b:128 * b + 128]
            top = np.abs(part).max(1)
            assert np.all(np.abs(scales[b] - top / 448) <= err * top / 448 + 2.0 ** -149)
            q = part / scales[b][:, None]
            half = np.maximum(2.0 ** (np.floor(np.log2(np.maximum(np.abs(q), 1e-30))) - 4), 2.0 ** -10)
            assert np.all(np.abs(c[:, 128 * b:128 * b + 128] - q) <= half * 1.001 + 2 * err * np.abs(q))
    return got


@pytest.mark.parametrize("n", [1, 7, 8, 63, 512, 513, 1000, 1024, 1025, 2048, 2880, 4096, 4097, 8192, 9001, 16384, 20000, 32768, 32769, 50000])
@pytest.mark.parametrize("rows", [1, 5])
def test_widths(lib, rows, n):
    """Every number of threads and runs per row, at its ends and between."""
    check(lib, rows, n, "bf16", "bf16")


@pytest.mark.parametrize("n", [600, 1024, 4096, 6000])
def test_many_rows(lib, n):
    """Past 256 rows a row takes fewer threads."""
    check(lib, 301, n, "f32", "bf16", kind=2, gate_rows=1)


@pytest.mark.parametrize("x_dtype,dtype", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("kind,gate_rows", [(0, 0), (1, 0), (2, 1), (3, 3)])
def test_types_and_gates(lib, x_dtype, dtype, kind, gate_rows):
    check(lib, 7, 544, x_dtype, dtype, kind=kind, gate_rows=gate_rows, offset=1.0, codes=True)


@pytest.mark.parametrize("post,pre", [(False, True), (True, False), (False, False)])
def test_absent_norms(lib, post, pre):
    check(lib, 6, 777, "bf16", "bf16", post=post, pre=pre)


@pytest.mark.parametrize("pad", [(3, 0, 0, 0), (0, 5, 0, 0), (0, 0, 7, 0), (0, 0, 0, 1), (8, 1, 2, 9)])
def test_strides(lib, pad):
    check(lib, 9, 261, "bf16", "bf16", gate_rows=2, pad=pad)


@pytest.mark.parametrize("n", [250, 4099])
def test_operands_at_their_own_alignment(lib, n):
    check(lib, 4, n, "bf16", "bf16", skip=1)
    check(lib, 4, n, "f32", "f16", skip=3)


@pytest.mark.parametrize("n", [384, 40000])
def test_in_place_equals_out_of_place(lib, n):
    a = check(lib, 5, n, "bf16", "bf16", inplace=False)
    b = check(lib, 5, n, "bf16", "bf16", inplace=True)
    np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("n", [16, 128, 144, 2880, 8192, 40000])
def test_codes_of_partial_blocks(lib, n):
    check(lib, 3, n, "f32", "bf16", codes=True)


def test_equals_add_norm_of_the_library(lib):
    """Without a post-norm, a gate and a scale: oco_add_norm's residual bit for bit, and its norm."""
    rng = np.random.default_rng(3)
    rows, n = 5, 2880
    x, y = stored(rng.normal(size=(rows, n)), "bf16")[0], stored(rng.normal(size=(rows, n)), "bf16")[0]
    w = dev(lib, (1 + 0.2 * rng.normal(size=n)).astype(np.float32))
    x1, y1, o1, x2, o2 = dev(lib, x), dev(lib, y), lib.DeviceBuffer(rows * n * 2), lib.DeviceBuffer(rows * n * 2), lib.DeviceBuffer(rows * n * 2)
    lib.block_norm(x1, y1, lib.Block(rows=rows, n=n, x_dtype=1, dtype=1, scale=1.0, epsilon=EPS), x_out=x2, pre_w=w, out=o2)
    lib.add_norm(x1, y1, w, o1, rows, n, EPS)
    lib.synchronize()
    np.testing.assert_array_equal(x1.download(np.uint16), x2.download(np.uint16))
    a, b = (values(o.download(np.uint8), "bf16", (rows, n)) for o in (o1, o2))
    # both within f32 roundings of the same value, rounded once: at most one step apart
    assert np.all(np.abs(a - b) <= 2 * HALF["bf16"] * np.abs(a) * 1.01)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_value_that_is_not_finite_stays_in_its_row(lib, bad):
    rng = np.random.default_rng(4)
    rows, n = 4, 1000
    y = rng.normal(size=(rows, n))
    y[2, 17] = bad
    x = stored(rng.normal(size=(rows, n)), "f32")[0]
    w = dev(lib, np.ones(n, np.float32))
    outs = []
    for q in (y, np.where(np.isfinite(y), y, 0.5)):
        x_out, out = lib.DeviceBuffer(rows * n * 4), lib.DeviceBuffer(rows * n * 2)
        lib.block_norm(dev(lib, x), dev(lib, stored(q, "bf16")[0]), lib.Block(rows=rows, n=n, x_dtype=0, dtype=1, scale=1.0, epsilon=EPS),
                       x_out=x_out, post_w=w, pre_w=w, out=out)
        lib.synchronize()
        outs.append((x_out.download(np.float32).reshape(rows, n), values(out.download(np.uint8), "bf16", (rows, n))))
    others = np.arange(rows) != 2
    assert np.isnan(outs[0][0][2, 17]) and np.all(np.isnan(outs[0][1][2]))
    for a, b in zip(*outs):
        np.testing.assert_array_equal(a[others], b[others])


def test_zero_rows_and_extreme_values(lib):
    """Rows of zeros stay zero (epsilon under the root), and bf16 rows whose
    squares are far from 1 keep the bounds."""
    rows, n = 2, 512
    z = dev(lib, np.zeros(rows * n, np.uint16))
    w = dev(lib, np.ones(n, np.float32))
    x_out, out = lib.DeviceBuffer(rows * n * 2), lib.DeviceBuffer(rows * n * 2)
    codes, scales = lib.DeviceBuffer(rows * n), lib.DeviceBuffer(4 * rows * 4)
    lib.block_norm(z, z, lib.Block(rows=rows, n=n, x_dtype=1, dtype=1, scale=1.0, epsilon=EPS), x_out=x_out, post_w=w, pre_w=w, out=out,
                   codes=codes, scales=scales)
    lib.synchronize()
    for b in (x_out, out):
        assert not b.download(np.uint16).any()
    assert not codes.download(np.uint8).any() and np.all(scales.download(np.float32) == 2.0 ** -126)
    check(lib, 3, 700, "bf16", "bf16", spread=2.0 ** 40)
    check(lib, 3, 700, "bf16", "bf16", spread=2.0 ** -40)


@pytest.mark.parametrize("rows,n", [(1, 16), (3, 512), (1030, 1024), (2, 2048), (3, 2064), (2, 4096), (1, 8192), (2, 16384), (1, 32768), (1, 40016)])
def test_8_bit_rows_at_every_width(lib, rows, n):
    check(lib, rows, n, "f32", "bf16", kind=1, codes=True)
    check(lib, rows, n, "bf16", "bf16", codes=True, inplace=True)


@pytest.mark.parametrize("n", [2049, 2560, 2561, 3584, 3585, 5120, 5121, 6144, 6145, 8185])
def test_threads_that_fit_the_row(lib, n):
    check(lib, 5, n, "bf16", "bf16", kind=3)
    check(lib, 3, n // 16 * 16, "f32", "f16", kind=2, gate_rows=2, codes=True)


def rounded_e4m3(q):
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -30))), -6) - 3)
    return np.rint(q / step) * step


@pytest.mark.parametrize("rows,n", [(3, 144), (33, 512), (1030, 1024), (70, 2880), (9, 8192), (5, 16384), (3, 32768), (3, 40000)])
@pytest.mark.parametrize("x_dtype,dtype,kind", [("f32", "bf16", 2), ("bf16", "bf16", 1), ("f32", "f32", 0), ("f16", "f16", 3)])
def test_codes_and_scales_are_those_of_the_64_bit_rows(lib, rows, n, x_dtype, dtype, kind):
    """Codes and scales from the x_out that the call returned, to the last bit
    but where the 64-bit roundings reach a border: at most 62 additions of squares
    (40 in a thread, 6 and 16 over the threads) and the oracle's 28, halved by the
    root, and 18 for roots, reciprocals and products: under 64 * 2^-53 together."""
    say("block codes", rows, n, x_dtype, dtype, kind)
    near = 64 * 2.0 ** -53
    rng = np.random.default_rng(rows + n)
    xb, yb = (stored(rng.normal(size=(rows, n)) * s, t)[0] for s, t in ((4, x_dtype), (1, dtype)))
    gb = stored(rng.normal(size=(rows, n)), dtype)[0]
    post_w, pre_w = (1 + 0.3 * rng.normal(size=n)).astype(np.float32), (1 + 0.3 * rng.normal(size=n)).astype(np.float32)
    x_out, codes, scales = Guarded(lib, rows * n * SIZE[x_dtype]), Guarded(lib, rows * n), Guarded(lib, -(-n // 128) * rows * 4)
    p = lib.Block(rows=rows, n=n, x_dtype=CODE[x_dtype], dtype=CODE[dtype], gate=kind, gate_rows=1, scale=0.5, epsilon=EPS, weight_offset=0.25)
    lib.block_norm(dev(lib, xb), dev(lib, yb), p, x_out=x_out.ptr, gate=dev(lib, gb), post_w=dev(lib, post_w), pre_w=dev(lib, pre_w),
                   codes=codes.ptr, scales=scales.ptr)
    lib.synchronize()
    kept = values(x_out.read(np.uint8), x_dtype, (rows, n))
    exact = kept / np.sqrt((kept * kept).mean(1, keepdims=True) + np.float64(np.float32(EPS))) * (pre_w.astype(np.float64) + 0.25)
    got, s = e4m3(codes.read(np.uint8), (rows, n)), scales.read(np.float32).reshape(-1, rows)
    for b in range(len(s)):
        part = exact[:, 128 * b:128 * b + 128]
        top = np.maximum(np.abs(part).max(1), 448 * 2.0 ** -126)
        lo, hi = ((top * (1 + e) / 448).astype(np.float32) for e in (-near, near))
        assert np.all((s[b] == lo) | (s[b] == hi))
        q, c = 448 * part / top[:, None], got[:, 128 * b:128 * b + 128]
        assert np.all((c == rounded_e4m3(q * (1 - near))) | (c == rounded_e4m3(q * (1 + near))))


@pytest.mark.parametrize("spread", [2.0 ** 80, 2.0 ** -90])
@pytest.mark.parametrize("n", [704, 40000])
def test_8_bit_rows_of_values_whose_squares_f32_cannot_hold(lib, spread, n):
    """With 8-bit rows the values between are 64-bit, the squares and their sums among them."""
    check(lib, 3, n, "bf16", "bf16", spread=spread, codes=True)
    check(lib, 3, n, "f32", "f32", kind=0, spread=spread, codes=True)


@pytest.mark.parametrize("n", [513, 600, 1023, 1024])
@pytest.mark.parametrize("x_dtype,dtype,kind,gate_rows", [("f32", "f32", 0, 0), ("f32", "bf16", 3, 7), ("bf16", "bf16", 1, 0), ("f16", "f16", 2, 1)])
def test_a_wavefront_per_row(lib, n, x_dtype, dtype, kind, gate_rows):
    """More than 1024 rows of 513 to 1024 columns, four to a workgroup, the last one's not whole."""
    check(lib, 1030, n, x_dtype, dtype, kind=kind, gate_rows=gate_rows)
