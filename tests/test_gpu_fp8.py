"""Rows in 8-bit floating point and their products against 64-bit forms."""
import numpy as np
import pytest

from _ops import CODE, HALF, LEAST, SIZE, U, dev, e4m3, quantized, stored, values
from _util import Guarded, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,pad", [(1, 16, 0), (3, 128, 0), (5, 144, 3), (17, 2880, 0), (2, 4096, 8), (1, 12288, 0)])
def test_quantize_is_exact(lib, dtype, rows, k, pad):
    """Codes and scales bit for bit: 16-bit rows by the real quotient, f32
    rows by the quotient of the two f32 operands."""
    say("quantize", dtype, rows, k, pad)
    rng = np.random.default_rng(rows + k)
    x = rng.normal(size=(rows, k + pad)) * np.where(rng.random(k + pad) < 0.02, 30.0, 1.0)
    x[0, :8] = [448, 1, 1.0625, 1.1875, 17, 19, 0, -0.0]  # quotients on borders between codes
    xb, x = stored(x, dtype)
    codes, scales = Guarded(lib, rows * k), Guarded(lib, -(-k // 128) * rows * 4)
    lib.fp8_quantize(dev(lib, xb), rows, k, codes.ptr, scales.ptr, CODE[dtype], k + pad if pad else 0)
    lib.synchronize()
    want_codes, want_scales = quantized(x[:, :k], dtype != "f32")
    np.testing.assert_array_equal(scales.read(np.float32).reshape(-1, rows), want_scales)
    np.testing.assert_array_equal(codes.read(np.uint8).reshape(rows, k), want_codes)


def test_quantize_extremes(lib):
    """Zeros, subnormal and largest values, and blocks that are not finite."""
    rows, k = 6, 256
    x = np.ones((rows, k), np.float32)
    x[0] = 0
    x[1, :128] = 2.0 ** -140
    x[2] = np.float32(3.0e38)
    x[3, 5] = np.nan
    x[4, 200] = np.inf
    x[5, :] = np.float32(2.0 ** -118) * np.arange(k)
    codes, scales = Guarded(lib, rows * k), Guarded(lib, 2 * rows * 4)
    lib.fp8_quantize(dev(lib, x), rows, k, codes.ptr, scales.ptr, CODE["f32"])
    lib.synchronize()
    s, c = scales.read(np.float32).reshape(2, rows), e4m3(codes.read(np.uint8), (rows, k))
    assert np.all(s[:, 0] == 2.0 ** -126) and not c[0].any()
    assert s[0, 1] == 2.0 ** -126 and s[1, 1] == np.float32(1) / np.float32(448)
    assert np.all(c[2] == 448) and np.all(np.isfinite(s[:, 2]))
    assert np.isnan(s[0, 3]) and np.all(np.isnan(c[3, :128])) and np.all(c[3, 128:] == 448)
    assert np.isnan(s[1, 4]) and np.all(np.isnan(c[4, 128:])) and np.all(c[4, :128] == 448)
    q = x[5].astype(np.float64) / np.repeat(s[:, 5].astype(np.float64), 128)
    assert np.all(np.abs(c[5] - q) <= np.maximum(np.abs(q) * 2.0 ** -4, 2.0 ** -10) * 1.001)


def operands(rng, m, n, k):
    """Random codes over the whole finite range of e4m3, and scales over several powers of two."""
    x, w = (rng.integers(0, 256, size=s).astype(np.uint8) for s in ((m, k), (n, k)))
    for a in (x, w):
        a[(a & 0x7F) == 0x7F] = 0x38  # NaN codes
    xs = (2.0 ** rng.uniform(-6, 2, size=(-(-k // 128), m))).astype(np.float32)
    ws = (2.0 ** rng.uniform(-8, 0, size=(-(-n // 128), -(-k // 128)))).astype(np.float32)
    return x, w, xs, ws


def product(x, w, xs, ws):
    """(sum, sum of magnitudes) in 64 bits."""
    (m, k), n = x.shape, w.shape[0]
    xv, wv = e4m3(x, x.shape), e4m3(w, w.shape)
    y, mag = np.zeros((m, n)), np.zeros((m, n))
    for b in range(len(xs)):
        c = slice(128 * b, 128 * b + 128)
        s = xs[b].astype(np.float64)[:, None] * ws[np.arange(n) // 128, b].astype(np.float64)
        y += (xv[:, c] @ wv[:, c].T) * s
        mag += (np.abs(xv[:, c]) @ np.abs(wv[:, c]).T) * s
    return y, mag


def dropped(x, w, xs, ws):
    """What the 8-bit matrix instruction may drop: in each group of eight
    consecutive k, seven products each lose under 2^-13 of the largest one's
    binade (codes of k, of the same group: |x| |w| at most)."""
    (m, k), n = x.shape, w.shape[0]
    xv, wv, out = np.abs(e4m3(x, x.shape)), np.abs(e4m3(w, w.shape)), np.zeros((m, n))
    for g in range(0, k, 8):
        s = xs[g // 128].astype(np.float64)[:, None] * ws[np.arange(n) // 128, g // 128].astype(np.float64)
        most = np.zeros((m, n))
        for j in range(g, min(g + 8, k)):
            np.maximum(most, xv[:, j:j + 1] * wv[:, j], out=most)
        out += 7 * 2.0 ** -13 * most * s
    return out


def check(lib, m, n, k, y_dtype="f32", bias=False, seed=0):
    say("fp8_matmul", m, n, k, y_dtype, bias)
    rng = np.random.default_rng(seed + m * 31 + n * 7 + k)
    x, w, xs, ws = operands(rng, m, n, k)
    b = rng.normal(size=n).astype(np.float32) if bias else None
    p = lib.Matrix(k, n, m, 0, 1, 1, 1 if bias else 0)
    need = lib.fp8_matmul_workspace(p)
    ws_buf = lib.DeviceBuffer(need) if need else None
    out = Guarded(lib, m * n * SIZE[y_dtype])
    bufs = [dev(lib, a) for a in (w, ws, x, xs)]
    bb = dev(lib, b) if bias else None
    lib.fp8_matmul(*bufs, out.ptr, p, CODE[y_dtype], bb, ws_buf, need)
    lib.synchronize()
    got = values(out.read(np.uint8), y_dtype, (m, n))
    want, mag = product(x, w, xs, ws)
    if bias:
        br = stored(b, "bf16")[1]
        want, mag = want + br, mag + np.abs(br)
    # a block's 128 exact products summed in f32 (two half steps each: the
    # matrix core may truncate), one FMA per block, the K parts, the scales' product and the bias
    bound = (2 * 128 + len(xs) + 12) * U * mag + HALF[y_dtype] * 1.01 * np.abs(want) + LEAST[y_dtype]
    if y_dtype != "f32":  # 16-bit outputs may take 8-bit matrix instructions
        bound = bound + dropped(x, w, xs, ws)
    if y_dtype == "f16":
        fits = np.abs(want) < 65000
        assert fits.any()
        got, want, bound = got[fits], want[fits], bound[fits]
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / bound))
    return out.read(np.uint8)


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 16, 128), (1, 17, 144), (2, 33, 272), (7, 129, 2880), (15, 100, 4096), (16, 31, 112),
                                   (1, 2880, 4096), (8, 1000, 1024)])
def test_few_rows(lib, m, n, k):
    check(lib, m, n, k)


@pytest.mark.parametrize("m,n,k", [(17, 40, 144), (31, 257, 1040), (32, 128, 128), (33, 129, 16), (63, 300, 2880), (64, 64, 4096), (65, 500, 400),
                                   (100, 127, 2064), (127, 256, 128), (129, 511, 640), (200, 1000, 1280), (257, 260, 4096), (300, 700, 96),
                                   (511, 513, 528), (1030, 255, 272)])
def test_many_rows(lib, m, n, k):
    check(lib, m, n, k)


@pytest.mark.parametrize("y_dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m", [1, 40, 130, 600])
def test_outputs_and_bias(lib, m, y_dtype):
    """Odd output widths: rows of y that are not 16-byte aligned."""
    check(lib, m, 333, 272, y_dtype, bias=True)
    check(lib, m, 336, 272, y_dtype, bias=True)


@pytest.mark.parametrize("m", [3, 70, 300])
def test_same_call_same_bits(lib, m):
    np.testing.assert_array_equal(check(lib, m, 200, 2880), check(lib, m, 200, 2880))


@pytest.mark.parametrize("m,bad", [(9, 4), (9, 0), (150, 149)])
def test_a_row_that_is_not_finite_stays_alone(lib, m, bad):
    """A NaN scale makes its row NaN and no other; so do NaN codes."""
    rng = np.random.default_rng(m)
    n, k = 144, 400
    x, w, xs, ws = operands(rng, m, n, k)
    xs[1, bad] = np.nan
    x[bad, 130] = 0x7F
    p = lib.Matrix(k, n, m, 0, 1, 1, 0)
    need = lib.fp8_matmul_workspace(p)
    out = Guarded(lib, m * n * 4)
    lib.fp8_matmul(dev(lib, w), dev(lib, ws), dev(lib, x), dev(lib, xs), out.ptr, p, 0, workspace=lib.DeviceBuffer(max(need, 16)), workspace_bytes=need)
    lib.synchronize()
    got = out.read(np.float32).reshape(m, n)
    assert np.all(np.isnan(got[bad])) and np.all(np.isfinite(got[np.arange(m) != bad]))


@pytest.mark.parametrize("m,k", [(1, 144), (20, 144), (140, 144), (300, 272)])
def test_what_lies_behind_a_row_is_not_read(lib, m, k):
    """K ends inside a block of 128: NaN codes in the next rows' place (the
    next weights row, and behind the last rows) do not reach a sum."""
    rng = np.random.default_rng(k)
    n = 64
    x, w, xs, ws = operands(rng, m, n, k)
    say("fp8 behind", m, k)
    x[1:], w[1:] = 0x7F, 0x7F  # every row but the first is NaN throughout
    pad = np.full(4096, 0x7F, np.uint8)
    p = lib.Matrix(k, n, m, 0, 1, 1, 0)
    need = lib.fp8_matmul_workspace(p)
    out = lib.DeviceBuffer(m * n * 4)
    lib.fp8_matmul(dev(lib, np.concatenate([w.ravel(), pad])), dev(lib, ws), dev(lib, np.concatenate([x.ravel(), pad])), dev(lib, xs), out, p, 0,
                   workspace=lib.DeviceBuffer(max(need, 16)), workspace_bytes=need)
    lib.synchronize()
    got = out.download(np.float32).reshape(m, n)
    want = product(x[:1], w[:1], xs[:, :1], ws)[0]
    assert abs(got[0, 0] - want[0, 0]) <= 300 * U * product(x[:1], w[:1], xs[:, :1], ws)[1][0, 0]
    assert np.all(np.isnan(got[0, 1:])) and np.all(np.isnan(got[1:]))


def test_quantized_rows_of_a_matrix(lib):
    """Fp8Matrix over quantised bf16 rows is near the product of the rows
    themselves: each value is off by at most 2^-4 of itself or 2^-10 of its
    block's scale."""
    rng = np.random.default_rng(8)
    m, n, k = 37, 96, 1296
    xb, x = stored(rng.normal(size=(m, k)), "bf16")
    _, w, _, ws = operands(rng, 1, n, k)
    codes, scales, y = lib.DeviceBuffer(m * k), lib.DeviceBuffer(-(-k // 128) * m * 4), lib.DeviceBuffer(m * n * 4)
    lib.fp8_quantize(dev(lib, xb), m, k, codes, scales)
    lib.Fp8Matrix(dev(lib, w), dev(lib, ws), k, n).apply(codes, scales, y, m)
    lib.synchronize()
    c, s = quantized(x, True)
    want, mag = product(c, w, s, ws)
    got = y.download(np.float32).reshape(m, n)
    assert np.all(np.abs(got - want) <= (2 * 128 + 11 + 12) * U * mag)
    wv = e4m3(w, w.shape) * np.repeat(np.repeat(ws.astype(np.float64), 128, 0), 128, 1)[:n, :k]
    step = np.maximum(np.abs(x) * 2.0 ** -4, np.repeat(s.T.astype(np.float64), 128, 1)[:, :k] * 2.0 ** -10)
    assert np.all(np.abs(got - x @ wv.T) <= (step @ np.abs(wv).T) * 1.01)


def test_workspaces_of_a_matrix(lib):
    """K in parts through Fp8Matrix: a captured call keeps its workspace when
    a larger eager one follows, two streams have their own, and one that the
    caller brings is used and checked."""
    rng = np.random.default_rng(21)
    n, k = 72, 784
    x, w, xs, ws = operands(rng, 300, n, k)
    few = np.ascontiguousarray(xs[:, :70])
    want_all, mag_all = product(x, w, xs, ws)
    bound = (256 + len(xs) + 12) * U * mag_all
    W = lib.Fp8Matrix(dev(lib, w), dev(lib, ws), k, n)
    xb, xsb, fewb = dev(lib, x), dev(lib, xs), dev(lib, few)
    y, ya, yb = (lib.DeviceBuffer(m * n * 4) for m in (300, 70, 300))
    a, b = lib.Stream(), lib.Stream()
    with lib.overridden(lib.Knob.FP8, (128, 3)):
        W.apply(xb, fewb, ya, 70, stream=a)
        a.sync()
        graph = lib.Graph(a, lambda: W.apply(xb, fewb, ya, 70, stream=a))
        for _ in range(3):
            ya.upload(np.zeros(70 * n, np.float32), 0)
            W.apply(xb, xsb, y, 300, stream=a)  # grows the stream's workspace
            W.apply(xb, xsb, yb, 300, stream=b)
            graph.launch()
            a.sync()
            b.sync()
            assert np.all(np.abs(ya.download(np.float32).reshape(70, n) - want_all[:70]) <= bound[:70])
            for full in (y, yb):
                assert np.all(np.abs(full.download(np.float32).reshape(300, n) - want_all) <= bound)
        own = lib.DeviceBuffer(lib.fp8_matmul_workspace(lib.Matrix(k, n, 300, 0, 1, 1, 0)))
        y.upload(np.zeros(300 * n, np.float32), 0)
        W.apply(xb, xsb, y, 300, workspace=own)
        lib.synchronize()
        assert np.all(np.abs(y.download(np.float32).reshape(300, n) - want_all) <= bound)
        with pytest.raises(Exception, match="workspace"):
            W.apply(xb, xsb, y, 300, workspace=lib.DeviceBuffer(1024))


@pytest.mark.parametrize("plan", [(0,), (128, 1), (128, 2), (128, 3), (128, 16), (256, 1), (256, 5)])
@pytest.mark.parametrize("m,n,k", [(61, 333, 2064), (64, 40, 1296), (300, 520, 400), (513, 260, 144)])
def test_every_kernel_and_k_split(lib, plan, m, n, k):
    """Each kernel on sizes that the rule would give to another: the few-row
    kernel up to its limit, both tiles at ragged edges, K in parts that are
    not even, of single blocks and of a last block that is not whole."""
    with lib.overridden(lib.Knob.FP8, plan):
        for y_dtype in ("f32", "bf16"):
            check(lib, m, n, k, y_dtype, bias=True)


@pytest.mark.parametrize("m,n", [(520, 8900), (2100, 2600)])
def test_workgroups_that_take_several_tiles(lib, m, n):
    """More tiles than workgroups: a tile's first stage is requested while the
    one before is written (every 37th column is checked)."""
    k = 272
    say("fp8 several tiles", m, n)
    rng = np.random.default_rng(m)
    x, w, xs, ws = operands(rng, m, n, k)
    p = lib.Matrix(k, n, m, 0, 1, 1, 0)
    bufs = [dev(lib, a) for a in (w, ws, x, xs)]
    cols = np.arange(0, n, 37)
    for plan, y_dtype in (((128, 1), "f32"), ((128, 1), "bf16"), ((256, 1), "bf16")):
        out = Guarded(lib, m * n * SIZE[y_dtype])
        with lib.overridden(lib.Knob.FP8, plan):
            lib.fp8_matmul(*bufs, out.ptr, p, CODE[y_dtype])
        lib.synchronize()
        got = values(out.read(np.uint8), y_dtype, (m, n))[:, cols]
        sub = ws[cols // 128]
        want, mag, lost = np.zeros((m, len(cols))), np.zeros((m, len(cols))), 0.0
        xv, wv = e4m3(x, x.shape), e4m3(w, w.shape)[cols]
        for b in range(len(xs)):
            c = slice(128 * b, 128 * b + 128)
            s = xs[b].astype(np.float64)[:, None] * sub[:, b].astype(np.float64)
            want += (xv[:, c] @ wv[:, c].T) * s
            mag += (np.abs(xv[:, c]) @ np.abs(wv[:, c]).T) * s
        if y_dtype != "f32":  # the largest of a group of eight products is at most their sum of magnitudes
            lost = 7 * 2.0 ** -13 * mag
        assert np.all(np.abs(got - want) <= (256 + len(xs) + 12) * U * mag + HALF[y_dtype] * 1.01 * np.abs(want) + lost)


@pytest.mark.parametrize("m,n,k", [(65, 500, 400), (130, 333, 2880), (300, 129, 1296), (600, 513, 272), (1030, 255, 2064)])
@pytest.mark.parametrize("plan", [(), (128, 1), (128, 3), (256, 1)])
def test_f16_outputs_keep_every_bit_of_the_products(lib, m, n, k, plan):
    """f16 rounds at 2^-11, which the bits that the 8-bit matrix instruction
    drops can exceed: f16 outputs are those of the f32 sums, at any number of rows."""
    say("fp8_matmul f16", m, n, k, plan)
    rng = np.random.default_rng(m + n + k)
    x, w, xs, ws = operands(rng, m, n, k)
    xs, ws = xs * np.float32(2.0 ** -8), ws * np.float32(2.0 ** -4)
    want, mag = product(x, w, xs, ws)
    with lib.overridden(lib.Knob.FP8, plan):
        need = lib.fp8_matmul_workspace(lib.Matrix(k, n, m, 0, 1, 1, 0))
        out = Guarded(lib, m * n * 2)
        lib.fp8_matmul(dev(lib, w), dev(lib, ws), dev(lib, x), dev(lib, xs), out.ptr, lib.Matrix(k, n, m, 0, 1, 1, 0), CODE["f16"],
                       workspace=lib.DeviceBuffer(max(need, 16)), workspace_bytes=need)
        lib.synchronize()
    got, fits = values(out.read(np.uint8), "f16", (m, n)), np.abs(want) < 65000
    assert fits.mean() > 0.9
    bound = (2 * 128 + len(xs) + 12) * U * mag + HALF["f16"] * 1.01 * np.abs(want) + LEAST["f16"]  # as check()'s
    assert np.all((np.abs(got - want) <= bound)[fits]), float(np.max(np.abs(got - want)[fits] / bound[fits]))


@pytest.mark.parametrize("exponent", [-100, -108, -110, -115, -118, -121, -124])
def test_blocks_of_tiny_values_are_exact_too(lib, exponent):
    """bf16 rows whose largest value is near the least normal one, with quotients on borders between codes."""
    say("quantize tiny", exponent)
    rng = np.random.default_rng(-exponent)
    rows, k = 64, 256
    x = rng.normal(size=(rows, k)) * 2.0 ** exponent
    top = np.abs(stored(x, "bf16")[1]).reshape(rows, 2, 128).max(2)
    borders = np.concatenate([(2 * np.arange(8, 16) + 1) / 2 * 2.0 ** e for e in range(-9, 5)] + [(2 * np.arange(8) + 1) / 2 * 2.0 ** -9])
    for b in range(2):  # the largest stays the largest
        x[:, 128 * b + 1:128 * b + 100] = top[:, b:b + 1] * rng.choice(borders, (rows, 99)) / 448
        x[:, 128 * b] = top[:, b]
    xb, x = stored(x, "bf16")
    codes, scales = Guarded(lib, rows * k), Guarded(lib, 2 * rows * 4)
    lib.fp8_quantize(dev(lib, xb), rows, k, codes.ptr, scales.ptr, CODE["bf16"])
    lib.synchronize()
    want_codes, want_scales = quantized(x, True)
    np.testing.assert_array_equal(scales.read(np.float32).reshape(2, rows), want_scales)
    np.testing.assert_array_equal(codes.read(np.uint8).reshape(rows, k), want_codes)


@pytest.mark.parametrize("y_dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,plan", [(9, ()), (150, (128, 1)), (150, (128, 2)), (300, (256, 1))])
def test_rows_that_are_not_finite_to_16_bit_outputs(lib, m, plan, y_dtype):
    """A NaN scale, and NaN codes of a row and of a weight row, on the matrix
    instructions of 16-bit outputs; K ends inside a block whose rest is NaN codes."""
    say("fp8 not finite", m, plan, y_dtype)
    rng = np.random.default_rng(m)
    n, k = 144, 400
    x, w, xs, ws = operands(rng, m, n, k)
    xs, ws = xs * np.float32(2.0 ** -8), ws * np.float32(2.0 ** -4)
    xs[1, 3] = np.nan
    x[5, 399], w[143, 0] = 0x7F, 0xFF
    pad = np.full(4096, 0x7F, np.uint8)
    with lib.overridden(lib.Knob.FP8, plan):
        p = lib.Matrix(k, n, m, 0, 1, 1, 0)
        need = lib.fp8_matmul_workspace(p)
        out = Guarded(lib, m * n * 2)
        lib.fp8_matmul(dev(lib, np.concatenate([w.ravel(), pad])), dev(lib, ws), dev(lib, np.concatenate([x.ravel(), pad])), dev(lib, xs), out.ptr, p,
                       CODE[y_dtype], workspace=lib.DeviceBuffer(max(need, 16)), workspace_bytes=need)
        lib.synchronize()
    got = values(out.read(np.uint8), y_dtype, (m, n))
    bad = np.zeros((m, n), bool)
    bad[[3, 5]], bad[:, 143] = True, True
    np.testing.assert_array_equal(np.isnan(got), bad)
