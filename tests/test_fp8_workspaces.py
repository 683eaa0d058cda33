"""The device memory that Fp8Matrix draws for its products, without a GPU: the
buffers and the products are stand-ins, the needs are the library's."""
import ctypes

import pytest

import oco_amd as oco


class Buffer:
    drawn = []

    def __init__(self, nbytes):
        self.nbytes, self.ptr = int(nbytes), 0x1000 * (len(Buffer.drawn) + 1)
        Buffer.drawn.append(self)


class Stream(oco.Stream):
    def __init__(self, handle):
        self.handle, self.scratch = ctypes.c_void_p(handle), oco.Scratch()


@pytest.fixture
def used(monkeypatch):
    """The workspaces of the products, in order; Buffer.drawn: what was allocated."""
    calls, Buffer.drawn = [], []
    monkeypatch.setattr(oco, "DeviceBuffer", Buffer)
    monkeypatch.setattr(oco, "fp8_matmul", lambda w, ws, c, s, y, p, dt, bias, workspace, nbytes, stream: calls.append((workspace, nbytes, need(p))))
    return calls


def need(p):
    return oco.fp8_matmul_workspace(p)


def matrix(n=4096, k=12288):
    return oco.Fp8Matrix(1, 1, k, n)


def apply(m, rows, stream=None):
    m.apply(1, 1, 1, rows, stream=stream)


@pytest.mark.parametrize("n,k", [(4096, 12288), (2880, 4096), (512, 2880)])
def test_rising_rows_keep_a_bounded_total(used, n, k):
    """At most four times the largest need: each buffer is under twice its need and the one before under half of it."""
    m = matrix(n, k)
    for rows in range(1, 2049, 7):
        apply(m, rows)
    assert all(w is None if not want else w.nbytes >= want and b == w.nbytes for w, b, want in used)
    largest = max(want for _, _, want in used)
    assert largest and sum(b.nbytes for b in Buffer.drawn) < 4 * largest


def test_matrices_on_one_stream_share(used):
    """Their products are ordered; other streams have their own."""
    s, t = Stream(5), Stream(6)
    for m in [matrix() for _ in range(10)]:
        apply(m, 200, s)
    assert len(Buffer.drawn) == 1
    apply(matrix(), 200, t)
    assert len(Buffer.drawn) == 2 and used[0][0] is not used[-1][0]


def test_a_stream_that_takes_a_closed_one_s_handle_has_its_own(used):
    m, a = matrix(), Stream(5)
    apply(m, 200, a)
    a.handle = None  # closed; graphs that were captured on it live
    apply(m, 200, Stream(5))
    assert used[0][0] is not used[1][0]


def test_streams_by_handle_and_the_default_one(used):
    m = matrix()
    for s in (None, 7, ctypes.c_void_p(7), None, 7):
        apply(m, 200, s)
    first, seven = used[0][0], used[1][0]
    assert [w for w, _, _ in used] == [first, seven, seven, first, seven] and first is not seven


@pytest.mark.parametrize("stream", [None, 5])
def test_reserved_rows_draw_nothing(used, stream):
    """Needs rise and fall with the rows: a warm-up call with the most rows is not enough, reserve() is."""
    m, s = matrix(), None if stream is None else Stream(stream)
    needs = [need(oco.Matrix(12288, 4096, r, 0, 1, 1, 0)) for r in range(1, 2049)]
    assert needs[-1] < max(needs)
    m.reserve(2048, s)
    drawn = len(Buffer.drawn)
    assert drawn == 1
    for rows in range(2048, 0, -1):
        apply(m, rows, s)
    assert len(Buffer.drawn) == drawn
    few = matrix(72, 64)
    few.reserve(16, s)  # no need, no buffer
    assert len(Buffer.drawn) == drawn
