"""The paged cache in 4 bits in plain numpy: blocks, pages, batches."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """f64 [..., d] -> (codes u8 [..., d], scale bytes u8 [..., d / 32]): the rule of the header, compared level by level."""
    b = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    top = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    with np.errstate(all="ignore"):
        e = np.frexp(np.where(bad, 1.0, top))[1] - 1 - 2 + 127
    e = np.where(top == 0, 1, np.maximum(e, 1))
    v = np.abs(np.where(bad[..., None], 0.0, b)) * np.ldexp(1.0, (127 - e))[..., None]
    far = np.abs(v[..., None] - LEVELS)
    near = far.min(-1, keepdims=True)
    ties = far == near
    # of two levels as near as each other, the one with the even code
    code = np.where(ties[..., 0::2].any(-1), 2 * ties[..., 0::2].argmax(-1), 2 * ties[..., 1::2].argmax(-1) + 1)
    code = np.where(bad[..., None], 0, code + 8 * np.signbit(b))
    return code.reshape(x.shape).astype(np.uint8), np.where(bad, 255, e).astype(np.uint8)


def dequantize(codes, scales):
    v = np.concatenate([LEVELS, -LEVELS])[codes].reshape(codes.shape[:-1] + (codes.shape[-1] // 32, 32))
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return (v * s[..., None]).reshape(codes.shape)


class Pool:
    """Pages as bytes [pages, kv_heads, head bytes], every byte 255 (blocks of NaN) until a token is written."""

    def __init__(self, pages, kv_heads, page_size, d):
        self.pages, self.kv, self.P, self.d = pages, kv_heads, page_size, d
        self.bytes = np.full((pages, kv_heads, page_size * d + page_size * d // 16), 255, np.uint8)

    def put(self, page, t, head, key, value):
        """key, value: (codes, scales) of one token and head."""
        P, d, b = self.P, self.d, self.bytes[page, head]
        low = key[0][0::2] | key[0][1::2] << 4
        b[t * d // 2:(t + 1) * d // 2] = low
        low = value[0][0::2] | value[0][1::2] << 4
        piece = d // 32
        at = P * d // 2 + t // 4 * 2 * d + t % 4 * piece
        for w in range(16):
            b[at + w * 4 * piece:at + w * 4 * piece + piece] = low[w * piece:(w + 1) * piece]
        b[P * d + t * piece:P * d + (t + 1) * piece] = key[1]
        at = P * d + P * piece + t // 4 * 4 * piece + t % 4
        b[at:at + 4 * piece:4] = value[1]


class Batch:
    """Sequences with rows and lengths on pages in any order."""

    def __init__(self, rng, rows, lengths, page_size, spare=2, extra_rows=0):
        self.rows, self.lengths, self.P = list(rows), list(lengths), page_size
        per = [max(1, -(-n // page_size)) for n in lengths]
        self.stride, self.pages = max(per) + 1, sum(per) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(per), self.stride), 0xFFFFFFFF, np.uint32)  # behind a sequence's tokens: no page
        at = 0
        for i, n in enumerate(per):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.uint32)
        self.total = int(self.starts[-1]) + extra_rows

    def place(self, s, t):
        return int(self.table[s, t // self.P]), t % self.P

    def row_positions(self):
        """(sequence, position) of every row that is a sequence's."""
        for s, (n, length) in enumerate(zip(self.rows, self.lengths)):
            for i in range(n):
                yield s, length - n + i

    def describe(self, lib, heads, kv_heads, d, dtype, **over):
        p = dict(head_dim=d, heads=heads, kv_heads=kv_heads, page_size=self.P, pages=self.pages, sequences=len(self.rows), rows=self.total,
                 max_rows=max(self.rows + [1]), max_length=max(self.lengths + [1]), table_stride=self.stride, dtype=dtype)
        p.update(over)
        return lib.Cache(**p)
