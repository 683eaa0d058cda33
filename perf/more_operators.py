"""Performance cases of attention over a paged cache in 4 bits and of what stands before and after it in a decoding step.

Operators that stand beside the library's products, norms and token selection:

- rotate:    rotary positions of query or key rows: pairs in halves or interleaved, part of a head, far positions;
- append:    rotated keys and values quantised into the pages of a cache, queries rotated on the way, and the
             cached rows read back as the values they stand for;
- attention: queries over the cached keys and values: one row per sequence, drafted rows, prompt chunks;
- logits:    penalties for repeated tokens, biases and a grammar's mask on the rows that a token is chosen from.

A page of the cache holds page_size tokens of each key-value head: the keys' codes (E2M1, two values per byte, the
lower four bits first), the values' codes (four tokens together: each 1/16 of a head's width of one token, then of the
next), the keys' scales (E8M0 per 32 values) and the values' scales (four tokens together per 32 values).

listed() names the cases, draw() gives further ones of the same ranges, exact() their results in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False  # true: run() calls the library; false: run() computes the plain form

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}  # oco.DType
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # The queries of one decoded token on their own. Latency alone.
        {"name": "rotate_one_token", "kind": "rotate", "rows": 1, "heads": 32, "head_dim": 128, "dim": 128, "interleaved": False,
         "dtype": "bf16", "far": 4096},
        # A long prompt whose heads turn by half, in adjacent pairs, at far positions: bound by memory.
        {"name": "rotate_prompt_half", "kind": "rotate", "rows": 8192, "heads": 32, "head_dim": 128, "dim": 64, "interleaved": True,
         "dtype": "f16", "far": 131072},
        # One decoding step of a batch: a token of each of 64 sequences.
        {"name": "append_step", "kind": "append", "sequences": 64, "max_rows": 1, "context": 2048, "ragged": True, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dim": 128, "interleaved": False, "dtype": "bf16", "page": 64, "scaled": False},
        # Prompt chunks of different lengths, small heads, frequencies scaled for long contexts, small pages.
        {"name": "append_chunks_ragged", "kind": "append", "sequences": 5, "max_rows": 511, "context": 1500, "ragged": True, "heads": 64,
         "kv_heads": 8, "head_dim": 64, "dim": 64, "interleaved": False, "dtype": "f16", "page": 16, "scaled": True},
        # A long prompt into an empty cache: bound by memory.
        {"name": "append_prompt", "kind": "append", "sequences": 1, "max_rows": 8192, "context": 0, "ragged": False, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dim": 128, "interleaved": False, "dtype": "bf16", "page": 64, "scaled": False},
        # One token of one sequence: few heads, work split along the keys.
        {"name": "attention_one", "kind": "attention", "sequences": 1, "max_rows": 1, "context": 4100, "ragged": False, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "page": 64, "window": 0, "sinks": False},
        # A decoding step of a batch with contexts of all lengths: bound by reading the cache.
        {"name": "attention_batch", "kind": "attention", "sequences": 32, "max_rows": 1, "context": 16384, "ragged": True, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "page": 64, "window": 0, "sinks": False},
        # Four drafted tokens and the last one, small heads with a sink each.
        {"name": "attention_drafts", "kind": "attention", "sequences": 8, "max_rows": 5, "context": 8192, "ragged": True, "heads": 64,
         "kv_heads": 8, "head_dim": 64, "dtype": "bf16", "page": 32, "window": 0, "sinks": True},
        # The second chunk of a long prompt: bound by the matrix cores.
        {"name": "attention_prompt", "kind": "attention", "sequences": 1, "max_rows": 4096, "context": 4096, "ragged": False, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "page": 64, "window": 0, "sinks": False},
        # Ragged prompt chunks with wide heads over a window of keys.
        {"name": "attention_chunks_wide", "kind": "attention", "sequences": 3, "max_rows": 777, "context": 3000, "ragged": True, "heads": 16,
         "kv_heads": 2, "head_dim": 256, "dtype": "f16", "page": 16, "window": 1024, "sinks": False},
        # One row: penalties over the tokens so far and a few biases.
        {"name": "logits_one", "kind": "logits", "rows": 1, "vocabulary": 151936, "dtype": "f32", "history": 512, "biases": 16, "mask": False},
        # A batch under a grammar.
        {"name": "logits_batch_mask", "kind": "logits", "rows": 64, "vocabulary": 151936, "dtype": "f32", "history": 2048, "biases": 32,
         "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "append", "attention", "attention", "attention", "logits"])
    if kind == "rotate":
        d = rng.choice([64, 80, 96, 128, 256])
        heads = rng.choice([2, 8, 14, 32, 64])
        return {"kind": kind, "rows": min(_log(rng, 1, 8192), 8192 * 32 * 128 // (heads * d)), "heads": heads, "head_dim": d,
                "dim": rng.choice([d, d // 2, 2 * rng.randint(1, d // 2)]), "interleaved": rng.random() < 0.5,
                "dtype": rng.choice(["f32", "bf16", "f16"]), "far": _log(rng, 100, 131072)}
    if kind == "logits":
        return {"kind": kind, "rows": _log(rng, 1, 64), "vocabulary": _log(rng, 30000, 151936), "dtype": rng.choice(["f32", "bf16", "f16"]),
                "history": rng.choice([0, _log(rng, 16, 8192)]), "biases": rng.choice([0, _log(rng, 1, 300)]), "mask": rng.random() < 0.5}
    d = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    c = {"kind": kind, "sequences": 1, "max_rows": 1, "context": 0, "ragged": rng.random() < 0.7, "heads": kv * rng.choice([1, 4, 5, 8]),
         "kv_heads": kv, "head_dim": d, "dtype": rng.choice(["bf16", "f16"]), "page": rng.choice([16, 32, 48, 64, 128, 256])}
    if kind == "append":
        c["sequences"] = _log(rng, 1, 64)
        c["max_rows"] = rng.choice([1, max(1, _log(rng, 2, 8192) // c["sequences"])])
        c.update(context=_log(rng, 1, 8192), dim=rng.choice([d, d // 2]), interleaved=rng.random() < 0.5, scaled=rng.random() < 0.5,
                 dtype=rng.choice(["f32", "bf16", "f16"]))
        return c
    if rng.random() < 0.6:  # single tokens and drafts
        c["sequences"], c["max_rows"] = _log(rng, 1, 32), rng.choice([1, 1, 2, 3, 5, 8])
        c["context"] = _log(rng, 1, 16384)
    else:
        c["sequences"] = rng.randint(1, 4)
        c["max_rows"], c["context"] = _log(rng, 9, 2048) // c["sequences"] + 1, _log(rng, 1, 4096)
    c.update(window=rng.choice([0, 0, _log(rng, 16, 4096)]), sinks=rng.random() < 0.4)
    return c


# ---- inputs ---------------------------------------------------------------------------------------------

def _batch(case):
    """Rows of each sequence and tokens in the cache with them, from the sizes alone."""
    q, n, c = case["sequences"], case["max_rows"], case["context"]
    rng = random.Random(q * 1000003 + n * 8191 + c)
    rows = [n if i == 0 or not case["ragged"] else rng.randint(max(1, n // 4), n) for i in range(q)]
    before = [c if i == 0 or not case["ragged"] else rng.randint(c // 8, c) for i in range(q)]
    return rows, [a + b for a, b in zip(rows, before)]


def _frequencies(case):
    """Radians per position of each pair, in 64 bits; scaled: by 8 where a pair turns less than once over 4096 positions, not at
    all where it turns more than 32 times, in between by its place between those two."""
    dim, base = case["dim"], 500000.0
    f = base ** (-np.arange(dim // 2) * 2.0 / dim)
    magnitude = 1.0
    if case.get("scaled"):
        def at(turns):
            return dim * math.log(4096.0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), dim - 1)
        ramp = np.clip((np.arange(dim // 2) - low) / max(high - low, 0.001), 0.0, 1.0)
        f = f / 8.0 * ramp + f * (1.0 - ramp)
        magnitude = 0.1 * math.log(8.0) + 1.0
    return torch.from_numpy(f).cuda(), magnitude


def _page_bytes(case):
    p, d = case["page"], case["head_dim"]
    return p * d + p * d // 16


def _tables(case, gen, lengths):
    """Pages of each sequence in any order, and a few that are nobody's."""
    per = [-(-n // case["page"]) for n in lengths]
    stride, total = max(per), sum(per) + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(per), stride), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    return table, total


def _random_cache(case, gen, pages):
    """Pages of normal values, quantised."""
    p, d, kv = case["page"], case["head_dim"], case["kv_heads"]
    cache = torch.empty((pages, kv, _page_bytes(case)), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (kv * p * d))
    for at in range(0, pages, step):
        part = cache[at:at + step]
        z = torch.randn((len(part), kv, p * d, 2), generator=gen, device="cuda", dtype=torch.bfloat16).mul_(2.4)
        code = torch.zeros(z.shape, dtype=torch.uint8, device="cuda")
        for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
            code += z.abs() > border
        code += 8 * (z < 0)
        part[..., :p * d] = code[..., 0] | code[..., 1] << 4
        # keys of about a quarter, values of about a half, a block in 16 four times as large
        s = torch.randint(0, 16, (len(part), kv, p * d // 16), generator=gen, device="cuda")
        half = p * d // 32
        part[..., p * d:p * d + half] = torch.where(s[..., :half] == 0, 126, 124).to(torch.uint8)
        part[..., p * d + half:] = torch.where(s[..., half:] == 0, 127, 125).to(torch.uint8)
    return cache


def _activations(gen, rows, n):
    """Unit normal rows with a few channels that are much larger, as trained models have them."""
    x = torch.randn((rows, n), generator=gen, device="cuda")
    return x.mul_(1.0 + 15.0 * (torch.rand(n, generator=gen, device="cuda") < 0.005))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 8191 + 71)
    kind, s = case["kind"], {"case": case}
    s["levels"] = torch.tensor(E2M1 + [-v for v in E2M1], device="cuda")
    s["pairs"] = s["levels"][torch.stack((torch.arange(256) & 15, torch.arange(256) >> 4), 1).cuda()]

    def empty(*shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    if kind == "rotate":
        dt = DTYPES[case["dtype"]]
        s["x"] = _activations(gen, case["rows"], case["heads"] * case["head_dim"]).to(dt).view(case["rows"], case["heads"], -1)
        s["positions"] = torch.randint(0, case["far"], (case["rows"],), generator=gen, device="cuda", dtype=torch.int32)
        s["frequencies"], s["magnitude"] = _frequencies(case)
        s["out"] = empty(*s["x"].shape, dtype=dt)
    elif kind in ("append", "attention"):
        dt, h, kv, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
        rows, lengths = _batch(case)
        t = sum(rows)
        s["starts"], s["lengths"] = ints([sum(rows[:i]) for i in range(len(rows) + 1)]), ints(lengths)
        s["total"], s["most"] = t, max(lengths)
        s["table"], s["pages"] = _tables(case, gen, lengths)
        if kind == "append":
            s["cache"] = torch.zeros((s["pages"], kv, _page_bytes(case)), dtype=torch.uint8, device="cuda")
            s["qkv"] = _activations(gen, t, (h + 2 * kv) * d).to(dt)  # as one product of a layer writes them
            s["frequencies"], s["magnitude"] = _frequencies(case)
            s["out"], s["k"], s["v"] = empty(t, h, d, dtype=dt), empty(t, kv, d, dtype=dt), empty(t, kv, d, dtype=dt)
        else:
            s["cache"] = _random_cache(case, gen, s["pages"])
            s["q"] = torch.randn((t, h, d), generator=gen, device="cuda").mul_(3.0).to(dt)
            s["sinks"] = torch.randn(h, generator=gen, device="cuda") if case["sinks"] else None
            s["out"] = empty(t, h, d, dtype=dt)
    else:
        n, v = case["rows"], case["vocabulary"]
        s["logits"] = torch.randn((n, v), generator=gen, device="cuda").mul_(3.0).to(DTYPES[case["dtype"]])
        s["out"] = torch.empty_like(s["logits"])
        s["history"] = s["bias_ids"] = s["mask"] = None
        if case["history"]:  # a few words come again and again
            u = torch.rand((n, case["history"]), generator=gen, device="cuda")
            s["history"] = (u.pow(4) * v).to(torch.int32)
            s["history_lengths"] = torch.randint(1, case["history"] + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)
            s["penalties"] = torch.tensor([1.3, 0.2, 0.4], device="cuda") + 0.1 * torch.rand((n, 3), generator=gen, device="cuda")
        if case["biases"]:  # other places for every row, none twice in one
            first = torch.randint(0, v, (n, 1), generator=gen, device="cuda")
            s["bias_ids"] = ((first + 97 * torch.arange(case["biases"], device="cuda")) % v).to(torch.int32)
            s["biases"] = torch.randn((n, case["biases"]), generator=gen, device="cuda").mul_(5.0)
        if case["mask"]:  # a grammar leaves a run of words here and there
            s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (n, -(-v // 32)), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
            s["mask"] *= torch.rand(s["mask"].shape, generator=gen, device="cuda") < 0.1
    return s


# ---- the library's calls --------------------------------------------------------------------------------

def _ptr(t, at=0):
    return None if t is None else t.data_ptr() + at * t.element_size()


def _kept(s):
    """What a program keeps beside its buffers: the call's description, and a workspace."""
    import oco_amd as oco
    if "oco" in s:
        return oco
    case, s["oco"] = s["case"], True
    kind = case["kind"]
    if kind in ("rotate", "append"):
        s["rotation"] = oco.Rotation(dim=case["dim"], layout=1 if case["interleaved"] else 0, magnitude=s["magnitude"],
                                     frequencies=s["frequencies"].data_ptr())
    if kind in ("append", "attention"):
        width = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"] if kind == "append" else 0
        s["p"] = oco.Cache(head_dim=case["head_dim"], heads=case["heads"], kv_heads=case["kv_heads"], page_size=case["page"],
                           pages=s["pages"], sequences=case["sequences"], rows=s["total"], max_rows=case["max_rows"],
                           max_length=s["most"], table_stride=s["table"].shape[1], dtype=CODES[case["dtype"]],
                           window=case.get("window", 0), q_stride=width, k_stride=width, v_stride=width)
        s["back"] = oco.Cache(**{n: getattr(s["p"], n) for n, _ in oco.Cache._fields_ if not n.endswith("_stride") or n == "table_stride"})
        s["need"] = oco.cache_attention_workspace(s["p"]) if kind == "attention" else 0
        s["workspace"] = torch.empty(max(s["need"], 16), dtype=torch.uint8, device="cuda")
    if kind == "logits":
        s["p"] = oco.Logits(rows=case["rows"], vocabulary=case["vocabulary"], dtype=CODES[case["dtype"]], history_stride=case["history"],
                            bias_stride=case["biases"])
    return oco


def _library(s):
    oco, case = _kept(s), s["case"]
    kind = case["kind"]
    if kind == "rotate":
        oco.rotate(_ptr(s["x"]), case["rows"], case["heads"], case["head_dim"], _ptr(s["out"]), s["rotation"], _ptr(s["positions"]),
                   CODES[case["dtype"]])
        return s["out"]
    if kind == "append":
        q, d = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        oco.cache_append(_ptr(s["cache"]), _ptr(s["table"]), _ptr(s["lengths"]), _ptr(s["qkv"], q), _ptr(s["qkv"], q + d), s["p"],
                         starts=_ptr(s["starts"]), q=_ptr(s["qkv"]), q_out=_ptr(s["out"]), rotation=s["rotation"])
        oco.cache_read(_ptr(s["cache"]), _ptr(s["table"]), _ptr(s["lengths"]), _ptr(s["k"]), _ptr(s["v"]), s["back"],
                       starts=_ptr(s["starts"]))
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    if kind == "attention":
        oco.cache_attention(_ptr(s["q"]), _ptr(s["cache"]), _ptr(s["table"]), _ptr(s["lengths"]), _ptr(s["out"]), s["p"],
                            starts=_ptr(s["starts"]), sinks=_ptr(s["sinks"]), workspace=_ptr(s["workspace"]), workspace_bytes=s["need"])
        return s["out"]
    history, biases = s["history"] is not None, s["bias_ids"] is not None
    oco.logits_adjust(_ptr(s["logits"]), _ptr(s["out"]), s["p"], history=_ptr(s["history"]),
                      history_lengths=_ptr(s["history_lengths"]) if history else None, penalties=_ptr(s["penalties"]) if history else None,
                      bias_ids=_ptr(s["bias_ids"]), biases=_ptr(s["biases"]) if biases else None, mask=_ptr(s["mask"]))
    return s["out"]


# ---- the plain forms ------------------------------------------------------------------------------------

def _turned(x, positions, case, s):
    """Rows [rows, heads, head_dim] by their positions, in 64 bits (far positions, and keys next to a border between two codes)."""
    dim, x = case["dim"], x.double()
    angle = positions.double().unsqueeze(1) * s["frequencies"]
    c, n = (torch.cos(angle) * s["magnitude"]).unsqueeze(1), (torch.sin(angle) * s["magnitude"]).unsqueeze(1)
    part = x[..., :dim]
    a, b = (part[..., 0::2], part[..., 1::2]) if case["interleaved"] else (part[..., :dim // 2], part[..., dim // 2:])
    u, w = a * c - b * n, b * c + a * n
    turned = torch.stack((u, w), -1).flatten(-2) if case["interleaved"] else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., dim:]), -1)


def _places(s):
    """Sequence and position of each row."""
    row = torch.arange(s["total"], device="cuda")
    q = torch.searchsorted(s["starts"].long(), row, right=True) - 1
    return q, row - s["starts"][q + 1] + s["lengths"][q]


def _held(x, s):
    """The values that E2M1 codes with a power of two per 32 stand for."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.clamp(torch.frexp(top).exponent - 3, min=-126).float())
    v = (b / scale).abs()
    code = sum((v > t if even else v >= t).to(torch.uint8) for t, even in
               ((0.25, 1), (0.75, 0), (1.25, 1), (1.75, 0), (2.5, 1), (3.5, 0), (5.0, 1)))
    v = s["levels"][code.int()] * scale
    return torch.where(b < 0, -v, v).flatten(-2)


def _plain_append(s):
    case = s["case"]
    h, kv, d, dt = case["heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    rows = s["qkv"].view(s["total"], h + 2 * kv, d)
    _, positions = _places(s)
    q, k = _turned(rows[:, :h], positions, case, s).to(dt), _turned(rows[:, h:h + kv], positions, case, s).to(dt)
    return {"q": q, "k": _held(k, s).to(dt), "v": _held(rows[:, h + kv:], s).to(dt)}


def _values(codes, scales, s):
    """Bytes of two E2M1 codes [..., d / 2] and E8M0 bytes [..., d / 32] as f32 [..., d]."""
    v = s["pairs"][codes.int()].flatten(-2)
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _cached(s):
    """Keys and values [sequences, kv_heads, tokens, head_dim] in f32."""
    case = s["case"]
    p, d = case["page"], case["head_dim"]
    c = s["cache"][s["table"].long()].transpose(1, 2)  # [sequences, kv_heads, pages, bytes]
    kc, vc, ks, vs = c.split([p * d // 2, p * d // 2, p * d // 32, p * d // 32], -1)
    vc = vc.unflatten(-1, (p // 4, 16, 4, d // 32)).transpose(-3, -2).flatten(-4)
    vs = vs.unflatten(-1, (p // 4, d // 32, 4)).transpose(-2, -1).flatten(-3)
    k = _values(kc.unflatten(-1, (p, d // 2)), ks.unflatten(-1, (p, d // 32)), s)
    v = _values(vc.unflatten(-1, (p, d // 2)), vs.unflatten(-1, (p, d // 32)), s)
    return k.flatten(2, 3), v.flatten(2, 3)


def _plain_attention(s):
    case = s["case"]
    h, kv, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["max_rows"]
    seq, position = _places(s)
    row = torch.arange(s["total"], device="cuda") - s["starts"][seq]
    q = torch.zeros((case["sequences"], n, h, d), device="cuda")
    q[seq, row] = s["q"].float()
    at = torch.full((case["sequences"], n), -1, device="cuda", dtype=torch.int64)
    at[seq, row] = position
    k, v = _cached(s)
    q = q.unflatten(2, (kv, h // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [sequences, kv_heads, rows * group, head_dim]
    score = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= at.unsqueeze(-1)
    if case["window"]:
        seen &= key > at.unsqueeze(-1) - case["window"]
    seen = seen.repeat_interleave(h // kv, 1).unsqueeze(1)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    sink = None
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, kv, 1, h // kv).expand(-1, -1, n, -1).reshape(1, kv, -1, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top > -math.inf, top, 0.0)  # a row of padding sees nothing
    e = torch.exp(score - top)
    total = e.sum(-1, keepdim=True) + (torch.exp(sink - top) if sink is not None else 0.0)
    out = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)
    out = out.unflatten(2, (n, h // kv)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out[seq, row].to(DTYPES[case["dtype"]])


def _plain_logits(s):
    case, x = s["case"], s["logits"].float()
    n, v = x.shape
    if s["history"] is not None:
        live = torch.arange(case["history"], device="cuda") < s["history_lengths"].unsqueeze(1)
        count = torch.zeros((n, v), device="cuda").scatter_add_(1, s["history"].long(), live.float())
        repetition, frequency, presence = s["penalties"].unsqueeze(-1).unbind(1)
        y = torch.where(x > 0, x / repetition, x * repetition) - (frequency * count + presence)
        x = torch.where(count > 0, y, x)
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["biases"])
    if s["mask"] is not None:
        bit = (s["mask"].unsqueeze(-1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = torch.where(bit.flatten(1)[:, :v] > 0, x, -math.inf)
    return x.to(s["logits"].dtype)


def run(s):
    if own:
        return _library(s)
    kind = s["case"]["kind"]
    if kind == "rotate":
        return _turned(s["x"], s["positions"], s["case"], s).to(s["x"].dtype)
    return {"append": _plain_append, "attention": _plain_attention, "logits": _plain_logits}[kind](s)


# ---- what a pass has to do ------------------------------------------------------------------------------

SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def work(case):
    kind, z = case["kind"], SIZE[case["dtype"]]
    if kind == "rotate":
        values = case["rows"] * case["heads"] * case["head_dim"]
        return {"bytes": 2 * values * z + 4 * case["rows"] + 4 * case["dim"], "flops": 3 * values * case["dim"] // case["head_dim"]}
    if kind == "logits":
        n, v = case["rows"], case["vocabulary"]
        byte = 2 * n * v * z + n * (2 * case["history"] + 8 * case["biases"] + case["mask"] * (v // 8))
        return {"bytes": byte, "flops": n * (v + 4 * case["history"] + case["biases"])}
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    rows, lengths = _batch(case)
    t = sum(rows)
    if kind == "append":
        byte = t * d * z * (2 * h + 4 * kv) + t * kv * (d + d // 16) + 4 * case["dim"]
        return {"bytes": byte, "flops": t * (3 * (h + kv) * case["dim"] + 6 * kv * d)}
    window, keys, seen = case["window"], 0, 0
    for n, length in zip(rows, lengths):
        far = window or length
        keys += min(length, far + n - 1)
        seen += sum(min(at + 1, far) for at in range(length - n, length))
    return {"bytes": keys * kv * (d + d // 16) + 2 * t * h * d * z, "flops": 4 * seen * h * d}


# ---- results in 64 bits ---------------------------------------------------------------------------------

def _exact_turn(x, positions, case, s):
    """Pairs as complex numbers."""
    dim, y = case["dim"], x.double().clone()
    angle = torch.outer(positions.double(), s["frequencies"])
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, None, :]
    first = slice(0, dim, 2) if case["interleaved"] else slice(0, dim // 2)
    second = slice(1, dim, 2) if case["interleaved"] else slice(dim // 2, dim)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_held(x):
    """Nearest E2M1 value of each block of 32 (ties: the even code), the block's largest between 4 and 8."""
    rows, h, d = x.shape
    out = torch.zeros((rows, h, d), dtype=torch.float64, device="cuda")
    for b in range(d // 32):
        part = x[..., 32 * b:32 * b + 32].double()
        power = torch.exp2(torch.clamp(torch.floor(torch.log2(part.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -149))) - 2.0, min=-126.0))
        v = part / power
        step = torch.where(v.abs() < 2.0, 0.5, torch.where(v.abs() < 4.0, 1.0, 2.0))
        out[..., 32 * b:32 * b + 32] = torch.clamp(torch.round(v / step) * step, -6.0, 6.0) * power
    return out


def _rows_of(s):
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    return [(i, slice(starts[i], starts[i + 1]), lengths[i]) for i in range(len(lengths))]


def _exact_append(s):
    case = s["case"]
    h, kv, d, dt = case["heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    x = s["qkv"].view(s["total"], -1, d)
    place = torch.cat([torch.arange(n - (r.stop - r.start), n, device="cuda") for _, r, n in _rows_of(s)])
    # the cache takes the keys as the model's type holds them
    return {"q": _exact_turn(x[:, :h], place, case, s), "k": _exact_held(_exact_turn(x[:, h:h + kv], place, case, s).to(dt)),
            "v": _exact_held(x[:, h + kv:])}


def _exact_cache(s, sequence, head, tokens):
    """Keys and values of one head of one sequence, code by code."""
    case = s["case"]
    p, d = case["page"], case["head_dim"]
    t = torch.arange(tokens, device="cuda")
    pages, within = s["table"][sequence].long()[t // p], t % p
    byte = s["cache"].view(s["pages"], case["kv_heads"], -1)[:, head]
    level = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    c = torch.arange(d, device="cuda")

    def numbers(at, scale_at, column):
        code = (byte[pages[:, None], at].int() >> (4 * (column % 2)).int()) & 15
        power = torch.exp2(byte[pages[:, None], scale_at].double() - 127.0)
        return torch.where(code >= 8, -1.0, 1.0) * level[(code & 7).long()] * power

    w = within[:, None]
    k = numbers(w * (d // 2) + c // 2, p * d + w * (d // 32) + c // 32, c)
    piece = c // (d // 16)
    v_at = p * d // 2 + (w // 4) * (2 * d) + piece * (d // 8) + (w % 4) * (d // 32) + (c % (d // 16)) // 2
    v = numbers(v_at, p * d + p * d // 32 + (w // 4) * (d // 8) + (c // 32) * 4 + w % 4, c)
    return k, v


def _exact_attention(s):
    case = s["case"]
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, r, n in _rows_of(s):
        place = torch.arange(n - (r.stop - r.start), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None, :]
        hidden = key > place
        if case["window"]:
            hidden = hidden | (key <= place - case["window"])
        for g in range(kv):
            k, v = _exact_cache(s, i, g, n)
            for j in range(g * (h // kv), (g + 1) * (h // kv)):
                z = (s["q"][r, j].double() @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
                if s["sinks"] is not None:
                    z = torch.cat((z, s["sinks"][j].double().expand(len(z), 1)), 1)
                out[r, j] = torch.softmax(z, 1)[:, :n] @ v
    return out


def _exact_logits(s):
    case, x = s["case"], s["logits"].double().cpu().numpy()
    v = case["vocabulary"]
    for i in range(case["rows"]):
        if s["history"] is not None:
            ids, count = np.unique(s["history"][i, :int(s["history_lengths"][i])].cpu().numpy(), return_counts=True)
            r, f, p = s["penalties"][i].double().tolist()
            x[i, ids] = np.where(x[i, ids] > 0, x[i, ids] / r, x[i, ids] * r) - f * count - p
        if s["bias_ids"] is not None:
            x[i, s["bias_ids"][i].cpu().numpy()] += s["biases"][i].double().cpu().numpy()
        if s["mask"] is not None:
            bits = np.unpackbits(s["mask"][i].cpu().numpy().view(np.uint8), bitorder="little")[:v]
            x[i, bits == 0] = -np.inf
    return torch.from_numpy(x)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotate":
        return _exact_turn(s["x"], s["positions"], case, s)
    return {"append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["kind"]](s)
