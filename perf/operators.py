"""Performance cases of the operators around a routed, 8-bit, speculatively decoded model step.

Four operators that stand beside the library's norms, products, routing and greedy selection:

- blocks:   the norms on either side of a block, its gate, its scale and the residual add in one pass,
            with the rows of the next product already in 8-bit floating point;
- products: rows in 8-bit floating point (a scale per 128 columns) times weights with a scale per block of 128 x 128;
- routing:  experts chosen by softmax or sigmoid scores, a balance bias and groups;
- drafts:   drafted tokens verified against the target's distribution, from given random numbers.

listed() names the cases, draw() gives further ones of the same ranges, exact() their results in 64 bits.
"""
import math

import numpy as np
import torch

own = False  # true: run() calls the library; false: run() computes the plain form

EPSILON = 1e-6
E4M3_MAX = 448.0
NONE = 0xFFFFFFFF - (1 << 32)  # "no token", as an int32 holds it
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}  # oco.DType
GATES = {"none": 0, "linear": 1, "sigmoid": 2, "tanh": 3}  # oco.Gate


def listed():
    return [
        # Residual step of one decoded token: post-norm, per-channel gate, add, next norm. Latency alone.
        {"name": "block_one_row", "kind": "block", "rows": 1, "n": 4096, "x": "bf16", "y": "bf16", "gate": "linear",
         "gate_rows": 0, "codes": False},
        # A prompt chunk of a model with an f32 residual stream and a gate per row, feeding an 8-bit product.
        {"name": "block_chunk_gated", "kind": "block", "rows": 512, "n": 2880, "x": "f32", "y": "bf16", "gate": "sigmoid",
         "gate_rows": 1, "codes": True},
        # A long prompt: four row passes, bound by memory.
        {"name": "block_prompt", "kind": "block", "rows": 8192, "n": 4096, "x": "bf16", "y": "bf16", "gate": "linear",
         "gate_rows": 0, "codes": False},
        # One token's attention output projection: the smallest product, quantisation included.
        {"name": "fp8_one_row", "kind": "product", "m": 1, "n": 2880, "k": 4096, "x": "bf16", "y": "bf16"},
        # lm_head over eight drafted tokens in f32: bound by reading the weights.
        {"name": "fp8_head_8_rows", "kind": "product", "m": 8, "n": 151936, "k": 4096, "x": "bf16", "y": "f32"},
        # Down projection of a ragged prompt chunk.
        {"name": "fp8_prompt_ragged", "kind": "product", "m": 1999, "n": 4096, "k": 12288, "x": "bf16", "y": "f32"},
        # Gate or up projection of a long prompt: bound by the matrix cores.
        {"name": "fp8_prompt", "kind": "product", "m": 4096, "n": 12288, "k": 4096, "x": "bf16", "y": "bf16"},
        # The router of one decoded token: softmax over 128 experts, eight chosen and renormalised.
        {"name": "route_one_token", "kind": "route", "tokens": 1, "experts": 128, "k": 8, "score": "softmax", "groups": 1,
         "kept": 1, "top2": False, "bias": False, "x": "f32"},
        # The router of a long prompt: sigmoid scores, a balance bias, four of eight groups by their two best.
        {"name": "route_prompt_groups", "kind": "route", "tokens": 8192, "experts": 256, "k": 8, "score": "sigmoid",
         "groups": 8, "kept": 4, "top2": True, "bias": True, "x": "f32"},
        # One sequence with four drafts: logits of the target, probabilities that the drafter kept.
        {"name": "draft_one", "kind": "draft", "sequences": 1, "drafts": 4, "vocabulary": 151936, "target": "f32",
         "draft": "probabilities", "temperature": 1.0, "ragged": False},
        # Eight sequences with drafts looked up in the prompt (no distribution), of different lengths, bf16 logits.
        {"name": "draft_lookup_ragged", "kind": "draft", "sequences": 8, "drafts": 5, "vocabulary": 100003, "target": "bf16",
         "draft": "none", "temperature": 0.7, "ragged": True},
        # A full batch: logits on both sides.
        {"name": "draft_batch", "kind": "draft", "sequences": 32, "drafts": 7, "vocabulary": 151936, "target": "f32",
         "draft": "logits", "temperature": 0.8, "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["block", "product", "product", "route", "draft"])
    if kind == "block":
        n = _log(rng, 256, 12288)
        n = n if rng.random() < 0.3 else -(-n // 16) * 16
        x = rng.choice(["bf16", "f32", "f16"])
        return {"kind": kind, "rows": max(1, min(_log(rng, 1, 8192), 8192 * 4096 // (2 * n))), "n": n, "x": x,
                "y": "f16" if x == "f16" else "bf16", "gate": rng.choice(["none", "linear", "sigmoid", "tanh"]),
                "gate_rows": rng.choice([0, 1, 7]), "codes": n % 16 == 0 and x == "f32"}
    if kind == "product":
        m, n, k = _log(rng, 1, 4096), _log(rng, 256, 12288), -(-_log(rng, 512, 12288) // 16) * 16
        while m * n * k > 4096 * 12288 * 4096:
            m = (m + 1) // 2
        return {"kind": kind, "m": m, "n": n, "k": k, "x": rng.choice(["bf16", "f16"]), "y": rng.choice(["bf16", "f32"])}
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * rng.randint(max(2, 16 // groups), 256 // groups)
        kept = groups if groups == 1 else rng.randint(max(1, groups // 4), groups - 1)
        return {"kind": kind, "tokens": _log(rng, 1, 8192), "experts": experts,
                "k": rng.randint(1, min(8, kept * experts // groups)), "score": rng.choice(["softmax", "sigmoid"]),
                "groups": groups, "kept": kept, "top2": rng.random() < 0.5, "bias": rng.random() < 0.6,
                "x": rng.choice(["f32", "bf16"])}
    return {"kind": kind, "sequences": _log(rng, 1, 32), "drafts": rng.randint(1, 7), "vocabulary": _log(rng, 30000, 151936),
            "target": rng.choice(["f32", "bf16"]), "draft": rng.choice(["none", "probabilities", "logits"]),
            "temperature": rng.choice([0.0, 0.6, 1.0]), "ragged": rng.random() < 0.5}


# ---- inputs ---------------------------------------------------------------------------------------------

def _activations(gen, rows, n):
    """Unit normal rows with a few channels that are much larger, as trained models have them."""
    x = torch.randn((rows, n), generator=gen, device="cuda")
    return x.mul_(1.0 + 15.0 * (torch.rand(n, generator=gen, device="cuda") < 0.005))


def _block_weights(gen, n, k):
    """Normal weights rounded to e4m3 with a scale per block of 128 x 128."""
    nb, kb = -(-n // 128), -(-k // 128)
    codes = torch.empty((n, k), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((nb, kb), device="cuda")
    step = max(1, (1 << 27) // (128 * k))  # block rows at a time: the values pass through f32
    for at in range(0, nb, step):
        end = min(nb, at + step)
        w = torch.zeros(((end - at) * 128, kb * 128), device="cuda")
        live = codes[at * 128:end * 128]
        w[:len(live), :k] = torch.randn((len(live), k), generator=gen, device="cuda").mul_(0.02)
        b = w.view(end - at, 128, kb, 128)
        scales[at:end] = b.abs().amax((1, 3)) / E4M3_MAX
        w = (b / scales[at:end].view(end - at, 1, kb, 1)).view(-1, kb * 128)
        live.copy_(w[:len(live), :k])
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 8191 + 29)
    kind, s = case["kind"], {"case": case}

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if kind == "block":
        rows, n, xt, yt = case["rows"], case["n"], DTYPES[case["x"]], DTYPES[case["y"]]
        s["x"], s["y"] = (4.0 * _activations(gen, rows, n)).to(xt), _activations(gen, rows, n).to(yt)
        shared = rows if case["gate_rows"] == 0 else case["gate_rows"]
        s["gate"] = None if case["gate"] == "none" else torch.randn((-(-rows // shared), n), generator=gen, device="cuda").to(yt)
        s["post"] = 1.0 + 0.1 * torch.randn(n, generator=gen, device="cuda")
        s["pre"] = 1.0 + 0.1 * torch.randn(n, generator=gen, device="cuda")
        s["x_out"], s["out"] = empty(rows, n, dtype=xt), empty(rows, n, dtype=yt)
        if case["codes"]:
            s["codes"], s["scales"] = empty(rows, n, dtype=torch.float8_e4m3fn), empty(-(-n // 128), rows)
    elif kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["w"], s["w_scales"] = _block_weights(gen, n, k)
        s["x"] = _activations(gen, m, k).to(DTYPES[case["x"]])
        s["codes"], s["scales"] = empty(m, k, dtype=torch.float8_e4m3fn), empty(-(-k // 128), m)
        s["out"] = empty(m, n, dtype=DTYPES[case["y"]])
    elif kind == "route":
        t, e = case["tokens"], case["experts"]
        s["logits"] = torch.randn((t, e), generator=gen, device="cuda").to(DTYPES[case["x"]])
        s["bias"] = 0.05 * torch.randn(e, generator=gen, device="cuda") if case["bias"] else None
        s["ids"], s["weights"] = empty(t, case["k"], dtype=torch.int32), empty(t, case["k"])
    else:
        q, d, v = case["sequences"], case["drafts"], case["vocabulary"]
        target = torch.randn((q, d + 1, v), generator=gen, device="cuda").mul_(3.0)
        # the drafter's logits are the target's with noise; its tokens are drawn from its own distribution
        draft = target[:, :d] + torch.randn((q, d, v), generator=gen, device="cuda").mul_(0.7)
        u = torch.rand((q, d, v), generator=gen, device="cuda").clamp_(1e-12, 1.0 - 1e-7)
        noisy = draft / max(case["temperature"], 1e-3) - torch.log(-torch.log(u))
        s["tokens_in"] = noisy.argmax(-1).to(torch.int32)
        s["target"] = target.to(DTYPES[case["target"]])
        s["draft"] = None
        if case["draft"] == "logits":
            s["draft"] = draft
        elif case["draft"] == "probabilities":
            s["draft"] = torch.softmax(draft / max(case["temperature"], 1e-3), -1)
        s["uniforms"] = torch.rand((q, d + 1), generator=gen, device="cuda")
        s["lengths"] = torch.randint(0, d + 1, (q,), generator=gen, device="cuda", dtype=torch.int32) if case["ragged"] else None
        s["accepted"], s["tokens"] = empty(q, dtype=torch.int32), empty(q, d + 1, dtype=torch.int32)
        s["probabilities"] = empty(q, d + 1)
    return s


# ---- the library's calls --------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _kept(s):
    """What a program keeps beside its buffers: the call's description, and a workspace."""
    import oco_amd as oco
    if "oco" in s:
        return oco
    case, s["oco"] = s["case"], True
    kind, need = case["kind"], 0
    if kind == "block":
        s["p"] = oco.Block(rows=case["rows"], n=case["n"], x_dtype=CODES[case["x"]], dtype=CODES[case["y"]],
                           gate=GATES[case["gate"]], gate_rows=case["gate_rows"], scale=0.5, epsilon=EPSILON)
    elif kind == "product":
        s["p"] = oco.Matrix(case["k"], case["n"], case["m"], 0, 1, 1, 0)
        need = oco.fp8_matmul_workspace(s["p"])
    elif kind == "route":
        s["p"] = oco.Routing(experts=case["experts"], k=case["k"], score=1 if case["score"] == "sigmoid" else 0,
                             groups=case["groups"], groups_kept=case["kept"], group_rank=1 if case["top2"] else 0,
                             renormalize=1, scale=2.5)
    else:
        s["p"] = oco.Draft(sequences=case["sequences"], drafts=case["drafts"], vocabulary=case["vocabulary"],
                           target_values=0, draft_values=1 if case["draft"] == "probabilities" else 0,
                           target_dtype=CODES[case["target"]], draft_dtype=0, temperature=case["temperature"])
        need = oco.draft_verify_workspace(s["p"])
    s["need"] = need
    s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return oco


def _library(s):
    oco, case = _kept(s), s["case"]
    kind = case["kind"]
    if kind == "block":
        codes, scales = s.get("codes"), s.get("scales")
        oco.block_norm(_ptr(s["x"]), _ptr(s["y"]), s["p"], x_out=_ptr(s["x_out"]), gate=_ptr(s["gate"]), post_w=_ptr(s["post"]),
                       pre_w=_ptr(s["pre"]), out=_ptr(s["out"]), codes=_ptr(codes), scales=_ptr(scales))
        return {"x": s["x_out"], "out": s["out"], "codes": codes, "scales": scales}
    if kind == "product":
        oco.fp8_quantize(_ptr(s["x"]), case["m"], case["k"], _ptr(s["codes"]), _ptr(s["scales"]), CODES[case["x"]])
        oco.fp8_matmul(_ptr(s["w"]), _ptr(s["w_scales"]), _ptr(s["codes"]), _ptr(s["scales"]), _ptr(s["out"]), s["p"],
                       CODES[case["y"]], workspace=_ptr(s["workspace"]), workspace_bytes=s["need"])
        return {"codes": s["codes"], "scales": s["scales"], "y": s["out"]}
    if kind == "route":
        oco.route_scores(_ptr(s["logits"]), case["tokens"], s["p"], _ptr(s["ids"]), _ptr(s["weights"]), CODES[case["x"]],
                         bias=_ptr(s["bias"]))
        return {"ids": s["ids"], "weights": s["weights"]}
    oco.draft_verify(_ptr(s["target"]), _ptr(s["draft"]), _ptr(s["tokens_in"]), _ptr(s["uniforms"]), _ptr(s["accepted"]),
                     _ptr(s["tokens"]), s["p"], lengths=_ptr(s["lengths"]), probabilities=_ptr(s["probabilities"]),
                     workspace=_ptr(s["workspace"]), workspace_bytes=s["need"])
    return {"accepted": s["accepted"], "tokens": s["tokens"], "probabilities": s["probabilities"]}


# ---- the plain forms ------------------------------------------------------------------------------------

def _rms(v, w):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPSILON) * w


def _quantized(x):
    """448 x / max|x| in e4m3 and the scale max|x| / 448 per 128 columns, scales as [block][row].  With 448 as
    0.875 * 512 the quotient's operands are exact for 16-bit x, so a quotient on a border stays there."""
    rows, k = x.shape
    kb = -(-k // 128)
    b = torch.nn.functional.pad(x.float(), (0, kb * 128 - k)).view(rows, kb, 128)
    top = b.abs().amax(-1).clamp_min(E4M3_MAX * 2.0 ** -126)
    codes = ((b * 0.875) / (top / 512.0).unsqueeze(-1)).view(rows, kb * 128)[:, :k].to(torch.float8_e4m3fn)
    return codes, (top / E4M3_MAX).T.contiguous()


def _spread(codes, row_scales):
    """e4m3 codes times a scale per row and 128 columns, in f32."""
    return codes.float() * row_scales.repeat_interleave(128, 1)[:, :codes.shape[1]]


def _plain_block(s):
    case, x, v = s["case"], s["x"].float(), _rms(s["y"].float(), s["post"])
    if s["gate"] is not None:
        g = s["gate"].float()
        g = torch.sigmoid(g) if case["gate"] == "sigmoid" else torch.tanh(g) if case["gate"] == "tanh" else g
        shared = case["gate_rows"] or case["rows"]
        v = v * (g if len(g) == 1 else g.repeat_interleave(shared, 0)[:case["rows"]])
    x_out = (x + 0.5 * v).to(s["x"].dtype)
    out = _rms(x_out.float(), s["pre"])
    codes, scales = _quantized(out) if case["codes"] else (None, None)
    return {"x": x_out, "out": out.to(s["y"].dtype), "codes": codes, "scales": scales}


def _plain_product(s):
    codes, scales = _quantized(s["x"])
    w = _spread(s["w"], s["w_scales"].repeat_interleave(128, 0)[:s["case"]["n"]])
    y = torch.matmul(_spread(codes, scales.T), w.T)
    return {"codes": codes, "scales": scales, "y": y.to(DTYPES[s["case"]["y"]])}


def _first(values, k):
    """The k largest of each row in order, ties to the lowest index."""
    return torch.sort(values, dim=-1, descending=True, stable=True).indices[..., :k]


def _plain_route(s):
    case, z = s["case"], s["logits"].double()  # choices next to a border need 64 bits
    t, e, g = case["tokens"], case["experts"], case["groups"]
    if case["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-z))
    else:
        score = torch.exp(z - z.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    choice = score if s["bias"] is None else score + s["bias"].double()
    if g > 1:
        by_group = choice.view(t, g, e // g)
        rank = by_group.topk(min(2, e // g), -1).values.sum(-1) if case["top2"] else by_group.amax(-1)
        kept = torch.zeros((t, g), dtype=torch.bool, device="cuda").scatter_(1, _first(rank, case["kept"]), True)
        choice = torch.where(kept.unsqueeze(-1), by_group, -math.inf).view(t, e)
    ids = _first(choice, case["k"])
    w = score.gather(1, ids)
    w = 2.5 * w / w.sum(-1, keepdim=True)
    return {"ids": ids.to(torch.int32), "weights": w.float()}


def _distribution(values, temperature):
    v = values.double()
    if temperature == 0.0:
        return torch.nn.functional.one_hot(_first_max(v), v.shape[-1]).double()
    v = torch.exp((v - v.amax(-1, keepdim=True)) / temperature)
    return v / v.sum(-1, keepdim=True)


def _first_max(v):
    return (v == v.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1)


def _plain_draft(s):
    case = s["case"]
    q, d, v = case["sequences"], case["drafts"], case["vocabulary"]
    row = torch.arange(q, device="cuda")
    length = torch.full((q,), d, device="cuda") if s["lengths"] is None else s["lengths"].long()
    ids, u = s["tokens_in"].long(), s["uniforms"].double()
    p = _distribution(s["target"], case["temperature"])
    p_id = p[:, :d].gather(2, ids.unsqueeze(2)).squeeze(2)
    # in 64 bits: an accepted token or the place where a running sum passes a number must not hang on a rounding
    if s["draft"] is None or case["temperature"] == 0.0:
        dist, q_id = None, torch.ones_like(p_id)
    else:
        dist = s["draft"].double() if case["draft"] == "probabilities" else _distribution(s["draft"], case["temperature"])
        q_id = dist.gather(2, ids.unsqueeze(2)).squeeze(2)
    place = torch.arange(d, device="cuda")
    good = (u[:, :d] * q_id < p_id) & (place < length.unsqueeze(1))
    accepted = good.long().cumprod(1).sum(1)
    last = p[row, accepted]
    stopped = (accepted < length).unsqueeze(1)  # a draft was refused: what is left of the target's distribution
    at = accepted.clamp_max(d - 1)
    minus = torch.nn.functional.one_hot(ids[row, at], v).double() if dist is None else dist[row, at]
    rest = torch.where(stopped, (last - minus).clamp_min(0.0), last)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, last)
    sums = rest.cumsum(1)
    mark = u[:, d:] * sums[:, -1:]
    token = ((sums > mark) & (rest > 0)).to(torch.uint8).argmax(1)
    place = torch.arange(d + 1, device="cuda")
    padded = torch.nn.functional.pad(ids, (0, 1))
    tokens = torch.where(place < accepted.unsqueeze(1), padded, NONE)
    tokens = torch.where(place == accepted.unsqueeze(1), token.unsqueeze(1), tokens)
    probability = p.gather(2, tokens.clamp_min(0).unsqueeze(2)).squeeze(2)
    probability = torch.where(place <= accepted.unsqueeze(1), probability, 0.0)
    return {"accepted": accepted.to(torch.int32), "tokens": tokens.to(torch.int32), "probabilities": probability.float()}


def run(s):
    if own:
        return _library(s)
    return {"block": _plain_block, "product": _plain_product, "route": _plain_route, "draft": _plain_draft}[s["case"]["kind"]](s)


# ---- what a pass has to do ------------------------------------------------------------------------------

SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def work(case):
    kind = case["kind"]
    if kind == "block":
        rows, n, x, y = case["rows"], case["n"], SIZE[case["x"]], SIZE[case["y"]]
        gates = 0 if case["gate"] == "none" else -(-rows // (case["gate_rows"] or rows))
        byte = rows * n * (2 * x + 2 * y) + gates * n * y + 8 * n
        byte += rows * (n + 4 * -(-n // 128)) if case["codes"] else 0
        return {"bytes": byte, "flops": rows * n * (12 + 3 * (case["gate"] != "none") + 3 * case["codes"])}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // 128)
        byte = n * k + 4 * -(-n // 128) * kb + m * k * (SIZE[case["x"]] + 1) + 4 * m * kb + m * n * SIZE[case["y"]]
        return {"bytes": byte, "flops": 2 * m * n * k + 3 * m * k}
    if kind == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        return {"bytes": t * e * SIZE[case["x"]] + 8 * t * k + 4 * e * case["bias"], "flops": t * e * (12 + k)}
    q, d, v = case["sequences"], case["drafts"], case["vocabulary"]
    rows = d / 2 + 1 if case["ragged"] else d + 1  # the rows of a sequence's own drafts
    drafts = {"none": 0, "probabilities": 1, "logits": rows - 1}[case["draft"]] * (case["temperature"] > 0)
    byte = q * v * (rows * SIZE[case["target"]] + 4 * drafts) + q * (d + 1) * 16
    return {"bytes": int(byte), "flops": int(q * v * (rows + drafts) * 4)}


# ---- results in 64 bits ---------------------------------------------------------------------------------

def _exact_codes(x):
    """The e4m3 values (round to nearest, ties to even) and scales of 64-bit rows."""
    rows, k = x.shape
    codes, scales = torch.empty_like(x), torch.empty((-(-k // 128), rows), dtype=torch.float64, device="cuda")
    for b in range(len(scales)):
        part = x[:, 128 * b:128 * b + 128]
        top = torch.clamp(part.abs().amax(1), min=448.0 * 2.0 ** -126)
        scales[b] = top / 448.0
        v = part * 448.0 / top.unsqueeze(1)
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=1e-30))), min=-6.0) - 3.0)
        codes[:, 128 * b:128 * b + 128] = torch.clamp(torch.round(v / step) * step, -448.0, 448.0)
    return codes, scales


def _exact_block(s):
    case, d = s["case"], torch.float64
    y = s["y"].to(d)
    y = y / torch.sqrt((y * y).sum(1, keepdim=True) / case["n"] + EPSILON) * s["post"].to(d)
    if s["gate"] is not None:
        g = s["gate"].to(d)
        if case["gate"] == "sigmoid":
            g = 1.0 / (1.0 + torch.exp(-g))
        elif case["gate"] == "tanh":
            g = 1.0 - 2.0 / (torch.exp(2.0 * g) + 1.0)
        which = torch.arange(case["rows"], device="cuda") // (case["gate_rows"] or case["rows"])
        y = y * g[which]
    x = s["x"].to(d) + 0.5 * y
    kept = x.to(s["x"].dtype).to(d)  # the residual stream holds rounded rows, and the norm reads those
    out = kept / torch.sqrt((kept * kept).sum(1, keepdim=True) / case["n"] + EPSILON) * s["pre"].to(d)
    codes, scales = _exact_codes(out) if case["codes"] else (None, None)
    return {"x": x, "out": out, "codes": codes, "scales": scales}


def _exact_product(s):
    case = s["case"]
    codes, scales = _exact_codes(s["x"].double())
    y = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
    for b in range(len(scales)):
        cols = slice(128 * b, 128 * b + 128)
        rows = torch.arange(case["n"], device="cuda") // 128
        y += (codes[:, cols] @ s["w"][:, cols].double().T) * scales[b].unsqueeze(1) * s["w_scales"][rows, b].double()
    return {"codes": codes, "scales": scales, "y": y}


def _exact_route(s):
    case, z = s["case"], s["logits"].double().cpu().numpy()
    if case["score"] == "sigmoid":
        score = 0.5 + 0.5 * np.tanh(0.5 * z)
    else:
        top = z.max(1, keepdims=True)
        score = np.exp(z - (top + np.log(np.exp(z - top).sum(1, keepdims=True))))
    choice = score + (0.0 if s["bias"] is None else s["bias"].double().cpu().numpy())
    size = case["experts"] // case["groups"]
    if case["groups"] > 1:
        best = -np.sort(-choice.reshape(-1, case["groups"], size), axis=2)
        rank = best[:, :, :2].sum(2) if case["top2"] else best[:, :, 0]
        out = np.argsort(-rank, axis=1, kind="stable")[:, case["kept"]:]
        for j in range(out.shape[1]):
            gone = out[:, j:j + 1] * size + np.arange(size)
            np.put_along_axis(choice, gone, -np.inf, 1)
    ids = np.argsort(-choice, axis=1, kind="stable")[:, :case["k"]]
    w = np.take_along_axis(score, ids, 1)
    return {"ids": torch.from_numpy(ids).int(), "weights": torch.from_numpy(2.5 * w / w.sum(1, keepdims=True))}


def _exact_row(values, temperature):
    z = values.double()
    if temperature == 0.0:
        row = torch.zeros_like(z)
        row[int(torch.nonzero(z == z.max())[0])] = 1.0
        return row
    return torch.softmax(z / temperature, 0)


def _exact_draft(s):
    case = s["case"]
    q, d, t = case["sequences"], case["drafts"], case["temperature"]
    ids, u = s["tokens_in"].tolist(), s["uniforms"].double().tolist()
    accepted, tokens, chances = [], [], []
    for i in range(q):
        length = d if s["lengths"] is None else int(s["lengths"][i])
        emitted, chance = [], []
        for j in range(length + 1):
            p, rest = _exact_row(s["target"][i, j], t), None
            if j < length:
                token = ids[i][j]
                if s["draft"] is None or t == 0.0:
                    other = torch.zeros_like(p)
                    other[token] = 1.0
                else:
                    other = s["draft"][i, j].double() if case["draft"] == "probabilities" else _exact_row(s["draft"][i, j], t)
                if u[i][j] * float(other[token]) < float(p[token]):
                    emitted.append(token)
                    chance.append(float(p[token]))
                    continue
                rest = torch.clamp(p - other, min=0.0)
            rest = p if rest is None or float(rest.sum()) <= 0.0 else rest
            sums = torch.cumsum(rest, 0)
            token = int(torch.searchsorted(sums, u[i][d] * float(sums[-1]), right=True))
            accepted.append(len(emitted))
            emitted.append(token)
            chance.append(float(p[token]))
            break
        tokens.append(emitted + [NONE] * (d + 1 - len(emitted)))
        chances.append(chance + [0.0] * (d + 1 - len(chance)))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "tokens": torch.tensor(tokens, dtype=torch.int32),
            "probabilities": torch.tensor(chances, dtype=torch.float64)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"block": _exact_block, "product": _exact_product, "route": _exact_route, "draft": _exact_draft}[case["kind"]](s)
