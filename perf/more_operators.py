"""Operators of attention with positions, a window and a cache in 4 bits, beside their plain forms.

  rotate        rows turned by their positions on one or several axes, and back (the gradient)
  append        new tokens' queries and keys turned, and keys and values put into a paged cache, in one call
  paged         one new token of each sequence against the pages its CSR list names, of a cache in 4 bits
  window        attention of each query to the last keys up to itself and to the first ones of all
  gradient      its backward pass
  step          one new token of each sequence against the window and the first tokens of a paged cache

A case is a dict of plain values.  ``listed()`` names the fixed ones, ``draw(rng)`` gives another case of the same
ranges, ``prepare(case, seed)`` makes what a program holds before the call, ``run(state)`` is one pass (the plain form, or
with ``own`` the library's entry points), ``exact(case, seed)`` the definition in 64 bits, ``work(case)`` the bytes and
floating-point operations a pass cannot do without.

Positions: pair i of a row of token t is turned by the sum over axes a of positions[a, t] * frequencies[a, i]; a pair is elements
i and i + pairs, or neighbours 2i and 2i + 1.  Windows: the query at position p sees key j <= p where j > p - window or
j < sink; query i stands at i + keys - queries.  A cache in 4 bits ("f4"): codes of 1 sign, 2 exponent and 1 mantissa bits (0, 0.5, 1,
1.5, 2, 3, 4, 6), two to a byte, the even element low, and for each 32 elements a power of two 2^(byte - 127), the smallest (from 2^-100
on) that leaves no element above 6.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f8": torch.float8_e4m3fn, "f4": torch.uint8}
_F8_MAX = 448.0


def listed():
    return [
        # Queries of a training step on video: axes of time, height and width, a third of the pairs each (16, 24, 24).
        {"name": "rotate_video_16k", "kind": "rotate", "batch": 2, "tokens": 8192, "heads": 32, "dim": 128, "pairs": 64, "axes": 3,
         "neighbours": False, "inverse": False, "dtype": "bf16", "start": 0},
        # The gradient of text positions: odd sizes, neighbours turned, part of each row left as it is.
        {"name": "rotate_back_odd_f16", "kind": "rotate", "batch": 3, "tokens": 1001, "heads": 6, "dim": 80, "pairs": 32, "axes": 1,
         "neighbours": True, "inverse": True, "dtype": "f16", "start": 70000},
        # One decoding step of 48 sequences into an 8-bit cache: the call itself counts.
        {"name": "append_step_f8", "kind": "append", "tokens": 48, "heads": 32, "kv_heads": 8, "dim": 128, "pairs": 64, "axes": 1,
         "neighbours": False, "page": 64, "dtype": "bf16", "cache": "f8", "scattered": True, "start": 20000},
        # A prompt of 32k tokens enters a 4-bit cache, and is read back for its own attention.
        {"name": "append_prompt_32k_f4", "kind": "append", "tokens": 32768, "heads": 32, "kv_heads": 8, "dim": 128, "pairs": 64, "axes": 1,
         "neighbours": False, "page": 64, "dtype": "bf16", "cache": "f4", "scattered": False, "start": 0},
        # A single user's next token after 16k in 4 bits: latency.
        {"name": "paged_one_16k_f4", "kind": "paged", "seqs": 1, "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "cache": "f4", "count": 0},
        # A batch in service: 64 ragged sequences of up to 8k tokens in 4 bits.
        {"name": "paged_batch_8k_f4", "kind": "paged", "seqs": 64, "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "cache": "f4", "count": 0},
        # The prompt pass of a long context: 32k tokens, each sees 2048 and the first 16.
        {"name": "window_32k_bf16", "kind": "window", "batch": 1, "queries": 32768, "keys": 32768, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 2048, "sink": 16, "dtype": "bf16", "packed": True},
        # Part of a prompt behind a kept prefix: odd sizes, a dimension between two tiles.
        {"name": "window_odd_f16", "kind": "window", "batch": 2, "queries": 1001, "keys": 2437, "heads": 12, "kv_heads": 4, "dim": 80,
         "window": 300, "sink": 37, "dtype": "f16", "packed": False},
        # A training step's backward pass.
        {"name": "gradient_8k_bf16", "kind": "gradient", "batch": 1, "queries": 8192, "keys": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 1024, "sink": 16, "dtype": "bf16", "packed": True},
        # Small and odd, more keys than queries, every head its own keys.
        {"name": "gradient_odd_f16", "kind": "gradient", "batch": 3, "queries": 701, "keys": 937, "heads": 6, "kv_heads": 6, "dim": 72,
         "window": 200, "sink": 5, "dtype": "f16", "packed": False},
        # Four users' next tokens far into their texts, pages behind the window given back.
        {"name": "step_four_bf16", "kind": "step", "seqs": 4, "tokens": 100000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 4096, "sink": 16, "dtype": "bf16", "cache": "bf16"},
        # A batch in service over a 4-bit cache, windows of 4k.
        {"name": "step_batch_f4", "kind": "step", "seqs": 128, "tokens": 32768, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 4096, "sink": 64, "dtype": "bf16", "cache": "f4"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "append", "paged", "window", "window", "gradient", "gradient", "step", "step"])
    dtype = rng.choice(["bf16", "f16"])
    cache = rng.choice(["f4", "f4", "f8", dtype]) if kind in ("append", "step") else "f4"
    dim = rng.choice([32, 64, 96, 128]) if cache == "f4" and kind in ("append", "step", "paged") else rng.choice([32, 64, 72, 80, 96, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    if kind in ("rotate", "append"):
        case = {"kind": kind, "heads": heads, "dim": dim, "pairs": rng.choice([dim // 2, dim // 2, dim // 4]), "axes": rng.choice([1, 1, 2, 3]),
                "neighbours": rng.random() < 0.4, "dtype": dtype, "start": rng.choice([0, rng.randint(0, 1000000)])}
        most = int(16384 * 32 * 128 / (max(heads, 2) * max(dim, 64)))
        if kind == "rotate":
            case.update(batch=rng.choice([1, 1, 2, 3]), inverse=rng.random() < 0.5)
            case["tokens"] = _log_int(rng, 1, min(65536, most // case["batch"]))
        else:
            case.update(tokens=_log_int(rng, 1, min(32768, most)), kv_heads=kv_heads, page=rng.choice([16, 32, 64, 128]), cache=cache)
            case["scattered"] = case["tokens"] <= 256
        return case
    if kind in ("paged", "step"):
        case = {"kind": kind, "seqs": _log_int(rng, 1, 64), "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
                "dtype": dtype, "cache": cache}
        if kind == "paged":
            case.update(tokens=_log_int(rng, 1, min(65536, 64 * 8192 * 8 // (case["seqs"] * kv_heads))), count=rng.choice([0, 0, _log_int(rng, 1, 64)]))
        else:
            case.update(tokens=_log_int(rng, 1, 131072), window=_log_int(rng, 1, 4096), sink=rng.choice([0, 1, 4, 64, rng.randint(0, 300)]))
        return case
    case = {"kind": kind, "batch": rng.choice([1, 1, 2, 3]), "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    top = 16384 if kind == "window" else 8192
    case["queries"] = _log_int(rng, 1, max(1, min(top, top * 32 // (case["batch"] * heads))))
    same = rng.random() < 0.5
    case["keys"] = case["queries"] if same else case["queries"] + rng.randint(0, top)
    case.update(window=_log_int(rng, 1, 2048 if kind == "window" else 1024), sink=rng.choice([0, 1, 4, 64, rng.randint(0, 300)]),
                packed=same and rng.random() < 0.5)
    return case


# ---- sizes --------------------------------------------------------------------------------------------------

def _blocks(n, size):
    return -(-n // size)


def _lengths(case):
    """Tokens of each sequence with the new one, from a quarter of ``tokens`` to all of it."""
    n, t = case["seqs"], case["tokens"]
    return [max(1, t - (t - t // 4) * i // max(1, n - 1)) for i in range(n)]


def _listed_tokens(case):
    """Tokens of the pages that a list names, for each sequence."""
    lengths = _lengths(case)
    if not case["count"]:
        return lengths
    page, count = case["page"], case["count"]
    return [t - (_blocks(t, page) - min(count, _blocks(t, page))) * page for t in lengths]


def _seen(case, p):
    """Keys that the query at each position of ``p`` sees."""
    before = np.maximum(0, p - case["window"] + 1)
    return np.where(p < 0, 0, np.maximum(0, p + 1 - before) + np.minimum(case["sink"], before))


def _row_bytes(case):
    """Bytes of a row of the cache with its scales."""
    d = case["dim"]
    return {"f8": d + 4, "f4": d // 2 + d // 32}.get(case["cache"], 2 * d)


def work(case):
    kind, d = case["kind"], case["dim"]
    if kind == "rotate":
        rows = case["batch"] * case["tokens"] * case["heads"]
        return {"bytes": 4 * rows * d + 4 * case["axes"] * case["batch"] * case["tokens"], "flops": 6 * rows * case["pairs"]}
    if kind == "append":
        tokens = case["tokens"]
        values = 2 * tokens * case["kv_heads"]
        moved = values * (2 * d + _row_bytes(case) + (2 * d if case["cache"] == "f4" else 0)) + 4 * tokens * case["heads"] * d
        return {"bytes": moved + 4 * tokens * (1 + case["axes"]), "flops": 6 * tokens * (case["heads"] + case["kv_heads"]) * case["pairs"] + 2 * values * d}
    if kind in ("paged", "step"):
        tokens = sum(_listed_tokens(case)) if kind == "paged" else int(_seen(case, np.array(_lengths(case)) - 1).sum())
        held = 2 * tokens * case["kv_heads"] * _row_bytes(case)
        lists = 4 * sum(_blocks(t, case["page"]) for t in _listed_tokens(case)) * (case["kv_heads"] if case["count"] else 1) if kind == "paged" else 4 * tokens // case["page"]
        return {"bytes": held + lists + 4 * case["seqs"] * case["heads"] * d, "flops": 4 * d * case["heads"] * tokens}
    queries = 2 * case["batch"] * case["queries"] * case["heads"] * d
    keys = 2 * case["batch"] * case["keys"] * case["kv_heads"] * d
    sums = 4 * case["batch"] * case["queries"] * case["heads"]
    pairs = int(_seen(case, np.arange(case["queries"]) + case["keys"] - case["queries"]).sum()) * case["batch"] * case["heads"]
    if kind == "window":
        return {"bytes": 2 * queries + 2 * keys + sums, "flops": 4 * d * pairs}
    return {"bytes": 4 * queries + 4 * keys + sums, "flops": 10 * d * pairs}


# ---- inputs -------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * spread).to(dtype)


def _keys_like(g, shape, dtype):
    """Keys as projections give them: a few channels are several times as large as the others."""
    channels = torch.ones(shape[-1], device="cuda")
    channels[:: max(1, shape[-1] // 4)] = 4.0
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * channels).to(dtype)


def _frequencies(case):
    """Radians a position of each pair, zero on the axes that a pair does not belong to: the last axes get as many pairs each."""
    axes, pairs = case["axes"], case["pairs"]
    i = torch.arange(pairs, device="cuda", dtype=torch.float64)
    f = 10000.0 ** (-i / pairs)
    each = 3 * pairs // (4 * (axes - 1)) if axes > 1 else 0
    first = pairs - each * (axes - 1)
    axis = torch.where(i < first, torch.zeros_like(i), torch.div(i - first, max(each, 1), rounding_mode="floor") + 1)
    return torch.where(axis == torch.arange(axes, device="cuda")[:, None], f, torch.zeros_like(f))


def _positions(case, g, batch, tokens):
    """One axis: where the tokens stand in their texts.  Several: frames of a grid."""
    t = torch.arange(tokens, device="cuda")
    start = case["start"] + torch.randint(0, 1000, (batch, 1), generator=g, device="cuda")
    if case["axes"] == 1:
        return (start + t)[None].to(torch.int32)
    width = 24
    of = [start + t // (width * 16), (t // width % 16)[None].expand(batch, -1), (t % width)[None].expand(batch, -1)]
    return torch.stack(of[:case["axes"]]).to(torch.int32)


def _quantised(x):
    scale = x.abs().amax(-1) / _F8_MAX
    codes = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x))
    return codes.to(torch.float8_e4m3fn), scale


def _power_of_two(e):
    return (e.to(torch.int32) + 127 << 23).view(torch.float32)


def _to_f4(x):
    """Bytes of two codes each and bytes of the scales, of rows in 32 bits."""
    groups = x.reshape(*x.shape[:-1], -1, 32)
    mantissa, exponent = torch.frexp(groups.abs().amax(-1))
    exponent = torch.where(mantissa > 0, torch.where(mantissa <= 0.75, exponent - 3, exponent - 2), -100).clamp(min=-100)
    y = groups * _power_of_two(-exponent[..., None])
    a = y.abs()
    code = torch.where(a < 2, (a * 2).round(), torch.where(a < 4, a.round() + 2, (a / 2).round() + 4))
    code = (code + 8 * (torch.signbit(y) & (code > 0))).to(torch.uint8).reshape(x.shape)
    return code[..., ::2] | code[..., 1::2] << 4, (exponent + 127).to(torch.uint8)


def _of_f4(codes, scales):
    """The values that they stand for, in 32 bits."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    grid = torch.cat([grid, -grid])
    x = grid[torch.stack([codes & 15, codes >> 4], -1).long()].reshape(*codes.shape[:-1], -1, 32)
    return (x * _power_of_two(scales.to(torch.int32)[..., None] - 127)).reshape(*codes.shape[:-1], -1)


def _cache(case, g, shape, empty=False):
    """k_cache, v_cache and their scales of random rows, or zeros."""
    s = {"k_scale": None, "v_scale": None}
    dtype = _TYPES[case["dtype"]]
    for name, make in (("k", _keys_like), ("v", _normal)):
        x = torch.zeros(shape, dtype=dtype, device="cuda") if empty else make(g, shape, dtype)
        if case["cache"] == "f8":
            s[name + "_cache"], s[name + "_scale"] = _quantised(x.float())
        elif case["cache"] == "f4":
            s[name + "_cache"], s[name + "_scale"] = _to_f4(x.float())
        else:
            s[name + "_cache"] = x
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    kind, d = case["kind"], case["dim"]
    dtype = _TYPES[case["dtype"]]
    empty = lambda shape, t=dtype: torch.empty(shape, dtype=t, device="cuda")  # noqa: E731
    if kind == "rotate":
        s["x"] = _normal(g, (case["batch"], case["tokens"], case["heads"], d), dtype)
        s["positions"], s["frequencies"] = _positions(case, g, case["batch"], case["tokens"]), _frequencies(case)
        s["out"] = torch.empty_like(s["x"])
        return s
    if kind == "append":
        tokens, kv_heads, page = case["tokens"], case["kv_heads"], case["page"]
        pages = tokens if case["scattered"] else _blocks(tokens, page) + 3
        order, at = torch.randperm(pages, generator=g, device="cuda"), torch.arange(tokens, device="cuda")
        # one token in each of that many pages, or one text
        s["slots"] = ((order[:tokens] if case["scattered"] else order[at // page]) * page + at % page).to(torch.int32)
        x = _keys_like(g, (tokens, case["heads"] + 2 * kv_heads, d), dtype)  # slices of one projection's output
        s["q"], s["k"], s["v"] = x[:, :case["heads"]], x[:, case["heads"]:case["heads"] + kv_heads], x[:, case["heads"] + kv_heads:]
        s["positions"], s["frequencies"] = _positions(case, g, 1, tokens)[:, 0].contiguous(), _frequencies(case)
        s["q_out"] = empty((tokens, case["heads"], d))
        if case["cache"] == "f4":
            s["k_back"], s["v_back"] = (empty((tokens, kv_heads, d)) for _ in range(2))
        s.update(_cache(case, g, (pages, kv_heads, page, d), empty=True))
        return s
    if kind in ("paged", "step"):
        seqs, page, kv_heads = case["seqs"], case["page"], case["kv_heads"]
        s["q"], s["out"] = _normal(g, (seqs, case["heads"], d), dtype), empty((seqs, case["heads"], d))
        s["softmax_scale"] = d ** -0.5
        lengths = _lengths(case)
        held = [_blocks(t, page) for t in lengths]
        if kind == "step":  # pages behind the window and past the first tokens were given back
            table = torch.full((seqs, max(held)), -1, dtype=torch.int64)
            keep = [[j for j in range(n) if j * page < case["sink"] or (j + 1) * page > t - case["window"]] for n, t in zip(held, lengths)]
            pages = sum(len(k) for k in keep)
            order, at = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)), 0
            for i, k in enumerate(keep):
                table[i, k] = order[at:at + len(k)]
                at += len(k)
            s["table"] = table.to(torch.int32).cuda()
            s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
            s.update(_cache(case, g, (pages, kv_heads, page, d)))
            return s
        order = torch.randperm(sum(held), generator=g, device="cuda").to(torch.int32)
        s.update(_cache(case, g, (sum(held), kv_heads, page, d)))
        tokens = torch.tensor(_listed_tokens(case), dtype=torch.int32, device="cuda")
        if not case["count"]:
            s["crd"], entries = order, torch.tensor(held, device="cuda")
        else:  # the last page and random others before it, for each key-value head its own
            chosen, at = [], 0
            for n in held:
                score = torch.rand((kv_heads, n), generator=g, device="cuda")
                score[:, -1] = 2.0
                chosen.append(order[at + score.topk(min(case["count"], n), dim=1).indices.sort(dim=1).values].reshape(-1))
                at += n
            s["crd"] = torch.cat(chosen)
            entries = torch.tensor([min(case["count"], n) for n in held], device="cuda").repeat_interleave(kv_heads)
            tokens = tokens.repeat_interleave(kv_heads)
        s["pos"] = torch.zeros(entries.numel() + 1, dtype=torch.int32, device="cuda")
        s["pos"][1:] = torch.cumsum(entries, 0)
        s["listed_tokens"], s["most"] = tokens, int(max(_blocks(t, page) for t in _listed_tokens(case)))
        return s
    batch, queries, keys, heads, kv_heads = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads"))
    if case["packed"]:  # slices of one projection's output
        x = _normal(g, (batch, queries, heads + 2 * kv_heads, d), dtype)
        s["q"], s["k"], s["v"] = x[:, :, :heads], x[:, :, heads:heads + kv_heads], x[:, :, heads + kv_heads:]
    else:
        s["q"] = _normal(g, (batch, queries, heads, d), dtype)
        s["k"], s["v"] = (_normal(g, (batch, keys, kv_heads, d), dtype) for _ in range(2))
    s["softmax_scale"] = d ** -0.5
    s["out"], s["lse"] = empty((batch, queries, heads, d)), empty((batch, heads, queries), torch.float32)
    if kind == "gradient":  # what the forward pass left
        out, lse = _window(s)
        s["out"].copy_(out)
        s["lse"].copy_(lse)
        s["dout"] = _normal(g, (batch, queries, heads, d), dtype)
        s["dq"] = empty((batch, queries, heads, d))
        s["dk"], s["dv"] = empty((batch, keys, kv_heads, d)), empty((batch, keys, kv_heads, d))
    return s


# ---- plain forms --------------------------------------------------------------------------------------------

def _turned(x, angle, neighbours, back=False):
    """Rows (... heads x dim) turned by the angles of their tokens (... x pairs), in 32 bits."""
    x, pairs = x.float(), angle.shape[-1]
    cos, sin = torch.cos(angle).float()[..., None, :], torch.sin(angle).float()[..., None, :]
    if back:
        sin = -sin
    y = x.clone()
    lo, hi = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if neighbours else (slice(0, pairs), slice(pairs, 2 * pairs))
    y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
    y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    return y


def _angles(s):
    at = s["positions"].double()[..., None]
    return (at * s["frequencies"].reshape(s["axes"], *(1,) * (at.dim() - 2), -1)).sum(0)


def _rotate(s):
    s["out"].copy_(_turned(s["x"], _angles(s), s["neighbours"], s["inverse"]))
    return s["out"]


def _append(s):
    angle = _angles(s)
    s["q_out"].copy_(_turned(s["q"], angle, s["neighbours"]))
    page, at = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    for name, x in (("k", _turned(s["k"], angle, s["neighbours"])), ("v", s["v"].float())):
        cache = s[name + "_cache"]
        if s["cache"] == "f8":
            codes, s[name + "_scale"][page, :, at] = _quantised(x)
            cache.view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
        elif s["cache"] == "f4":
            cache[page, :, at], s[name + "_scale"][page, :, at] = _to_f4(x)
            s[name + "_back"].copy_(_of_f4(cache[page, :, at], s[name + "_scale"][page, :, at]))
        else:
            cache[page, :, at] = x.to(cache.dtype)
    return _appended(s)


def _appended(s):
    if s["cache"] == "f4":
        return [s["q_out"], s["k_back"], s["v_back"]]
    return [t for t in (s["q_out"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]) if t is not None]


def _softmax_parts(scores, mask):
    """exp(scores - maximum), its sums and the maxima over the last axis; rows without an entry have sum 0."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    return p, p.sum(-1, keepdim=True), top


def _values(s, name, page, head, at=slice(None)):
    """Rows of the cache in 32 bits."""
    x, scale = s[name + "_cache"], s[name + "_scale"]
    if s["cache"] == "f8":
        return x.view(torch.uint8)[page, head, at].view(torch.float8_e4m3fn).float() * scale[page, head, at][..., None]
    return _of_f4(x[page, head, at], scale[page, head, at]) if s["cache"] == "f4" else x[page, head, at].float()


def _tokens_attended(s, k, v, mask):
    """One query of each sequence over its tokens: k, v sequences x key-value heads x tokens x dim."""
    seqs, heads, d = s["q"].shape
    q = s["q"].float().reshape(seqs, s["kv_heads"], -1, d)
    p, total, _ = _softmax_parts(q @ k.transpose(2, 3) * s["softmax_scale"], mask[:, :, None])
    out = p @ v / total
    s["out"].copy_(torch.where(total > 0, out, torch.zeros_like(out)).reshape(seqs, heads, d))
    return s["out"]


def _paged(s):
    seqs, kv_heads, page, d = s["seqs"], s["kv_heads"], s["page"], s["dim"]
    index = s["pos"][:-1, None].long() + torch.arange(s["most"], device="cuda")
    pages = s["crd"][index.clamp(max=s["crd"].numel() - 1)].long()  # rows x most
    mask = torch.arange(s["most"] * page, device="cuda") < s["listed_tokens"][:, None]
    if s["count"]:
        pages, mask = pages.reshape(seqs, kv_heads, -1), mask.reshape(seqs, kv_heads, -1)
    else:
        pages, mask = pages[:, None].expand(-1, kv_heads, -1), mask[:, None].expand(-1, kv_heads, -1)
    head = torch.arange(kv_heads, device="cuda")[None, :, None]
    return _tokens_attended(s, *(_values(s, name, pages, head).reshape(seqs, kv_heads, -1, d) for name in ("k", "v")), mask)


def _step(s):
    sink, window, page = s["sink"], s["window"], s["page"]
    j = torch.arange(sink + window, device="cuda")
    first = (s["lengths"].long() - window).clamp(min=0)[:, None]  # of the window
    at = torch.where(j < sink, j, first + j - sink)
    mask = torch.where(j < sink, j < first, j - sink < s["lengths"][:, None] - first)
    at = torch.where(mask, at, s["lengths"].long()[:, None] - 1)
    pages = s["table"].long().gather(1, at // page)[:, None]
    head = torch.arange(s["kv_heads"], device="cuda")[None, :, None]
    return _tokens_attended(s, *(_values(s, name, pages, head, at[:, None] % page) for name in ("k", "v")), mask[:, None].expand(-1, s["kv_heads"], -1))


def _gathered(s):
    """Queries in blocks, the keys and values that each block may see and the mask, in 32 bits: (batch entry, key-value
    head, block) x queries times heads of the group; where the keys came from."""
    batch, queries, heads, d = s["q"].shape
    keys, kv_heads, sink, window = s["keys"], s["kv_heads"], s["sink"], s["window"]
    m = min(256, queries)
    rows, group, shift = _blocks(queries, m), heads // kv_heads, keys - queries
    row = torch.arange(batch * kv_heads * rows, device="cuda")
    b, h, r = row // (kv_heads * rows), row // rows % kv_heads, row % rows
    j = torch.arange(sink + window + m - 1, device="cuda")
    first = (torch.arange(rows, device="cuda") * m + shift - window + 1).clamp(min=0)[:, None]  # of the window
    key = torch.where(j < sink, j, first + j - sink)
    there = torch.where(j < sink, j < first, key < keys) & (key < keys)
    at = (torch.arange(rows, device="cuda")[:, None] * m + torch.arange(m, device="cuda"))[..., None] + shift
    key, there = key[:, None], there[:, None]
    mask = there & (key <= at) & ((key > at - window) | (key < sink)) & (at < keys)
    mask = mask[r][:, :, None].expand(-1, -1, group, -1).reshape(row.numel(), m * group, -1)
    place = (b[:, None], key[r, 0].clamp(max=keys - 1), h[:, None])
    rows_of = lambda x: torch.nn.functional.pad(x.float(), (0, 0) * (x.dim() - 2) + (0, rows * m - queries)).reshape(  # noqa: E731
        batch, rows, m, kv_heads, group, -1).permute(0, 3, 1, 2, 4, 5).reshape(batch * kv_heads * rows, m * group, -1)
    back = lambda x: x.reshape(batch, kv_heads, rows, m, group, -1).permute(0, 2, 3, 1, 4, 5).reshape(batch, rows * m, heads, -1)[:, :queries]  # noqa: E731
    return rows_of, back, s["k"][place].float(), s["v"][place].float(), mask, place


def _window(s):
    rows_of, back, k, v, mask, _ = _gathered(s)
    p, total, top = _softmax_parts(rows_of(s["q"]) @ k.transpose(1, 2) * s["softmax_scale"], mask)
    out = p @ v / total
    out = back(torch.where(total > 0, out, torch.zeros_like(out)))
    return out.to(s["q"].dtype), back(top + torch.log(total))[..., 0].transpose(1, 2).contiguous()


def _gradient(s):
    rows_of, back, k, v, mask, (b, key, h) = _gathered(s)
    q, dout = rows_of(s["q"]), rows_of(s["dout"])
    lse = rows_of(s["lse"].transpose(1, 2)[..., None])
    p = torch.exp((q @ k.transpose(1, 2) * s["softmax_scale"] - lse).masked_fill(~mask, -math.inf))
    delta = rows_of(s["dout"].float() * s["out"].float()).sum(-1, keepdim=True)
    ds = p * (dout @ v.transpose(1, 2) - delta) * s["softmax_scale"]
    s["dq"].copy_(back(ds @ k))
    place = ((b * s["keys"] + key) * s["kv_heads"] + h).reshape(-1)
    for name, x in (("dk", ds.transpose(1, 2).contiguous() @ q), ("dv", p.transpose(1, 2).contiguous() @ dout)):
        total = torch.zeros((s[name].numel() // s["dim"], s["dim"]), dtype=torch.float32, device="cuda")
        s[name].copy_(total.index_add_(0, place, x.reshape(-1, s["dim"])).reshape(s[name].shape))
    return s["dq"], s["dk"], s["dv"]


# ---- one pass -----------------------------------------------------------------------------------------------

def run(state):
    s, kind = state, state["kind"]
    if not own:
        if kind == "window":
            out, lse = _window(s)
            s["out"].copy_(out)
            s["lse"].copy_(lse)
            return s["out"], s["lse"]
        return {"rotate": _rotate, "append": _append, "paged": _paged, "step": _step, "gradient": _gradient}[kind](s)
    from lapis_amd import hip
    if kind == "rotate":
        return hip.rotate(s["x"], s["positions"], s["frequencies"], s["out"], neighbours=s["neighbours"], inverse=s["inverse"])
    if kind == "append":
        hip.kv_append(s["k"], s["v"], s["positions"], s["frequencies"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                      q=s["q"], q_out=s["q_out"], neighbours=s["neighbours"])
        if s["cache"] == "f4":
            hip.kv_load(s["k_cache"], s["v_cache"], s["slots"], s["k_back"], s["v_back"], s["k_scale"], s["v_scale"])
        return _appended(s)
    if kind == "paged":
        return hip.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["pos"], s["crd"], s["listed_tokens"], s["out"],
                                   scale=s["softmax_scale"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "step":
        return hip.paged_window_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["out"], s["window"], s["sink"],
                                          scale=s["softmax_scale"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "window":
        return hip.window_attention(s["q"], s["k"], s["v"], s["out"], s["window"], s["sink"], lse=s["lse"], scale=s["softmax_scale"])
    return hip.window_attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["dq"], s["dk"], s["dv"], s["window"],
                                         s["sink"], scale=s["softmax_scale"])


# ---- the definitions in 64 bits -----------------------------------------------------------------------------

def _exact_turned(x, s, sign=1.0):
    """Pairs as complex numbers, turned."""
    d, pairs = s["dim"], s["pairs"]
    angle = sum(s["positions"][a].double()[..., None] * s["frequencies"][a] for a in range(s["axes"]))
    x = x.double()
    some, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    shape = (pairs, 2) if s["neighbours"] else (2, pairs)
    some = some.reshape(*x.shape[:-1], *shape)
    if not s["neighbours"]:
        some = some.transpose(-1, -2)
    z = torch.view_as_complex(some.contiguous()) * torch.polar(torch.ones_like(angle), sign * angle)[..., None, :]
    z = torch.view_as_real(z)
    if not s["neighbours"]:
        z = z.transpose(-1, -2)
    return torch.cat([z.reshape(*x.shape[:-1], 2 * pairs), rest], -1).reshape(*x.shape[:-1], d)


def _exact_f4(x):
    """The nearest value of the grid to each element, ties to the even code."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    scale = 2.0 ** torch.ceil(torch.log2(y.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -90) / 6)).clamp(min=-100)
    y = y / scale
    a, step = y.abs(), torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
    below = torch.floor(a / step)
    code = below + ((a / step - below > 0.5) | ((a / step - below == 0.5) & (below % 2 == 1)))
    return (torch.sign(y) * code * step * scale).reshape(x.shape)


def _exact_append(s):
    q, k = _exact_turned(s["q"], s), _exact_turned(s["k"], s)
    if s["cache"] == "f4":
        return [q, _exact_f4(k), _exact_f4(s["v"].double())]
    caches, scales = [], []
    for name, x in (("k", k), ("v", s["v"].double())):
        top = x.abs().amax(-1) / _F8_MAX
        pages, heads, page, d = s[name + "_cache"].shape
        cache = torch.zeros((pages, page, heads, d), dtype=torch.float64, device="cuda")
        cache.view(-1, heads, d)[s["slots"].long()] = x if s["cache"] != "f8" else torch.nan_to_num(x / top[..., None])
        held = torch.zeros((pages, page, heads), dtype=torch.float64, device="cuda")
        held.view(-1, heads)[s["slots"].long()] = top
        caches.append(cache.transpose(1, 2))
        scales.append(held.transpose(1, 2))
    return [q] + caches + (scales if s["cache"] == "f8" else [])


def _exact_rows(s, name, page, h):
    """Pages of one head in 64 bits, page after page."""
    x = s[name + "_cache"][page, h]
    if s["cache"] == "f8":
        return (x.double() * s[name + "_scale"][page, h].double()[..., None]).reshape(-1, s["dim"])
    if s["cache"] == "f4":
        code = torch.stack([x & 15, x >> 4], -1).reshape(*x.shape[:-1], s["dim"]).long()
        e, m = code >> 1 & 3, (code & 1).double()
        value = torch.where(e == 0, m / 2, (1 + m / 2) * 2.0 ** (e - 1).double()) * torch.where(code >= 8, -1.0, 1.0)
        return (value * (2.0 ** (s[name + "_scale"][page, h].double() - 127)).repeat_interleave(32, -1)).reshape(-1, s["dim"])
    return x.double().reshape(-1, s["dim"])


def _exact_tokens(s):
    seqs, heads, d = s["q"].shape
    kv_heads, page = s["kv_heads"], s["page"]
    out = torch.zeros((seqs, kv_heads, heads // kv_heads, d), dtype=torch.float64, device="cuda")
    q = s["q"].double().reshape(out.shape)
    if s["kind"] == "paged":
        pos, tokens = s["pos"].tolist(), s["listed_tokens"].tolist()
    else:
        lengths = s["lengths"].tolist()
    for i in range(seqs):
        if s["kind"] == "step":
            n = _blocks(lengths[i], page)
            table = s["table"][i, :n].long()
            t = torch.arange(n * page, device="cuda")
            seen = (t < lengths[i]) & ((t >= lengths[i] - s["window"]) | (t < s["sink"]))
            used = seen.reshape(n, page).any(1)
            pages, seen = table[used], seen.reshape(n, page)[used].reshape(-1)
        for h in range(kv_heads):
            if s["kind"] == "paged":
                row = i * kv_heads + h if s["count"] else i
                pages = s["crd"][pos[row]:pos[row + 1]].long()
                seen = torch.arange(pages.numel() * page, device="cuda") < tokens[row]
            k, v = (_exact_rows(s, name, pages, h)[seen] for name in ("k", "v"))
            out[i, h] = torch.softmax(q[i, h] @ k.T * s["softmax_scale"], -1) @ v
    return out.reshape(seqs, heads, d)


def _exact_parts(s):
    """(batch entry, key-value head, queries, heads, keys, mask) of chunks of queries; ``keys`` up to the last one seen."""
    queries, keys, group = s["queries"], s["keys"], s["heads"] // s["kv_heads"]
    step = max(1, min(2048, int(2e8) // (keys * group)))
    for b in range(s["batch"]):
        for h in range(s["kv_heads"]):
            for i0 in range(0, queries, step):
                p = torch.arange(i0, min(queries, i0 + step), device="cuda")[:, None] + keys - queries
                first, last = max(0, int(p[0]) - s["window"] + 1), int(p[-1])
                j = torch.arange(0 if s["sink"] else first, last + 1, device="cuda")
                j = j[(j < s["sink"]) | (j >= first)]
                mask = (j <= p) & ((j < s["sink"]) | (p - j < s["window"]))
                yield b, h, slice(i0, i0 + p.shape[0]), slice(h * group, (h + 1) * group), j, mask


def _exact_window(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    for b, h, rows, heads, j, mask in _exact_parts(s):
        q = s["q"][b, rows, heads].double().transpose(0, 1)
        score = torch.where(mask, q @ s["k"][b, j, h].double().T * s["softmax_scale"], -math.inf)
        lse[b, heads, rows] = torch.logsumexp(score, -1)
        out[b, rows, heads] = (torch.nan_to_num(torch.softmax(score, -1)) @ s["v"][b, j, h].double()).transpose(0, 1)
    return out, lse


def _exact_gradient(s):
    zeros = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    dq, dk, dv = zeros(s["q"]), zeros(s["k"]), zeros(s["v"])
    for b, h, rows, heads, j, mask in _exact_parts(s):
        q, dout, out = (x[b, rows, heads].double().transpose(0, 1) for x in (s["q"], s["dout"], s["out"]))
        k, v = s["k"][b, j, h].double(), s["v"][b, j, h].double()
        p = torch.where(mask, torch.exp(q @ k.T * s["softmax_scale"] - s["lse"][b, heads, rows, None].double()), 0.0)
        ds = p * (dout @ v.T - (dout * out).sum(-1, keepdim=True)) * s["softmax_scale"]
        dq[b, rows, heads] = (ds @ k).transpose(0, 1)
        dk[b, j, h] += ds.flatten(0, 1).T @ q.flatten(0, 1)
        dv[b, j, h] += p.flatten(0, 1).T @ dout.flatten(0, 1)
    return dq, dk, dv


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotate":
        return _exact_turned(s["x"], s, -1.0 if s["inverse"] else 1.0)
    return {"append": _exact_append, "paged": _exact_tokens, "step": _exact_tokens, "window": _exact_window, "gradient": _exact_gradient}[case["kind"]](s)
