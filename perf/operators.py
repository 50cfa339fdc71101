"""The operators of block-sparse attention that this library is measured on, beside their plain forms.

  store, load   new tokens' keys and values into a paged cache, quantised on the way where the cache holds 8 bits, and
                back out of it
  paged         one new token of each sequence against the pages its CSR list names
  pool          8-bit means of blocks of tokens, what blocks are scored by
  select        the best-scoring blocks of keys of each block of queries, as a CSR structure
  attend        attention over the blocks that a CSR structure lists: the output and the logarithms of the row sums
  gradient      its backward pass: gradients of queries, keys and values

A case is a dict of plain values.  ``listed()`` names the fixed ones, ``draw(rng)`` gives another case of the same
ranges, ``prepare(case, seed)`` makes what a program holds before the call, ``run(state)`` is one pass (the plain form, or
with ``own`` the library's entry points), ``exact(case, seed)`` the definition in 64 bits, ``work(case)`` the bytes and
floating-point operations a pass cannot do without.

Structures: row (batch, key-value head, block of ``block_m`` queries), columns blocks of ``block_n`` keys; the heads of
a group (heads / kv_heads of them) share their key-value head's rows.  Query i stands at position i + keys - queries.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f8": torch.float8_e4m3fn}
_F8_MAX = 448.0


def listed():
    return [
        # One decoding step of 48 sequences writes its tokens into an 8-bit cache: the call itself counts.
        {"name": "store_step_f8", "kind": "store", "tokens": 48, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16",
         "cache": "f8", "scattered": True},
        # A prompt of 32k tokens enters the 8-bit cache.
        {"name": "store_prompt_32k_f8", "kind": "store", "tokens": 32768, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16",
         "cache": "f8", "scattered": False},
        # A kept prefix is read back in 16 bits, for a prompt that goes on from it.
        {"name": "load_prefix_20k_f8", "kind": "load", "tokens": 20000, "kv_heads": 8, "dim": 96, "page": 32, "dtype": "f16",
         "cache": "f8", "scattered": False},
        # A single user's next token after 16k: latency, all compute units on one sequence.
        {"name": "paged_one_16k_bf16", "kind": "paged", "seqs": 1, "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "cache": "bf16", "count": 0},
        # A batch in service: 64 ragged sequences of up to 8k tokens in the 8-bit cache.
        {"name": "paged_batch_8k_f8", "kind": "paged", "seqs": 64, "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "cache": "f8", "count": 0},
        # Sparse decoding: each key-value head reads only the 24 pages selected for it; no heads share keys.
        {"name": "paged_selected_f16", "kind": "paged", "seqs": 24, "tokens": 30000, "heads": 12, "kv_heads": 12, "dim": 64,
         "page": 32, "dtype": "f16", "cache": "f16", "count": 24},
        # Means of the key blocks of a 32k prompt.
        {"name": "pool_keys_32k", "kind": "pool", "batch": 1, "tokens": 32768, "heads": 8, "kv_heads": 8, "dim": 128, "block": 64,
         "dtype": "bf16"},
        # Blocks for each single query of a 16k prompt: 131 thousand rows of up to 256 blocks.
        {"name": "select_queries_16k", "kind": "select", "batch": 1, "queries": 16384, "keys": 16384, "kv_heads": 8, "dim": 128,
         "block_m": 1, "block_n": 64, "count": 16, "causal": True},
        # The prompt pass of a long context: 32k tokens, each block of 128 queries against 16 blocks of 128 keys.
        {"name": "attend_32k_bf16", "kind": "attend", "batch": 1, "queries": 32768, "keys": 32768, "heads": 32, "kv_heads": 8,
         "dim": 128, "block_m": 128, "block_n": 128, "count": 16, "causal": True, "dtype": "bf16", "packed": True},
        # Lists of each query's own: 16 heads of one query share the blocks.
        {"name": "attend_queries_4k_f16", "kind": "attend", "batch": 1, "queries": 4096, "keys": 4096, "heads": 32, "kv_heads": 2,
         "dim": 64, "block_m": 1, "block_n": 32, "count": 16, "causal": True, "dtype": "f16", "packed": False},
        # A training step's backward pass.
        {"name": "gradient_8k_bf16", "kind": "gradient", "batch": 1, "queries": 8192, "keys": 8192, "heads": 32, "kv_heads": 8,
         "dim": 128, "block_m": 64, "block_n": 64, "count": 16, "causal": True, "dtype": "bf16", "packed": True},
        # Odd sizes, a head dimension between two tiles, more keys than queries (a prefix in front).
        {"name": "gradient_odd_f16", "kind": "gradient", "batch": 3, "queries": 1001, "keys": 1437, "heads": 6, "kv_heads": 3,
         "dim": 80, "block_m": 40, "block_n": 32, "count": 9, "causal": True, "dtype": "f16", "packed": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_heads(rng, groups):
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    return {"heads": kv_heads * rng.choice(groups), "kv_heads": kv_heads, "dim": rng.choice([32, 64, 72, 80, 96, 128])}


def draw(rng):
    kind = rng.choice(["store", "load", "paged", "paged", "paged", "pool", "select", "select", "attend", "attend", "attend",
                       "gradient", "gradient", "gradient"])
    dtype = rng.choice(["bf16", "f16"])
    if kind in ("store", "load"):
        h = _draw_heads(rng, [1])
        tokens = _log_int(rng, 1, int(32768 * 8 * 128 / (max(h["kv_heads"], 2) * 128)))
        return {"kind": kind, "tokens": min(tokens, 65536), "kv_heads": h["kv_heads"], "dim": h["dim"],
                "page": rng.choice([16, 32, 64, 128]), "dtype": dtype, "cache": rng.choice(["f8", "f8", dtype]),
                "scattered": tokens <= 256}
    if kind == "paged":
        case = dict({"kind": kind, "seqs": _log_int(rng, 1, 64)}, **_draw_heads(rng, [1, 2, 3, 4, 7, 8, 16]))
        case.update(tokens=_log_int(rng, 1, min(65536, int(64 * 8192 * 8 / (case["seqs"] * case["kv_heads"])))),
                    page=rng.choice([16, 32, 64, 128]), dtype=dtype, cache=rng.choice(["f8", dtype, dtype]),
                    count=rng.choice([0, 0, _log_int(rng, 1, 64)]))
        return case
    if kind == "pool":
        h = _draw_heads(rng, [1, 1, 4, 8])
        batch = rng.choice([1, 1, 2, 5])
        return {"kind": kind, "batch": batch, "tokens": _log_int(rng, 1, int(32768 * 8 / (h["heads"] * batch))), "heads": h["heads"],
                "kv_heads": h["kv_heads"], "dim": h["dim"], "block": rng.choice([1, 16, 32, 64, 100, 128]), "dtype": dtype}
    case = {"kind": kind, "batch": rng.choice([1, 1, 2, 3])}
    case.update(_draw_heads(rng, [1, 2, 4, 5, 8, 16]))
    each = rng.random() < 0.3
    case["block_m"] = 1 if each else rng.choice([16, 37, 64, 128])
    case["block_n"] = rng.choice([16, 32, 64, 128])
    case["count"] = _log_int(rng, 1, max(1, 2048 // case["block_n"]))
    top = {"select": 16384 if each else 65536, "attend": 4096 if each else 16384, "gradient": 2048 if each else 8192}[kind]
    most = 32 if kind != "select" else 8
    case["queries"] = _log_int(rng, 1, max(1, min(top, top * most // (case["batch"] * case["heads" if kind != "select" else "kv_heads"]))))
    case["causal"] = rng.random() < 0.8
    same = rng.random() < 0.6
    case["keys"] = case["queries"] if same else _log_int(rng, 1, 2 * top) if not case["causal"] else case["queries"] + rng.randint(0, top)
    if kind == "select":  # long enough for a choice beside the first and the last block
        del case["heads"]
        more = max(0, 20 * case["block_n"] - min(case["queries"], case["keys"]))
        case["queries"], case["keys"] = case["queries"] + more, case["keys"] + more
        case["count"] = max(4, min(case["count"], case["keys"] // case["block_n"] // 4))
        return case
    case.update(dtype=dtype, packed=same and rng.random() < 0.5)
    return case


# ---- sizes --------------------------------------------------------------------------------------------------

def _blocks(n, size):
    return -(-n // size)


def _allowed(case):
    """Blocks of keys that each block of queries may see."""
    rows, columns = _blocks(case["queries"], case["block_m"]), _blocks(case["keys"], case["block_n"])
    if not case["causal"]:
        return np.full(rows, columns, dtype=np.int64)
    last = np.minimum((np.arange(rows, dtype=np.int64) + 1) * case["block_m"], case["queries"]) - 1
    return np.clip((last + case["keys"] - case["queries"]) // case["block_n"] + 1, 0, columns)


def _entries(case):
    """Blocks listed for each block of queries."""
    return np.minimum(_allowed(case), case["count"])


def _pairs(case):
    """Pairs of a query and a key that attention over the structure computes, of one head and batch entry: the last
    allowed block of a row is always listed, so of the listed blocks only that one is cut by the end or the diagonal."""
    queries, keys, m, n = case["queries"], case["keys"], case["block_m"], case["block_n"]
    allowed, entries = _allowed(case), _entries(case)
    total = 0
    for r in range(allowed.size):
        first = r * m
        held = min(m, queries - first)
        if entries[r] == 0:
            continue
        total += held * n * (int(entries[r]) - 1)
        start = (int(allowed[r]) - 1) * n
        seen = np.minimum(n, keys - start)
        if case["causal"]:
            at = first + np.arange(held) + keys - queries - start + 1
            total += int(np.clip(at, 0, seen).sum())
        else:
            total += held * int(seen)
    return total


def _lengths(case):
    """Tokens in the cache of each sequence, from a quarter of ``tokens`` to all of it."""
    n, t = case["seqs"], case["tokens"]
    return [max(1, t - (t - t // 4) * i // max(1, n - 1)) for i in range(n)]


def _listed_tokens(case):
    """Tokens of the pages that a list names, for each sequence."""
    lengths = _lengths(case)
    if not case["count"]:
        return lengths
    page, count = case["page"], case["count"]
    return [t - (_blocks(t, page) - min(count, _blocks(t, page))) * page for t in lengths]


def _size_of(name):
    return {"f8": 1}.get(name, 2)


def work(case):
    kind, d = case["kind"], case["dim"]
    if kind in ("store", "load"):
        values = 2 * case["tokens"] * case["kv_heads"]
        return {"bytes": values * (d * (2 + _size_of(case["cache"])) + (4 if case["cache"] == "f8" else 0)) + 4 * case["tokens"],
                "flops": 2 * values * d}
    if kind == "paged":
        tokens = sum(_listed_tokens(case))
        held = 2 * tokens * case["kv_heads"] * (d * _size_of(case["cache"]) + (4 if case["cache"] == "f8" else 0))
        lists = 4 * sum(_blocks(t, case["page"]) for t in _listed_tokens(case)) * (case["kv_heads"] if case["count"] else 1)
        return {"bytes": held + lists + 4 * case["seqs"] * case["heads"] * d, "flops": 4 * d * case["heads"] * tokens}
    if kind == "pool":
        blocks = case["batch"] * case["kv_heads"] * _blocks(case["tokens"], case["block"])
        values = case["batch"] * case["tokens"] * case["heads"] * d
        return {"bytes": 2 * values + blocks * (d + 4), "flops": values + 3 * blocks * d}
    lists = case["batch"] * case["kv_heads"]
    rows, columns = _blocks(case["queries"], case["block_m"]), _blocks(case["keys"], case["block_n"])
    entries = int(_entries(case).sum())
    if kind == "select":
        return {"bytes": lists * (rows * (d + 4) + columns * (d + 4) + 4 * entries), "flops": 2 * d * lists * int(_allowed(case).sum())}
    structure = 4 * lists * (rows + entries)
    queries = 2 * case["batch"] * case["queries"] * case["heads"] * d
    keys = 2 * case["batch"] * case["keys"] * case["kv_heads"] * d
    sums = 4 * case["batch"] * case["queries"] * case["heads"]
    pairs = _pairs(case) * case["batch"] * case["heads"]
    if kind == "attend":
        return {"bytes": structure + 2 * queries + 2 * keys + sums, "flops": 4 * d * pairs}
    return {"bytes": structure + 4 * queries + 4 * keys + sums, "flops": 10 * d * pairs}


# ---- inputs -------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * spread).to(dtype)


def _keys_like(g, shape, dtype):
    """Keys as projections give them: a few channels are several times as large as the others."""
    channels = torch.ones(shape[-1], device="cuda")
    channels[:: max(1, shape[-1] // 4)] = 4.0
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * channels).to(dtype)


def _lists(case, g):
    """Positions and coordinates: the first block, the last allowed one and random ones between, ascending."""
    lists, count, n = case["batch"] * case["kv_heads"], case["count"], case["block_n"]
    columns = _blocks(case["keys"], n)
    allowed = torch.from_numpy(_allowed(case)).cuda()
    entries = torch.from_numpy(_entries(case)).cuda()
    rows = allowed.numel()
    score = torch.rand((lists, rows, columns), generator=g, device="cuda")
    at = torch.arange(columns, device="cuda")
    score[:, :, 0] = 2.0
    score.masked_fill_(at == allowed[:, None] - 1, 3.0)
    score.masked_fill_(at >= allowed[:, None], -1.0)
    best = score.topk(min(count, columns), dim=2).indices
    best = torch.where(torch.arange(best.shape[2], device="cuda") < entries[:, None], best, columns).sort(dim=2).values
    pos = torch.zeros(lists * rows + 1, dtype=torch.int32, device="cuda")
    pos[1:] = torch.cumsum(entries.repeat(lists), 0)
    return pos, best[best < columns].to(torch.int32)


def _quantised(x):
    scale = x.abs().amax(-1) / _F8_MAX
    codes = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros_like(x))
    return codes.to(torch.float8_e4m3fn), scale


def _slots(case, g, pages):
    tokens, page = case["tokens"], case["page"]
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(tokens, device="cuda")
    if case["scattered"]:  # one token in each of that many pages
        return (order[:tokens] * page + at % page).to(torch.int32)
    return (order[at // page] * page + at % page).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    kind, d = case["kind"], case["dim"]
    dtype = _TYPES[case.get("dtype", "bf16")]
    empty = lambda shape, t=dtype: torch.empty(shape, dtype=t, device="cuda")  # noqa: E731
    if kind in ("store", "load"):
        tokens, heads, page = case["tokens"], case["kv_heads"], case["page"]
        pages = tokens if case["scattered"] else _blocks(tokens, page) + 3
        s["slots"] = _slots(case, g, pages)
        s["k"], s["v"] = _keys_like(g, (tokens, heads, d), dtype), _normal(g, (tokens, heads, d), dtype)
        shape = (pages, heads, page, d)
        s["k_scale"] = s["v_scale"] = None
        if kind == "store":
            for name in ("k", "v"):
                s[name + "_cache"] = torch.zeros(shape, dtype=dtype, device="cuda").to(_TYPES[case["cache"]])
                if case["cache"] == "f8":
                    s[name + "_scale"] = torch.zeros(shape[:3], device="cuda")
        else:
            for name, make in (("k", _keys_like), ("v", _normal)):
                x = make(g, shape, dtype)
                s[name + "_cache"] = x
                if case["cache"] == "f8":
                    s[name + "_cache"], s[name + "_scale"] = _quantised(x.float())
                s[name] = empty((tokens, heads, d))
        return s
    if kind == "paged":
        seqs, page, heads = case["seqs"], case["page"], case["kv_heads"]
        held = [_blocks(t, page) for t in _lengths(case)]
        shape = (sum(held), heads, page, d)
        order = torch.randperm(shape[0], generator=g, device="cuda").to(torch.int32)
        s["k_scale"] = s["v_scale"] = None
        for name, make in (("k", _keys_like), ("v", _normal)):
            x = make(g, shape, dtype)
            s[name + "_cache"] = x
            if case["cache"] == "f8":
                s[name + "_cache"], s[name + "_scale"] = _quantised(x.float())
        s["q"], s["out"] = _normal(g, (seqs, case["heads"], d), dtype), empty((seqs, case["heads"], d))
        tokens = torch.tensor(_listed_tokens(case), dtype=torch.int32, device="cuda")
        if not case["count"]:
            s["crd"], entries = order, torch.tensor(held, device="cuda")
        else:  # the last page and random others before it, for each key-value head its own
            chosen, at = [], 0
            for n in held:
                c = min(case["count"], n)
                score = torch.rand((heads, n), generator=g, device="cuda")
                score[:, -1] = 2.0
                chosen.append(order[at + score.topk(c, dim=1).indices.sort(dim=1).values].reshape(-1))
                at += n
            s["crd"] = torch.cat(chosen)
            entries = torch.tensor([min(case["count"], n) for n in held], device="cuda").repeat_interleave(heads)
            tokens = tokens.repeat_interleave(heads)
        s["pos"] = torch.zeros(entries.numel() + 1, dtype=torch.int32, device="cuda")
        s["pos"][1:] = torch.cumsum(entries, 0)
        s["listed_tokens"], s["most"] = tokens, int(max(_blocks(t, page) for t in _listed_tokens(case)))
        s["softmax_scale"] = d ** -0.5
        return s
    if kind == "pool":
        s["x"] = _keys_like(g, (case["batch"], case["tokens"], case["heads"], d), dtype)
        shape = (case["batch"], case["kv_heads"], _blocks(case["tokens"], case["block"]), d)
        s["codes"], s["scales"] = empty(shape, torch.int8), empty(shape[:3], torch.float32)
        return s
    batch, kv_heads = case["batch"], case["kv_heads"]
    rows, columns = _blocks(case["queries"], case["block_m"]), _blocks(case["keys"], case["block_n"])
    if kind == "select":
        whole = lambda n: (torch.randn((batch, kv_heads, n, d), generator=g, device="cuda") * 36).round().clamp(-127, 127).to(torch.int8)  # noqa: E731
        s["q_codes"], s["k_codes"] = whole(rows), whole(columns)
        s["k_scales"] = torch.rand((batch, kv_heads, columns), generator=g, device="cuda") * 0.02 + 0.005
        s["pos"] = torch.zeros(batch * kv_heads * rows + 1, dtype=torch.int32, device="cuda")
        s["crd"] = torch.full((batch * kv_heads * int(_entries(case).sum()),), -1, dtype=torch.int32, device="cuda")
        s["allowed"] = torch.from_numpy(_allowed(case)).cuda()
        return s
    queries, keys, heads = case["queries"], case["keys"], case["heads"]
    if case["packed"]:  # slices of one projection's output
        x = _normal(g, (batch, queries, heads + 2 * kv_heads, d), dtype)
        s["q"], s["k"], s["v"] = x[:, :, :heads], x[:, :, heads:heads + kv_heads], x[:, :, heads + kv_heads:]
    else:
        s["q"] = _normal(g, (batch, queries, heads, d), dtype)
        s["k"], s["v"] = (_normal(g, (batch, keys, kv_heads, d), dtype) for _ in range(2))
    s["pos"], s["crd"] = _lists(case, g)
    s["most"] = int(_entries(case).max())
    s["softmax_scale"] = d ** -0.5
    if kind == "attend":
        s["out"], s["lse"] = empty((batch, queries, heads, d)), empty((batch, heads, queries), torch.float32)
    else:
        s["out"], s["lse"] = _attend(s)  # what the forward pass left
        s["dout"] = _normal(g, (batch, queries, heads, d), dtype)
        s["dq"] = empty((batch, queries, heads, d))
        s["dk"], s["dv"] = empty((batch, keys, kv_heads, d)), empty((batch, keys, kv_heads, d))
    return s


# ---- plain forms --------------------------------------------------------------------------------------------

def _store(s):
    page, at = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    for name in ("k", "v"):
        x, cache = s[name], s[name + "_cache"]
        if s["cache"] == "f8":
            codes, scale = _quantised(x.float())
            cache.view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
            s[name + "_scale"][page, :, at] = scale
        else:
            cache[page, :, at] = x
    return [t for t in (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]) if t is not None]


def _load(s):
    page, at = s["slots"].long() // s["page"], s["slots"].long() % s["page"]
    for name in ("k", "v"):
        cache = s[name + "_cache"]
        if s["cache"] == "f8":
            x = cache.view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn).float() * s[name + "_scale"][page, :, at][..., None]
        else:
            x = cache[page, :, at]
        s[name].copy_(x)
    return s["k"], s["v"]


def _softmax_parts(scores, mask):
    """exp(scores - maximum), its sums and the maxima over the last axis; rows without an entry have sum 0."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    return p, p.sum(-1, keepdim=True), top


def _paged(s):
    seqs, heads, d = s["q"].shape
    kv_heads, page = s["kv_heads"], s["page"]
    group = heads // kv_heads
    each = s["pos"].numel() - 1 == seqs * kv_heads and s["count"] > 0
    index = s["pos"][:-1, None].long() + torch.arange(s["most"], device="cuda")
    pages = s["crd"][index.clamp(max=s["crd"].numel() - 1)].long().clamp(min=0)  # rows x most
    mask = torch.arange(s["most"] * page, device="cuda") < s["listed_tokens"][:, None]
    if each:
        pages, mask = pages.reshape(seqs, kv_heads, -1), mask.reshape(seqs, kv_heads, -1)
    else:
        pages, mask = pages[:, None].expand(-1, kv_heads, -1), mask[:, None].expand(-1, kv_heads, -1)
    head = torch.arange(kv_heads, device="cuda")[None, :, None]

    def values(name):
        x = s[name + "_cache"]
        if s["cache"] == "f8":
            x = x.view(torch.uint8)[pages, head].view(torch.float8_e4m3fn).float() * s[name + "_scale"][pages, head][..., None]
        else:
            x = x[pages, head].float()
        return x.reshape(seqs, kv_heads, -1, d)

    q = s["q"].float().reshape(seqs, kv_heads, group, d)
    p, total, _ = _softmax_parts(q @ values("k").transpose(2, 3) * s["softmax_scale"], mask[:, :, None])
    out = p @ values("v") / total
    s["out"].copy_(torch.where(total > 0, out, torch.zeros_like(out)).reshape(seqs, heads, d))
    return s["out"]


def _pool(s):
    batch, tokens, heads, d = s["x"].shape
    kv_heads, block = s["kv_heads"], s["block"]
    blocks = _blocks(tokens, block)
    x = torch.nn.functional.pad(s["x"].float(), (0, 0, 0, 0, 0, blocks * block - tokens))
    held = (tokens - torch.arange(blocks, device="cuda") * block).clamp(max=block) * (heads // kv_heads)
    mean = x.reshape(batch, blocks, block, kv_heads, heads // kv_heads, d).sum((2, 4)) / held[:, None, None]
    mean = mean.transpose(1, 2)
    scale = mean.abs().amax(-1) / 127.0
    codes = torch.where(scale[..., None] > 0, mean / scale[..., None], torch.zeros_like(mean)).round()
    s["codes"].copy_(codes)
    s["scales"].copy_(scale)
    return _pooled(s)


def _pooled(s):
    """The values that the 8-bit means stand for."""
    return (s["codes"] * s["scales"][..., None]).to(_TYPES[s["dtype"]])


def _select(s):
    score = (s["q_codes"].float() @ s["k_codes"].float().transpose(2, 3)) * s["k_scales"][:, :, None]
    columns, allowed = score.shape[3], s["allowed"][:, None]
    at = torch.arange(columns, device="cuda")
    score = score.masked_fill(at == allowed - 1, math.inf)
    score[..., 0] = math.inf
    score = score.masked_fill(at >= allowed, -math.inf)
    best = score.sort(dim=3, descending=True, stable=True).indices[..., :s["count"]]
    entries = s["allowed"].clamp(max=s["count"])
    best = torch.where(torch.arange(best.shape[3], device="cuda") < entries[:, None], best, columns).sort(dim=3).values
    s["crd"].copy_(best[best < columns])
    s["pos"][1:] = torch.cumsum(entries.repeat(score.shape[0] * score.shape[1]), 0)
    return s["pos"], s["crd"]


def _gathered(s):
    """Queries, keys and values of every row of the structure, in 32 bits: rows x queries x heads of the group, rows x
    listed keys; the mask; where the keys came from."""
    batch, queries, heads, d = s["q"].shape
    keys, kv_heads, m, n = s["k"].shape[1], s["kv_heads"], s["block_m"], s["block_n"]
    rows, group = _blocks(queries, m), heads // kv_heads
    index = s["pos"][:-1, None].long() + torch.arange(s["most"], device="cuda")
    there = index < s["pos"][1:, None]
    blocks = s["crd"][index.clamp(max=max(0, s["crd"].numel() - 1))].long() if s["crd"].numel() else torch.zeros_like(index)
    key = (blocks[:, :, None] * n + torch.arange(n, device="cuda")).reshape(index.shape[0], -1)
    there = there.repeat_interleave(n, 1) & (key < keys)
    key = key.clamp(max=keys - 1)
    row = torch.arange(batch * kv_heads * rows, device="cuda")
    b, h, r = row // (kv_heads * rows), row // rows % kv_heads, row % rows
    query = r[:, None] * m + torch.arange(m, device="cuda")
    mask = there[:, None, :] & (query < queries)[:, :, None]
    if s["causal"]:
        mask &= key[:, None, :] <= (query + keys - queries)[:, :, None]
    mask = mask[:, :, None].expand(-1, -1, group, -1).reshape(row.numel(), m * group, -1)
    at = (b[:, None], key, h[:, None])
    rows_of = lambda x: torch.nn.functional.pad(x.float(), (0, 0) * (x.dim() - 2) + (0, rows * m - queries)).reshape(  # noqa: E731
        batch, rows, m, kv_heads, group, -1).permute(0, 3, 1, 2, 4, 5).reshape(batch * kv_heads * rows, m * group, -1)
    return rows_of, s["k"][at].float(), s["v"][at].float(), mask, at


def _back(x, s):
    """Rows of the structure back to batch x queries x heads x the rest."""
    batch, queries, heads, _ = s["q"].shape
    kv_heads, m = s["kv_heads"], s["block_m"]
    rows = _blocks(queries, m)
    x = x.reshape(batch, kv_heads, rows, m, heads // kv_heads, -1).permute(0, 2, 3, 1, 4, 5)
    return x.reshape(batch, rows * m, heads, -1)[:, :queries]


def _attend(s):
    rows_of, k, v, mask, _ = _gathered(s)
    p, total, top = _softmax_parts(rows_of(s["q"]) @ k.transpose(1, 2) * s["softmax_scale"], mask)
    out = p @ v / total
    out = _back(torch.where(total > 0, out, torch.zeros_like(out)), s)
    return out.to(s["q"].dtype), _back(top + torch.log(total), s)[..., 0].transpose(1, 2).contiguous()


def _gradient(s):
    rows_of, k, v, mask, at = _gathered(s)
    q, dout = rows_of(s["q"]), rows_of(s["dout"])
    lse = rows_of(s["lse"].transpose(1, 2)[..., None])
    p = torch.exp(torch.where(mask, q @ k.transpose(1, 2) * s["softmax_scale"] - lse, torch.full_like(lse, -math.inf)))
    delta = rows_of(s["dout"].float() * s["out"].float()).sum(-1, keepdim=True)
    ds = p * (dout @ v.transpose(1, 2) - delta) * s["softmax_scale"]
    s["dq"].copy_(_back(ds @ k, s))
    for name, x in (("dk", ds.transpose(1, 2).contiguous() @ q), ("dv", p.transpose(1, 2).contiguous() @ dout)):
        total = torch.zeros(s[name].shape, dtype=torch.float32, device="cuda")
        s[name].copy_(total.index_put_(at, x, accumulate=True))
    return s["dq"], s["dk"], s["dv"]


# ---- one pass -----------------------------------------------------------------------------------------------

def run(state):
    s, kind = state, state["kind"]
    if not own:
        if kind == "attend":
            out, lse = _attend(s)
            s["out"].copy_(out)
            s["lse"].copy_(lse)
            return s["out"], s["lse"]
        return {"store": _store, "load": _load, "paged": _paged, "pool": _pool, "select": _select, "gradient": _gradient}[kind](s)
    from lapis_amd import hip
    if kind == "store":
        hip.kv_store(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        return [t for t in (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]) if t is not None]
    if kind == "load":
        return hip.kv_load(s["k_cache"], s["v_cache"], s["slots"], s["k"], s["v"], s["k_scale"], s["v_scale"])
    if kind == "paged":
        return hip.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["pos"], s["crd"], s["listed_tokens"], s["out"],
                                   scale=s["softmax_scale"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "pool":
        hip.block_pool(s["x"], s["block"], s["codes"], s["scales"])
        return _pooled(s)
    if kind == "select":
        return hip.block_select(s["q_codes"], s["k_codes"], s["k_scales"], s["count"], s["pos"], s["crd"], queries=s["queries"],
                                keys=s["keys"], block_m=s["block_m"], block_n=s["block_n"], causal=s["causal"], sink=1, local=1)
    if kind == "attend":
        return hip.block_attention(s["q"], s["k"], s["v"], s["pos"], s["crd"], s["out"], s["lse"], block_m=s["block_m"],
                                   block_n=s["block_n"], causal=s["causal"], scale=s["softmax_scale"])
    return hip.block_attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["pos"], s["crd"], s["dq"], s["dk"],
                                        s["dv"], block_m=s["block_m"], block_n=s["block_n"], causal=s["causal"],
                                        scale=s["softmax_scale"])


# ---- the definitions in 64 bits -----------------------------------------------------------------------------

def _exact_cache(s, name):
    x = s[name + "_cache"].double()
    return x * s[name + "_scale"].double()[..., None] if s["cache"] == "f8" else x


def _exact_store(s):
    caches, scales = [], []
    for name in ("k", "v"):
        x = s[name].double()
        top = x.abs().amax(-1) / _F8_MAX
        cache = torch.zeros(s[name + "_cache"].shape, dtype=torch.float64, device="cuda").transpose(1, 2).contiguous()
        cache.view(-1, *cache.shape[2:])[s["slots"].long()] = x if s["cache"] != "f8" else torch.nan_to_num(x / top[..., None])
        caches.append(cache.transpose(1, 2))
        held = torch.zeros(cache.shape[:3], dtype=torch.float64, device="cuda")
        held.view(-1, held.shape[2])[s["slots"].long()] = top
        scales.append(held.transpose(1, 2))
    return caches + (scales if s["cache"] == "f8" else [])


def _exact_load(s):
    return [_exact_cache(s, name).transpose(1, 2).reshape(-1, s["kv_heads"], s["dim"])[s["slots"].long()] for name in ("k", "v")]


def _exact_paged(s):
    k, v = _exact_cache(s, "k"), _exact_cache(s, "v")
    seqs, heads, d = s["q"].shape
    kv_heads = s["kv_heads"]
    pos, tokens = s["pos"].tolist(), s["listed_tokens"].tolist()
    out = torch.zeros((seqs, kv_heads, heads // kv_heads, d), dtype=torch.float64, device="cuda")
    q = s["q"].double().reshape(out.shape)
    for i in range(seqs):
        for h in range(kv_heads):
            row = i * kv_heads + h if s["count"] else i
            pages = s["crd"][pos[row]:pos[row + 1]].long()
            kk, vv = (x[pages, h].reshape(-1, d)[:tokens[row]] for x in (k, v))
            out[i, h] = torch.softmax(q[i, h] @ kk.T * s["softmax_scale"], -1) @ vv
    return out.reshape(seqs, heads, d)


def _exact_pool(s):
    batch, tokens, heads, d = s["x"].shape
    blocks = [s["x"][:, at:at + s["block"]].double().mean(1).reshape(batch, s["kv_heads"], -1, d).mean(2)
              for at in range(0, tokens, s["block"])]
    return torch.stack(blocks, 2)


def _dense(s, list_index):
    """Which key each query of one (batch, key-value head) sees, as a dense mask of rows of blocks by keys."""
    m, n, keys = s["block_m"], s["block_n"], s["k"].shape[1]
    rows = _blocks(s["q"].shape[1], m)
    pos = s["pos"].long()[list_index * rows:(list_index + 1) * rows + 1]
    crd = s["crd"].long()[int(pos[0]):int(pos[-1])]
    seen = torch.zeros((rows, _blocks(keys, n)), dtype=torch.bool, device="cuda")
    seen[torch.repeat_interleave(torch.arange(rows, device="cuda"), pos[1:] - pos[:-1]), crd] = True
    return seen


def _exact_rows(s):
    """(batch entry, key-value head, first query, mask queries x keys) of chunks of the whole problem."""
    queries, keys, m, n = s["q"].shape[1], s["k"].shape[1], s["block_m"], s["block_n"]
    group = s["heads"] // s["kv_heads"]
    step = max(1, int(2e8) // (keys * group * m)) * m
    for b in range(s["q"].shape[0]):
        for h in range(s["kv_heads"]):
            seen = _dense(s, b * s["kv_heads"] + h)
            for at in range(0, queries, step):
                i = torch.arange(at, min(queries, at + step), device="cuda")
                mask = seen[i // m][:, torch.arange(keys, device="cuda") // n]
                if s["causal"]:
                    mask &= torch.arange(keys, device="cuda") <= i[:, None] + keys - queries
                yield b, h, slice(at, at + i.numel()), slice(h * group, (h + 1) * group), mask


def _exact_attend(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((s["q"].shape[0], s["heads"], s["q"].shape[1]), -math.inf, dtype=torch.float64, device="cuda")
    for b, h, rows, heads, mask in _exact_rows(s):
        q = s["q"][b, rows, heads].double().transpose(0, 1)
        score = torch.where(mask, q @ s["k"][b, :, h].double().T * s["softmax_scale"], -math.inf)
        lse[b, heads, rows] = torch.logsumexp(score, -1)
        out[b, rows, heads] = (torch.nan_to_num(torch.softmax(score, -1)) @ s["v"][b, :, h].double()).transpose(0, 1)
    return out, lse


def _exact_gradient(s):
    zeros = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    dq, dk, dv = zeros(s["q"]), zeros(s["k"]), zeros(s["v"])
    for b, h, rows, heads, mask in _exact_rows(s):
        q, dout, out = (x[b, rows, heads].double().transpose(0, 1) for x in (s["q"], s["dout"], s["out"]))
        k, v = s["k"][b, :, h].double(), s["v"][b, :, h].double()
        p = torch.where(mask, torch.exp(q @ k.T * s["softmax_scale"] - s["lse"][b, heads, rows, None].double()), 0.0)
        ds = p * (dout @ v.T - (dout * out).sum(-1, keepdim=True)) * s["softmax_scale"]
        dq[b, rows, heads] = (ds @ k).transpose(0, 1)
        dk[b, :, h] += (ds.flatten(0, 1).T @ q.flatten(0, 1))
        dv[b, :, h] += (p.flatten(0, 1).T @ dout.flatten(0, 1))
    return dq, dk, dv


def exact(case, seed):
    if case["kind"] == "select":
        return None  # whole numbers only
    s = prepare(case, seed)
    return {"store": _exact_store, "load": _exact_load, "paged": _exact_paged, "pool": _exact_pool, "attend": _exact_attend,
            "gradient": _exact_gradient}[case["kind"]](s)
