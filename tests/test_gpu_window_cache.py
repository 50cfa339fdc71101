"""The cache in 4 bits, and single tokens over the window and the first tokens of a cache."""
import math

import pytest
import torch

import attention_ref as ref
import f4_ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f8": torch.float8_e4m3fn}


def f4_cache(pages, heads, page, dim, token_major=False):
    shape = (pages, page, heads) if token_major else (pages, heads, page)
    turn = lambda t: t.transpose(1, 2) if token_major else t  # noqa: E731
    return [turn(torch.full((*shape, n), fill, dtype=torch.uint8, device="cuda")) for n, fill in ((dim // 2, 0x77), (dim // 2, 0x77), (dim // 32, 255), (dim // 32, 255))]


@pytest.mark.parametrize("token_major", [False, True], ids=["heads first", "slots first"])
@pytest.mark.parametrize("tokens,heads,dim,page,dtype", [
    (1, 1, 32, 1, "bf16"), (1, 8, 128, 64, "bf16"), (7, 3, 96, 16, "f16"), (130, 2, 64, 32, "bf16"), (33, 5, 256, 8, "f16"), (300, 4, 224, 128, "bf16"),
    (9000, 4, 128, 1024, "f16")])
def test_store_and_load(gpu, tokens, heads, dim, page, dtype, token_major):
    g = torch.Generator().manual_seed(tokens)
    dt = TYPES[dtype]
    pages = -(-tokens // page) + 2
    # rows of many magnitudes, and values on the grid, between its values and on the borders of scales
    k = (torch.randn((tokens, heads, dim), generator=g) * 2.0 ** torch.randint(-9, 9, (tokens, heads, 1), generator=g)).to(dt)
    v = (torch.randint(-24, 25, (tokens, heads, dim), generator=g) * 0.25).to(dt)
    k[0, 0] = 0.0
    v[-1, -1, 0] = 1000.0
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    if tokens > 4:
        slots[2], slots[3] = -1, pages * page
    kc, vc, ks, vs = f4_cache(pages, heads, page, dim, token_major)
    gpu.kv_store(k.cuda(), v.cuda(), slots.cuda(), kc, vc, ks, vs)
    live = (slots >= 0) & (slots < pages * page)
    where = slots[live].long()
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[where] = False
    flat = lambda t: t.cpu().transpose(1, 2).reshape(pages * page, *t.shape[1:2], *t.shape[3:])  # noqa: E731
    ko, vo = (torch.full((tokens, heads, dim), 7.0, dtype=dt, device="cuda") for _ in range(2))
    gpu.kv_load(kc, vc, slots.cuda(), ko, vo, ks, vs)
    for x, c, s, o in ((k, kc, ks, ko), (v, vc, vs, vo)):
        assert bool((flat(c)[rest] == 0x77).all()) and bool((flat(s)[rest] == 255).all())
        scales = f4_ref.scale_bytes(x[live].double(), dt)
        assert torch.equal(flat(s)[where], scales)
        want = f4_ref.nearest(x[live].double(), scales)
        assert torch.equal(f4_ref.values(flat(c)[where], scales), want)
        back = torch.zeros((tokens, heads, dim), dtype=dt)
        back[live] = want.to(dt)
        assert torch.equal(o.cpu(), back)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_at_the_ends_of_the_types(gpu, dtype):
    """Infinities and NaN take their 32 elements with them; the largest and the smallest numbers."""
    dt = TYPES[dtype]
    x = torch.ones((6, 1, 64), dtype=dt)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 5] = math.inf, math.nan, -math.inf
    x[3, 0, 0], x[3, 0, 40] = torch.finfo(dt).max, -torch.finfo(dt).max
    x[4] = torch.finfo(dt).smallest_normal
    x[5], x[5, 0, 1] = 0.0, torch.finfo(dt).smallest_normal
    kc, vc, ks, vs = f4_cache(1, 1, 8, 64)
    slots = torch.arange(6, dtype=torch.int32, device="cuda")
    gpu.kv_store(x.cuda(), x.cuda(), slots, kc, vc, ks, vs)
    k, v = (torch.zeros_like(x).cuda() for _ in range(2))
    gpu.kv_load(kc, vc, slots, k, v, ks, vs)
    assert torch.equal(ks, vs) and torch.equal(kc, vc) and torch.equal(k.nan_to_num(7.0), v.nan_to_num(7.0))
    k = k.cpu().double()
    assert bool(torch.isnan(k[0, 0, :32]).all() and torch.isnan(k[1, 0, 32:]).all() and torch.isnan(k[2, 0, :32]).all())
    assert bool((k[0, 0, 32:] == 1).all() and (k[1, 0, :32] == 1).all() and (k[2, 0, 32:] == 1).all())
    assert k[3, 0, 0] == f4_ref.MOST[dt] and k[3, 0, 40] == -f4_ref.MOST[dt]
    assert torch.equal(ks.cpu()[0, 0, 3:6], f4_ref.scale_bytes(x[3:, 0].double(), dt))
    assert torch.equal(k[3:, 0], f4_ref.nearest(x[3:, 0].double(), ks.cpu()[0, 0, 3:6]).to(dt).double())


def rows_of_cache(kind, dt, pages, heads, page, dim, g, token_major=False):
    """A cache of random rows, as its tensors and as the values in 64 bits that they stand for (pages x heads x page x dim)."""
    shape = (pages, page, heads, dim) if token_major else (pages, heads, page, dim)
    turn = lambda t: t.transpose(1, 2) if token_major else t  # noqa: E731
    tensors, values, scales = [], [], []
    for _ in range(2):
        x = (torch.randn(shape, generator=g) * 2.0 ** torch.randint(-2, 2, (*shape[:3], 1), generator=g)).to(dt)
        if kind == "f4":
            codes, s = f4_ref.pack(x, dt)
            tensors.append(turn(codes.cuda()))
            scales.append(turn(s.cuda()))
            values.append(turn(f4_ref.values(codes, s)))
        elif kind == "f8":
            s = x.float().abs().amax(-1) / 448.0
            codes = (x.float() / s[..., None]).to(TYPES["f8"])
            tensors.append(turn(codes.cuda()))
            scales.append(turn(s.cuda()))
            values.append(turn(codes.double() * s.double()[..., None]))
        else:
            tensors.append(turn(x.cuda()))
            values.append(turn(x.double()))
    return tensors, scales or [None, None], values


def check_row(out, lse, q, k, v, scale, what):
    """One query's heads against 64 bits; q: heads x dim, k, v: tokens x key-value heads x dim."""
    w = torch.ones((1, k.shape[1], 1, k.shape[0]), dtype=torch.float64)
    want, want_lse, bound, lse_bound = ref.forward(q[None, None], k[None], v[None], w, scale)
    # weights times scales of values are rounded once more, and sums of units are joined in 32 bits
    ref.assert_within(out, want[0, 0], 2 * bound[0, 0], what + " out")
    if lse is not None:
        ref.assert_within(lse, want_lse[0, :, 0], 2 * lse_bound[0, :, 0], what + " lse")


@pytest.mark.parametrize("each", [False, True], ids=["a list", "a list each head"])
@pytest.mark.parametrize("seqs,heads,kv_heads,dim,page,longest,dtype", [
    (1, 1, 1, 32, 1, 3, "bf16"), (3, 8, 2, 64, 16, 100, "f16"), (2, 20, 1, 128, 64, 700, "bf16"), (1, 32, 8, 128, 32, 5000, "f16"), (4, 6, 3, 96, 128, 300, "bf16"),
    (2, 4, 2, 256, 16, 500, "bf16"), (1, 4, 4, 160, 64, 130, "f16"), (2, 40, 2, 64, 1024, 3000, "bf16")])
def test_lists_of_pages_in_4_bits(gpu, seqs, heads, kv_heads, dim, page, longest, dtype, each):
    g = torch.Generator().manual_seed(seqs + dim)
    dt = TYPES[dtype]
    lists = seqs * kv_heads if each else seqs
    counts = [longest] + [int(x) for x in torch.randint(0, longest + 1, (lists - 1,), generator=g)]
    if lists > 2:
        counts[1] = 0
    held = [-(-t // page) for t in counts]
    pages = max(held) + 2
    (kc, vc), (ks, vs), (kv, vv) = rows_of_cache("f4", dt, pages, kv_heads, page, dim, g)
    chosen = [torch.randperm(pages, generator=g)[:n] for n in held]
    crd = torch.cat(chosen).to(torch.int32)
    pos = torch.zeros(lists + 1, dtype=torch.int32)
    pos[1:] = torch.cumsum(torch.tensor(held), 0)
    q = torch.randn((seqs, heads, dim), generator=g).to(dt)
    out, lse = torch.full_like(q, 9.0).cuda(), torch.full((seqs, heads), 9.0, device="cuda")
    gpu.paged_attention(q.cuda(), kc, vc, pos.cuda(), crd.cuda(), torch.tensor(counts, dtype=torch.int32).cuda(), out, lse=lse, k_scale=ks, v_scale=vs)
    group = heads // kv_heads
    for r in range(lists):
        s, kh = (r // kv_heads, slice(r % kv_heads, r % kv_heads + 1)) if each else (r, slice(None))
        h = slice(kh.start * group, kh.stop * group) if each else slice(None)
        k, v = (x[chosen[r]][:, kh].transpose(1, 2).reshape(-1, x[:, kh].shape[1], dim)[:counts[r]] for x in (kv, vv))
        check_row(out[s, h], lse[s, h], q[s, h], k, v, dim ** -0.5, "list %d" % r)


def window_case(kind, dt, seqs, heads, kv_heads, dim, page, lengths, window, sink, g, token_major=False):
    """Tables whose pages without a token that counts point nowhere, and the tokens that count in 64 bits."""
    width = max(1, max(-(-t // page) for t in lengths)) + 1
    seen = [[t for t in range(n) if t >= n - window or t < sink] for n in lengths]
    used = [sorted({t // page for t in s}) for s in seen]
    pages = sum(len(u) for u in used) + 1
    tensors, scales, values = rows_of_cache(kind, dt, pages, kv_heads, page, dim, g, token_major)
    order, at = torch.randperm(pages, generator=g), 0
    table = torch.full((seqs, width), -7, dtype=torch.int32)
    for s, u in enumerate(used):
        table[s, u] = order[at:at + len(u)].to(torch.int32)
        at += len(u)
    rows = []
    for s, tokens in enumerate(seen):
        t = torch.tensor(tokens, dtype=torch.long)
        rows.append([x[table[s, t // page].long(), :, t % page] for x in values])
    q = torch.randn((seqs, heads, dim), generator=g).to(dt)
    return q, tensors, scales, table, rows


@pytest.mark.parametrize("kind", ["same", "f8", "f4"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,lengths,window,sink,dtype,token_major", [
    (1, 1, 32, 16, [1], 1, 0, "bf16", False), (8, 2, 64, 16, [0, 5, 100, 33], 30, 3, "f16", False), (32, 8, 128, 64, [9000], 4096, 16, "bf16", False),
    (20, 1, 128, 32, [700, 701, 64], 128, 64, "f16", True), (6, 3, 96, 128, [300, 1, 1000], 5000, 7, "bf16", False), (4, 4, 256, 8, [77, 500], 33, 500, "bf16", False),
    (6, 2, 160, 1, [40, 90], 17, 9, "f16", False), (4, 2, 64, 64, [2000, 64, 63, 65], 64, 64, "bf16", True)])
def test_window_of_a_cache(gpu, heads, kv_heads, dim, page, lengths, window, sink, dtype, token_major, kind):
    g = torch.Generator().manual_seed(dim + len(lengths))
    dt, seqs = TYPES[dtype], len(lengths)
    q, (kc, vc), (ks, vs), table, rows = window_case(kind, dt, seqs, heads, kv_heads, dim, page, lengths, window, sink, g, token_major)
    out, lse = torch.full_like(q, 9.0).cuda(), torch.full((seqs, heads), 9.0, device="cuda")
    got = gpu.paged_window_attention(q.cuda(), kc, vc, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), out, window, sink, lse=lse, k_scale=ks, v_scale=vs)
    assert got is out
    for s in range(seqs):
        check_row(out[s], lse[s], q[s], *rows[s], dim ** -0.5, "sequence %d" % s)
    again = torch.full_like(out, 3.0)
    gpu.paged_window_attention(q.cuda(), kc, vc, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), again, window, sink, k_scale=ks, v_scale=vs)
    assert torch.equal(out, again)


@pytest.mark.parametrize("kind", ["same", "f8", "f4"])
def test_slots_without_a_token_that_counts_hold_anything(gpu, kind):
    """Slots past the length, between the first tokens and the window, and pages that an entry out of range would name."""
    g = torch.Generator().manual_seed(21)
    page, n, window, sink = 16, 100, 20, 5
    q, (kc, vc), (ks, vs), table, rows = window_case(kind, torch.bfloat16, 1, 4, 2, 64, page, [n], window, sink, g)
    length = torch.tensor([n], dtype=torch.int32).cuda()
    out = torch.empty_like(q).cuda()
    gpu.paged_window_attention(q.cuda(), kc, vc, table.cuda(), length, out, window, sink, k_scale=ks, v_scale=vs)
    counted = torch.zeros((kc.shape[0], page), dtype=torch.bool)
    for t in range(n):
        if t >= n - window or t < sink:
            counted[table[0, t // page].long(), t % page] = True
    spoil = ~counted[:, None].expand(-1, 2, -1).cuda()
    for c, s in ((kc, ks), (vc, vs)):
        if kind == "same":
            c[spoil] = math.nan
        elif kind == "f8":
            s[spoil] = math.inf
        else:
            s[spoil] = 255
    again = torch.empty_like(out)
    table[0, table[0] < 0] = 2 ** 31 - 1
    gpu.paged_window_attention(q.cuda(), kc, vc, table.cuda(), length, again, window, sink, k_scale=ks, v_scale=vs)
    assert torch.equal(out, again)


def test_lengths_and_tables_out_of_range(gpu):
    """Negative lengths see nothing; tokens beyond the table, and those of entries out of range, do not exist."""
    g = torch.Generator().manual_seed(22)
    (kc, vc), _, (kv, vv) = rows_of_cache("same", torch.bfloat16, 4, 2, 16, 64, g)
    q = torch.randn((4, 2, 64), generator=g).bfloat16()
    table = torch.tensor([[0, 1], [2, 3], [-1, 1], [4, 2 ** 30]], dtype=torch.int32)
    lengths = torch.tensor([-3, 2 ** 31 - 1, 32, 32], dtype=torch.int32)
    out, lse = torch.full_like(q, 9.0).cuda(), torch.full((4, 2), 9.0, device="cuda")
    gpu.paged_window_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda(), out, 2 ** 40, 2 ** 40, lse=lse)
    rows = lambda x, pages: x[torch.tensor(pages, dtype=torch.long)].transpose(1, 2).reshape(-1, 2, 64)  # noqa: E731
    for s, pages in enumerate(([], [2, 3], [1], [])):
        check_row(out[s], lse[s], q[s], rows(kv, pages), rows(vv, pages), 0.125, "sequence %d" % s)
    empty = torch.zeros((4, 0), dtype=torch.int32, device="cuda")
    gpu.paged_window_attention(q.cuda(), kc, vc, empty, lengths.cuda(), out, 5, lse=lse)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    none = kc[:0]
    gpu.paged_window_attention(q.cuda(), none, none, table.cuda(), lengths.cuda(), out.fill_(1.0), 5, lse=lse.fill_(1.0))
    assert not bool(out.any()) and bool((lse == -math.inf).all())


def test_a_large_4_bit_cache(gpu):
    """Codes beyond 4 GB and 2^32 elements, found through a table and through a list."""
    pages, heads, page, dim = 150000, 8, 64, 128
    g = torch.Generator().manual_seed(23)
    (kc, vc), (ks, vs), (kv, vv) = rows_of_cache("f4", torch.bfloat16, 3, heads, page, dim, g)
    big = [torch.zeros((pages, *x.shape[1:]), dtype=torch.uint8, device="cuda") for x in (kc, vc, ks, vs)]  # 4.9 GB, twice
    at = torch.tensor([5, pages - 2, pages - 1])
    for b, x in zip(big, (kc, vc, ks, vs)):
        b[at.cuda()] = x
    q = torch.randn((1, 16, dim), generator=g).bfloat16()
    out = torch.empty_like(q).cuda()
    k, v = (x.transpose(1, 2).reshape(-1, heads, dim)[:170] for x in (kv, vv))
    gpu.paged_window_attention(q.cuda(), big[0], big[1], at.to(torch.int32)[None].cuda(), torch.tensor([170], dtype=torch.int32).cuda(), out, 1000,
                               k_scale=big[2], v_scale=big[3])
    check_row(out[0], None, q[0], k, v, dim ** -0.5, "table")
    gpu.paged_attention(q.cuda(), big[0], big[1], torch.tensor([0, 3], dtype=torch.int32).cuda(), at.to(torch.int32).cuda(),
                        torch.tensor([170], dtype=torch.int32).cuda(), out.fill_(2.0), k_scale=big[2], v_scale=big[3])
    check_row(out[0], None, q[0], k, v, dim ** -0.5, "list")


@pytest.mark.parametrize("kind", ["same", "f4"])
def test_streams_and_graphs(gpu, kind):
    """Two captured steps replayed in turn, with eager work between, and steps on two streams at once."""
    g = torch.Generator().manual_seed(24)
    q, (kc, vc), (ks, vs), table, rows = window_case(kind, torch.bfloat16, 3, 8, 2, 64, 16, [3000, 20, 600], 2000, 4, g)
    table, length = table.cuda(), torch.tensor([3000, 20, 600], dtype=torch.int32).cuda()
    qs = [q.cuda(), q.cuda() * 0.5]
    step = lambda i, out, **more: gpu.paged_window_attention(qs[i], kc, vc, table, length, out, 2000, 4, k_scale=ks, v_scale=vs, **more)  # noqa: E731
    want = [step(i, torch.empty_like(qs[i])) for i in range(2)]
    outs, graphs = [torch.empty_like(x) for x in qs], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(i, outs[i])
        graphs.append(graph)
    eager = torch.empty_like(qs[0])
    for turn in range(3):
        for x in outs:
            x.fill_(3.0)
        for graph in graphs:
            graph.replay()
        step(0, eager)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(a, b) for a, b in zip(outs, want)), turn
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(0, outs[0].fill_(1.0))
    step(1, outs[1], stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
