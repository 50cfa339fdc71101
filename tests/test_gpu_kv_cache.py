"""The paged cache: storing with and without 8-bit codes, loading, and attention of one token over its pages."""
import ctypes
import math

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f8": torch.float8_e4m3fn}


def empty_cache(pages, heads, page, dim, dtype, token_major=False):
    shape = (pages, page, heads, dim) if token_major else (pages, heads, page, dim)
    make = lambda: torch.full(shape, math.nan, device="cuda").to(dtype)  # noqa: E731
    k, v = make(), make()
    ks = vs = None
    if dtype == TYPES["f8"]:
        ks, vs = (torch.full(shape[:3], math.nan, device="cuda") for _ in range(2))
    if token_major:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
        ks, vs = (None if s is None else s.transpose(1, 2) for s in (ks, vs))
    return k, v, ks, vs


def read(cache, scale):
    x = cache.cpu().double()
    return x if scale is None else x * scale.cpu().double()[..., None]


@pytest.mark.parametrize("token_major", [False, True], ids=["heads first", "slots first"])
@pytest.mark.parametrize("cache", ["f8", "same"])
@pytest.mark.parametrize("tokens,heads,dim,page,dtype", [
    (1, 1, 8, 1, "bf16"), (1, 8, 128, 64, "bf16"), (7, 3, 72, 16, "f16"), (130, 2, 64, 32, "bf16"), (33, 5, 256, 8, "f16"),
    (300, 4, 200, 128, "bf16"), (65, 1, 136, 1024, "f16")])
def test_store_and_load(gpu, tokens, heads, dim, page, dtype, cache, token_major):
    g = torch.Generator().manual_seed(tokens)
    dt = TYPES[dtype]
    pages = -(-tokens // page) + 2
    k, v = ((torch.randn((tokens, heads, dim), generator=g) * 5).to(dt) for _ in range(2))
    k[0, 0] = 0.0
    v[-1, -1, 0] = 1000.0
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    if tokens > 4:
        slots[2], slots[3] = -1, pages * page
    print("case", tokens, heads, dim, page, dtype, cache, flush=True)
    kc, vc, ks, vs = empty_cache(pages, heads, page, dim, TYPES["f8"] if cache == "f8" else dt, token_major)
    gpu.kv_store(k.cuda(), v.cuda(), slots.cuda(), kc, vc, ks, vs)
    torch.cuda.synchronize()
    live = (slots >= 0) & (slots < pages * page)
    where = slots[live].long()
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[where] = False
    flat = lambda t: t.cpu().transpose(1, 2).reshape(pages * page, *t.shape[1:2], *t.shape[3:])  # noqa: E731
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        got = flat(c.float())
        assert bool(torch.isnan(got[untouched]).all())
        if cache == "same":
            assert torch.equal(got[where], x[live].float())
            continue
        scale = x[live].float().abs().amax(-1) / 448.0
        assert torch.equal(flat(s)[where], scale)
        assert bool(torch.isnan(flat(s)[untouched]).all())
        codes = torch.where(scale[..., None] > 0, x[live].float() / scale[..., None], torch.zeros(())).to(TYPES["f8"])
        assert torch.equal(got[where], codes.float())
        # and against the value itself: half a step of three stored bits, or of the smallest step 2^-9
        err = (got[where].double() * scale.double()[..., None] - x[live].double()).abs()
        assert bool((err <= torch.maximum(2.0 ** -4 * x[live].double().abs(), 2.0 ** -10 * scale.double()[..., None]) * (1 + 1e-5)).all())
    ko, vo = (torch.full((tokens, heads, dim), 7.0, dtype=dt, device="cuda") for _ in range(2))
    gpu.kv_load(kc, vc, slots.cuda(), ko, vo, ks, vs)
    torch.cuda.synchronize()
    for o, c, s in ((ko, kc, ks), (vo, vc, vs)):
        want = torch.zeros((tokens, heads, dim), dtype=dt)
        want[live] = (flat(c.float())[where] * (1.0 if s is None else flat(s)[where][..., None])).to(dt)
        assert torch.equal(o.cpu(), want)


def test_values_that_are_not_finite(gpu):
    x = torch.ones((4, 1, 16), dtype=torch.bfloat16)
    x[0, 0, 3] = math.nan
    x[1, 0, 5] = math.inf
    x[2] = math.nan
    x[3] *= 1e-38
    kc, vc, ks, vs = empty_cache(1, 1, 4, 16, TYPES["f8"])
    slots = torch.arange(4, dtype=torch.int32).cuda()
    gpu.kv_store(x.cuda(), x.cuda(), slots, kc, vc, ks, vs)
    out, _ = gpu.kv_load(kc, vc, slots, torch.empty_like(x, device="cuda"), torch.empty_like(x, device="cuda"), ks, vs)
    got = out.cpu().float()
    others = torch.arange(16) != 3
    assert math.isnan(got[0, 0, 3]) and bool((got[0, 0, others] == 1.0).all())
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[2]).all())
    assert bool(((got[3] - x[3].float()).abs() <= 2.0 ** -7 * 1e-38).all())


def test_rows_as_slices_of_a_projection(gpu):
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn((50, 4 + 2 + 2, 64), generator=g).to(torch.bfloat16).cuda()
    kc, vc, _, _ = empty_cache(2, 2, 32, 64, torch.bfloat16)
    slots = torch.arange(50, dtype=torch.int32).cuda()
    gpu.kv_store(qkv[:, 4:6], qkv[:, 6:], slots, kc, vc)
    out = torch.zeros_like(qkv)
    gpu.kv_load(kc, vc, slots, out[:, 4:6], out[:, 6:])
    torch.cuda.synchronize()
    assert torch.equal(out[:, 4:], qkv[:, 4:]) and bool((out[:, :4] == 0).all())


# ---- attention over the cache --------------------------------------------------------------------------------

def paged_case(seqs, lengths, heads, kv_heads, dim, page, dtype, cache, each, seed, token_major=False):
    """A cache filled through kv_store, page lists in random order, NaN in every slot that holds no token."""
    from lapis_amd import hip
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + 3
    kc, vc, ks, vs = empty_cache(pages, kv_heads, page, dim, TYPES["f8"] if cache == "f8" else dtype, token_major)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    at, tables, slots = 0, [], []
    for n, h in zip(lengths, held):
        tables.append(order[at:at + h])
        t = torch.arange(n)
        slots.append(order[at:at + h][t // page].long() * page + t % page if n else torch.zeros(0, dtype=torch.int64))
        at += h
    slots = torch.cat(slots).to(torch.int32).cuda()
    k, v = (torch.randn((slots.numel(), kv_heads, dim), generator=g).to(dtype).cuda() for _ in range(2))
    hip.kv_store(k, v, slots, kc, vc, ks, vs)
    q = torch.randn((seqs, heads, dim), generator=g).to(dtype).cuda()
    lists, tokens = [], []
    for n, table in zip(lengths, tables):
        for _ in range(kv_heads if each else 1):
            if each and len(table) > 2:  # some pages and the last one
                keep = torch.rand(len(table), generator=g) < 0.5
                keep[-1] = True
                lists.append(table[keep])
                tokens.append(n - int((~keep).sum()) * page)
            else:
                lists.append(table)
                tokens.append(n)
    pos = torch.tensor([0] + [sum(len(x) for x in lists[:i + 1]) for i in range(len(lists))], dtype=torch.int32).cuda()
    crd = torch.cat(lists).to(torch.int32).cuda()
    return q, kc, vc, pos, crd, torch.tensor(tokens, dtype=torch.int32).cuda(), ks, vs


def paged_reference(q, kc, vc, pos, crd, tokens, ks, vs, scale):
    seqs, heads, dim = q.shape
    kv_heads, page = kc.shape[1], kc.shape[2]
    group = heads // kv_heads
    K, V = read(kc, ks), read(vc, vs)
    out, lse, bound, lse_bound = (torch.zeros((seqs, heads, dim), dtype=torch.float64), torch.full((seqs, heads), -math.inf, dtype=torch.float64),
                                  torch.zeros((seqs, heads, dim), dtype=torch.float64), torch.zeros((seqs, heads), dtype=torch.float64))
    p, c, t = pos.clamp(0, crd.numel()).tolist(), crd.cpu().long(), tokens.tolist()
    u, tiny = ref.HALF_ULP[q.dtype], ref.TINY[q.dtype]
    each = len(t) != seqs
    Q = q.cpu().double()
    for s in range(seqs):
        for h in range(heads):
            kh = h // group
            row = s * kv_heads + kh if each else s
            pages = c[p[row]:p[row + 1]]
            there = ((pages >= 0) & (pages < kc.shape[0])).repeat_interleave(page)[:max(0, t[row])]
            pages = pages.clamp(0, kc.shape[0] - 1)
            kk, vv = (x[pages, kh].reshape(-1, dim)[:max(0, t[row])][there] for x in (K, V))
            if kk.shape[0] == 0:
                continue
            score = scale * (kk @ Q[s, h])
            weight = torch.softmax(score, 0)
            ds = float((dim * 2.0 ** -23 * abs(scale) * (kk.abs() @ Q[s, h].abs())).max())
            out[s, h] = weight @ vv
            lse[s, h] = torch.logsumexp(score, 0)
            # 8-bit codes are multiplied as they are, their scales go into the weights before these are rounded
            bound[s, h] = u * out[s, h].abs() + (weight @ vv.abs()) * (u + 2 * ds + 2.0 ** -18) + tiny * vv.abs().sum(0)
            lse_bound[s, h] = 2 * ds + 2.0 ** -18 + u / 4 + 2.0 ** -22 * lse[s, h].abs()
    return out, lse, bound, lse_bound


def check_paged(gpu, what, case, scale=None):
    q, kc, vc, pos, crd, tokens, ks, vs = case
    print("case", what, flush=True)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    gpu.paged_attention(q, kc, vc, pos, crd, tokens, out, lse=lse, scale=scale, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    want, want_lse, bound, lse_bound = paged_reference(*case[:6], ks, vs, q.shape[2] ** -0.5 if scale is None else scale)
    ref.assert_within(out, want, bound, what + ": out")
    ref.assert_within(lse, want_lse, lse_bound, what + ": lse")
    return out


@pytest.mark.parametrize("cache", ["f8", "same"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", [
    ([1], 1, 1, 64, 64), ([0], 4, 2, 64, 16), ([17, 0, 16, 15, 1], 4, 4, 64, 16), ([300], 8, 1, 128, 32), ([64, 65, 63], 6, 2, 72, 64),
    ([1000, 3, 129], 16, 2, 96, 128), ([257], 7, 1, 80, 8), ([200, 31], 32, 2, 40, 1), ([1500], 5, 5, 8, 16), ([700, 900], 12, 4, 256, 64),
    ([513], 34, 2, 136, 256), ([2000], 3, 1, 200, 1024)])
def test_paged_attention(gpu, lengths, heads, kv_heads, dim, page, dtype, cache):
    case = paged_case(len(lengths), lengths, heads, kv_heads, dim, page, TYPES[dtype], cache, False, dim)
    check_paged(gpu, "%s, %d heads over %d, %d x %d, %s %s" % (lengths, heads, kv_heads, page, dim, dtype, cache), case)


@pytest.mark.parametrize("cache", ["f8", "same"])
@pytest.mark.parametrize("token_major", [False, True])
def test_a_list_for_each_head(gpu, cache, token_major):
    case = paged_case(3, [700, 5, 333], 12, 4, 64, 32, torch.bfloat16, cache, True, 3, token_major)
    check_paged(gpu, "lists of each head", case)


@pytest.mark.parametrize("cache", ["f8", "same"])
def test_a_long_sequence_beside_short_ones(gpu, cache):
    case = paged_case(5, [40000, 1, 70, 0, 9000], 8, 2, 128, 64, torch.bfloat16, cache, False, 3)
    out = check_paged(gpu, "40000 tokens", case)
    for _ in range(3):
        again = torch.empty_like(out)
        gpu.paged_attention(*case[:6], again, k_scale=case[6], v_scale=case[7])
        assert torch.equal(out, again)


def test_tokens_and_lists_that_disagree(gpu):
    q, kc, vc, pos, crd, tokens, ks, vs = paged_case(3, [100, 100, 100], 4, 2, 64, 16, torch.bfloat16, "same", False, 8)
    for slots in (kc, vc):
        slots.copy_(torch.nan_to_num(slots, nan=0.5))
    crd[3], crd[9] = -7, 1 << 29                                        # pages that do not exist are absent
    tokens = torch.tensor([1000, -4, 50], dtype=torch.int32).cuda()     # more than listed, fewer than none, fewer than listed
    check_paged(gpu, "disagreement", (q, kc, vc, pos, crd, tokens, ks, vs))
    pos = torch.tensor([-3, 5, 2, 1 << 30], dtype=torch.int32).cuda()
    check_paged(gpu, "positions", (q, kc, vc, pos, crd, torch.full((3,), 90, dtype=torch.int32).cuda(), ks, vs))


def test_scores_of_hundreds_and_scales(gpu):
    case = list(paged_case(2, [300, 40], 4, 2, 64, 16, torch.float16, "same", False, 8))
    case[0] = case[0] * 12
    check_paged(gpu, "large scores", case, scale=1.0)
    check_paged(gpu, "scale 0", case, scale=0.0)


def test_a_cache_beyond_32_bits(gpu):
    """Pages 2^31 and more elements into the cache."""
    pages, page, dim = 9000, 64, 256
    kc = torch.empty((pages, 16, page, dim), dtype=torch.bfloat16, device="cuda")
    assert kc.numel() > 1 << 31
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn((130, 16, dim), generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    slots = torch.cat([torch.arange(64) + 64 * 8999, torch.arange(64) + 64 * 8500, torch.arange(2) + 64 * 3]).to(torch.int32).cuda()
    vc = torch.empty_like(kc)
    gpu.kv_store(k, v, slots, kc, vc)
    q = torch.randn((1, 16, dim), generator=g).to(torch.bfloat16).cuda()
    pos, crd = torch.tensor([0, 3], dtype=torch.int32).cuda(), torch.tensor([8999, 8500, 3], dtype=torch.int32).cuda()
    out, lse = torch.empty_like(q), torch.empty((1, 16), device="cuda")
    gpu.paged_attention(q, kc, vc, pos, crd, torch.tensor([130], dtype=torch.int32).cuda(), out, lse=lse)
    ko, vo = gpu.kv_load(kc, vc, slots, torch.empty_like(k), torch.empty_like(v))
    torch.cuda.synchronize()
    assert torch.equal(ko, k) and torch.equal(vo, v)
    small = [x.transpose(0, 1)[None].reshape(1, 16, 130, dim) for x in (k, v)]
    padded = [torch.nn.functional.pad(x, (0, 0, 0, 1024 - 130)) for x in small]
    want = paged_reference(q, *padded, torch.tensor([0, 1]), torch.tensor([0]), torch.tensor([130]), None, None, dim ** -0.5)
    ref.assert_within(out, want[0], want[2], "far pages: out")
    ref.assert_within(lse, want[1], want[3], "far pages: lse")


def test_another_stream_and_a_captured_graph(gpu):
    q, kc, vc, pos, crd, tokens, ks, vs = case = paged_case(4, [3000, 10, 0, 900], 8, 2, 128, 64, torch.bfloat16, "f8", False, 5)
    want = check_paged(gpu, "plain", case)
    side = torch.cuda.Stream()
    out = torch.empty_like(q)
    gpu.paged_attention(q, kc, vc, pos, crd, tokens, out, k_scale=ks, v_scale=vs, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.paged_attention(q, kc, vc, pos, crd, tokens, out, k_scale=ks, v_scale=vs)
    for _ in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        eager = torch.empty_like(out)
        gpu.paged_attention(q, kc, vc, pos, crd, tokens, eager, k_scale=ks, v_scale=vs)
        torch.cuda.synchronize()
        assert torch.equal(eager, want)


def test_the_c_entries_refuse(gpu):
    k = torch.zeros((4, 1, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(4, dtype=torch.int32, device="cuda")
    for pages, page, dim in ((1, 24, 64), (1, 2048, 64), (1, 16, 264), (1, 16, 12)):
        kc, vc, _, _ = empty_cache(pages, 1, page, dim, torch.bfloat16)
        x = torch.zeros((4, 1, dim), dtype=torch.bfloat16, device="cuda")
        with pytest.raises(gpu.LapisHipError, match="INVALID_ARGUMENT"):
            gpu.kv_store(x, x, slots, kc, vc)
    flat = torch.empty(4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 1, 64)
    kc, vc, _, _ = empty_cache(1, 1, 16, 64, torch.bfloat16)
    with pytest.raises(gpu.LapisHipError, match="16-byte"):
        gpu.kv_store(flat, k, slots, kc, vc)


@pytest.mark.parametrize("cache", ["f8", "same"])
@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "f16"), (168, "bf16")])
def test_many_rows_move_as_few_do(gpu, cache, dim, dtype):
    """Enough rows for four to a thread, an odd number of them: the same bits as in calls of fewer
    rows, which the tests above hold to the formulas."""
    heads, tokens, page = 8, 70001 if dim == 64 else 35003, 64
    dt = TYPES[dtype]
    pages = -(-tokens // page) + 1
    g = torch.Generator().manual_seed(dim)
    k, v = (torch.randn((tokens, heads, dim), generator=g).to(dt).cuda() for _ in range(2))
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    slots[5::1000] = -1
    slots = slots.cuda()
    print("case", cache, dim, dtype, flush=True)
    stored, loaded = [], []
    for step in (tokens, 4001):
        c = empty_cache(pages, heads, page, dim, TYPES["f8"] if cache == "f8" else dt)
        ko, vo = (torch.full_like(k, 7.0) for _ in range(2))
        for i in range(0, tokens, step):
            gpu.kv_store(k[i:i + step], v[i:i + step], slots[i:i + step], *c)
            gpu.kv_load(*c[:2], slots[i:i + step], ko[i:i + step], vo[i:i + step], *c[2:])
        torch.cuda.synchronize()
        stored.append([x.view(torch.uint8) for x in c if x is not None])
        loaded.append((ko, vo))
    assert all(torch.equal(x, y) for x, y in zip(*stored)) and all(torch.equal(x, y) for x, y in zip(*loaded))
    live = slots >= 0
    assert bool((loaded[0][0][~live] == 0).all()) and bool((loaded[0][1][~live] == 0).all())
    if cache == "same":
        assert torch.equal(loaded[0][0][live], k[live]) and torch.equal(loaded[0][1][live], v[live])


def test_partial_results_of_calls_on_two_streams_are_not_shared(gpu):
    """Both calls cut their lists into units and join them, at the same time on two streams."""
    case = paged_case(3, [40000, 9000, 20000], 8, 2, 128, 64, torch.bfloat16, "f8", False, 3)
    q, kc, vc, pos, crd, tokens, ks, vs = case
    want = check_paged(gpu, "by itself", case)
    other = (q.float() * 0.5).to(q.dtype)
    want_other = check_paged(gpu, "other queries", (other,) + case[1:])
    got, got_other = torch.zeros_like(q), torch.zeros_like(q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(8):
        gpu.paged_attention(q, kc, vc, pos, crd, tokens, got, k_scale=ks, v_scale=vs)
        gpu.paged_attention(other, kc, vc, pos, crd, tokens, got_other, k_scale=ks, v_scale=vs, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(got_other, want_other)


@pytest.mark.parametrize("cache", ["f8", "same"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_values_of_no_weight_beside_many_small_ones(gpu, dtype, cache):
    """In every stretch that a wavefront takes: one token of weight 1, one of next to none whose value row is 60000 in size, and a few
    hundred ordinary ones of 2^-10.5 each, a sixth of the sum.  In an 8-bit cache the large row's scale must not cost theirs."""
    tokens, heads, page, dim = 65536, 8, 64, 64
    g = torch.Generator().manual_seed(3)
    v = torch.randn((tokens, heads, dim), generator=g) + 1.0
    score = torch.full((tokens,), -10.5 * math.log(2))
    at = torch.arange(tokens)
    first = (at // 32) % 32 < 4  # the first tile of each of four wavefronts in each 1024 tokens
    score[first & (at % 32 == 5)] = 2.0 ** -9
    score[first & (at % 32 == 17)] = -40.0
    v[first & (at % 32 == 17)] = 60000.0
    k = torch.zeros((tokens, heads, dim))
    k[..., 0] = score[:, None]
    k, v = (x.to(TYPES[dtype]).cuda() for x in (k, v))
    kc, vc, ks, vs = empty_cache(tokens // page, heads, page, dim, TYPES["f8"] if cache == "f8" else TYPES[dtype])
    gpu.kv_store(k, v, torch.arange(tokens, dtype=torch.int32).cuda(), kc, vc, ks, vs)
    q = torch.zeros((1, heads, dim))
    q[..., 0] = 1.0
    pos, crd = torch.tensor([0, tokens // page], dtype=torch.int32).cuda(), torch.arange(tokens // page, dtype=torch.int32).cuda()
    out = torch.empty((1, heads, dim), dtype=TYPES[dtype], device="cuda")
    gpu.paged_attention(q.to(TYPES[dtype]).cuda(), kc, vc, pos, crd, torch.tensor([tokens], dtype=torch.int32).cuda(), out, scale=1.0,
                        k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    u, tiny = ref.HALF_ULP[TYPES[dtype]], ref.TINY[TYPES[dtype]]
    for h in range(heads):
        kk, vv = (read(x, s)[:, h].reshape(-1, dim) for x, s in ((kc, ks), (vc, vs)))
        s = kk[:, 0]
        p = torch.exp(s - s.max())
        want, spread = p @ vv / p.sum(), p @ vv.abs() / p.sum()
        # as everywhere: weights and results are rounded once to the type; a weight, 1 for the best token, also to a multiple of 2^-24
        bound = u * want.abs() + spread * (u + 2 * dim * 2.0 ** -23 * 40 + 2.0 ** -18) + tiny * vv.abs().sum(0) / p.sum()
        assert float((tiny * vv.abs().sum(0) / p.sum()).max()) < 0.01 and bool((spread < 4).all())
        ref.assert_within(out[0, h], want, bound, "%s %s, head %d" % (dtype, cache, h))


def test_scales_that_differ_by_powers_of_two_and_are_not_numbers(gpu):
    """float16 with an 8-bit cache whose scales are 2^-15 to 2^7 in any order, each row the only one of a query: nothing is rounded, codes and
    scales come out as they are.  Rows of zeros; an infinity and a NaN only where a sequence holds them."""
    dim, page = 64, 16
    g = torch.Generator().manual_seed(4)
    sizes = 2.0 ** torch.tensor([0, 7, -15, 3, -9, 6, -12, 5, -3, -14, 4, 0, 2, -6, 1, -1], dtype=torch.float64)
    every = torch.arange(127, dtype=torch.uint8).view(TYPES["f8"]).double()  # 0 to 448
    v = every[torch.randint(0, 127, (3, 16, 1, dim), generator=g)] * torch.where(torch.rand((3, 16, 1, dim), generator=g) < 0.5, -1.0, 1.0)
    v[..., 0] = 448.0
    v *= sizes[None, :, None, None]
    v[:, 11] = 0.0
    v[1, 4, 0, 3], v[1, 9, 0, 5] = math.inf, math.nan
    held, v = v[:, :, 0], v.to(torch.float16)
    assert torch.equal(v[::2, :, 0].double(), held[::2])
    k = torch.zeros((3, 16, 1, dim), dtype=torch.float16)
    k[:, range(16), 0, range(16)] = 1.0
    kc, vc, ks, vs = empty_cache(3, 1, page, dim, TYPES["f8"])
    gpu.kv_store(k.reshape(48, 1, dim).cuda(), v.reshape(48, 1, dim).cuda(), torch.arange(48, dtype=torch.int32).cuda(), kc, vc, ks, vs)
    q = torch.zeros((3, 16, dim), dtype=torch.float16)
    q[:, range(16), range(16)] = 200.0  # a query for each key: the others' weights are 0
    out = torch.empty((3, 16, dim), dtype=torch.float16, device="cuda")
    gpu.paged_attention(q.cuda(), kc, vc, torch.arange(4, dtype=torch.int32).cuda(), torch.arange(3, dtype=torch.int32).cuda(),
                        torch.full((3,), 16, dtype=torch.int32).cuda(), out, scale=1.0, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    for s in (0, 2):
        assert torch.equal(out[s].cpu().double(), held[s])
    assert bool(torch.isnan(out[1]).any())  # whatever a token holds that is no number, its sequence shows it


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride", ctypes.c_int64 * 3)]


class Cache(ctypes.Structure):
    """lapis_hip_kv_cache"""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + [("stride", ctypes.c_int64 * 3), ("scale_stride", ctypes.c_int64 * 3)] +
                [("pages", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("heads", "page", "dim", "dtype")])


class PagedArgs(ctypes.Structure):
    """lapis_hip_paged_args"""
    _fields_ = ([(n, ctypes.c_int64) for n in ("seqs", "lists", "heads", "nnz")] + [("q", Rows), ("out", Rows), ("dtype", ctypes.c_int)] +
                [(n, ctypes.c_void_p) for n in ("pos", "crd", "tokens", "lse")] + [("scale", ctypes.c_float), ("work", ctypes.c_void_p)])


def test_partial_results_of_more_tokens_times_heads_than_31_bits(gpu):
    """2^31 tokens of 1024 heads: units of 1024 tokens."""
    gpu.init()
    nnz, bytes_ = (1 << 31) - 1, ctypes.c_int64(-1)
    cache, args = Cache(heads=1024, page=1, dim=8), PagedArgs(seqs=2, lists=2, heads=1024, nnz=nnz)
    gpu.check(gpu.load().lapis_hip_paged_attention_work(ctypes.byref(cache), ctypes.byref(args), ctypes.byref(bytes_)))
    assert bytes_.value == (nnz // 1024 + 2) * 1024 * 16 * (64 + 2) * 4


@pytest.mark.parametrize("cache,args,what", [
    (dict(heads=65535, page=16, dim=8), dict(seqs=65535, lists=65535 * 65535, heads=65535, nnz=0), "4294836225 lists"),
    (dict(heads=32768, page=1, dim=8), dict(seqs=65535, lists=65535 * 32768, heads=32768, nnz=2147483647), "2149548031 units of work"),
    (dict(heads=4, page=16, dim=8, pages=1 << 60), dict(seqs=1, lists=1, heads=4, nnz=0), "slots are numbered with 31 bits")])
def test_sizes_that_numbers_do_not_hold_are_refused(gpu, cache, args, what):
    x, i = torch.full((8, 8), 7.0, dtype=torch.bfloat16, device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    c = Cache(k=x.data_ptr(), v=x.data_ptr(), **cache)
    a = PagedArgs(pos=i.data_ptr(), crd=i.data_ptr(), tokens=i.data_ptr(), q=Rows(x.data_ptr()), out=Rows(x.data_ptr()), work=x.data_ptr(), **args)
    gpu.init()
    with pytest.raises(gpu.LapisHipError, match=what):
        gpu.check(gpu.load().lapis_hip_paged_attention(ctypes.byref(c), ctypes.byref(a), None))
    if "pages" in cache:
        rows = Rows(x.data_ptr())
        with pytest.raises(gpu.LapisHipError, match=what):
            gpu.check(gpu.load().lapis_hip_kv_store(ctypes.byref(c), 1, ctypes.byref(rows), ctypes.byref(rows), 0, i.data_ptr(), None))
    torch.cuda.synchronize()
    assert bool((x == 7.0).all())


def test_more_tokens_than_numbers_hold_are_refused(gpu):
    x, i = torch.full((8, 8), 7.0, dtype=torch.bfloat16, device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    c, rows = Cache(k=x.data_ptr(), v=x.data_ptr(), heads=4, page=1, dim=8, pages=1), Rows(x.data_ptr())
    gpu.init()
    for tokens in (1 << 62, 1 << 29, (1 << 63) - 1):  # times four heads: 0, 2^31 and -4 in 64 and 32 bits
        for call in (lambda n: gpu.load().lapis_hip_kv_store(ctypes.byref(c), n, ctypes.byref(rows), ctypes.byref(rows), 0, i.data_ptr(), None),
                     lambda n: gpu.load().lapis_hip_kv_load(ctypes.byref(c), n, i.data_ptr(), ctypes.byref(rows), ctypes.byref(rows), 0, None)):
            with pytest.raises(gpu.LapisHipError, match="tokens of 4 heads"):
                gpu.check(call(tokens))
    torch.cuda.synchronize()
    assert bool((x == 7.0).all())
