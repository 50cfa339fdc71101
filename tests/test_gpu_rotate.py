"""Rows turned by their positions, and on their way into the cache."""
import math

import pytest
import torch

import attention_ref as ref
import f4_ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f8": torch.float8_e4m3fn}


def frequencies(axes, pairs, g):
    """Every pair on an axis of its own choice, the last on all of them."""
    f = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    axis = torch.randint(0, axes, (pairs,), generator=g)
    out = torch.where(axis == torch.arange(axes)[:, None], f, 0.0)
    if pairs:
        out[:, -1] = f[-1]
    return out


def turned(x, positions, freq, neighbours, inverse=False):
    """(rows turned in 64 bits, what 32-bit products and cosines of 32 bits may be off by)."""
    x = x.cpu().double()
    pairs = freq.shape[1]
    angle = (positions.cpu().double()[..., None] * freq.cpu().reshape(freq.shape[0], *(1,) * (positions.dim() - 1), pairs)).sum(0)
    c, s = torch.cos(angle)[..., None, :], torch.sin(angle)[..., None, :] * (-1 if inverse else 1)
    i = torch.arange(pairs)
    lo, hi = (2 * i, 2 * i + 1) if neighbours else (i, i + pairs)
    y, off = x.clone(), torch.zeros_like(x)
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    off[..., lo] = off[..., hi] = x[..., lo].abs() + x[..., hi].abs()
    return y, off * 2.0 ** -22  # a rounding each of cosine, product and sum: 3 * 2^-24


SIZES = [  # batch, tokens, heads, dim, pairs, axes, neighbours, dtype
    (1, 1, 1, 8, 4, 1, False, "bf16"), (1, 1, 40, 128, 64, 1, False, "bf16"), (2, 33, 6, 128, 64, 3, False, "bf16"),
    (3, 17, 5, 80, 32, 1, True, "f16"), (1, 50, 3, 72, 36, 2, False, "f16"), (2, 9, 7, 64, 11, 1, False, "bf16"), (1, 65, 2, 256, 128, 2, True, "bf16"),
    (1, 300, 1, 256, 128, 1, False, "f16"), (2, 700, 1, 128, 64, 1, False, "bf16"), (1, 3000, 8, 128, 40, 3, False, "f16"), (1, 5000, 1, 64, 32, 1, True, "bf16"),
    (5, 7, 3, 96, 0, 1, False, "bf16"), (1, 20, 4, 40, 5, 8, True, "f16"), (1, 4100, 3, 200, 52, 2, False, "bf16")]


@pytest.mark.parametrize("inverse", [False, True], ids=["forward", "inverse"])
@pytest.mark.parametrize("batch,tokens,heads,dim,pairs,axes,neighbours,dtype", SIZES)
def test_rotate(gpu, batch, tokens, heads, dim, pairs, axes, neighbours, dtype, inverse):
    g = torch.Generator().manual_seed(dim + tokens)
    dt = TYPES[dtype]
    x = torch.randn((batch, tokens, heads, dim), generator=g).to(dt)
    positions = torch.randint(-5, 1000000, (axes, batch, tokens), generator=g, dtype=torch.int32)
    freq = frequencies(axes, pairs, g)
    out = torch.full((batch, tokens, heads, dim), 7.0, dtype=dt).cuda()
    got = gpu.rotate(x.cuda(), positions.cuda(), freq.cuda(), out, neighbours=neighbours, inverse=inverse)
    assert got is out
    want, off = turned(x, positions, freq, neighbours, inverse)
    ref.assert_within(out, want, want.abs() * ref.HALF_ULP[dt] + off, "turned")
    assert torch.equal(out.cpu()[..., 2 * pairs:], x[..., 2 * pairs:])
    here = x.cuda()  # and in place
    gpu.rotate(here, positions.cuda(), freq.cuda(), here, neighbours=neighbours, inverse=inverse)
    assert torch.equal(here, out)


def test_rotate_strides_and_broadcasts(gpu):
    """Slices of a packed projection, tokens first or heads first, one row of positions for all batch entries."""
    g = torch.Generator().manual_seed(1)
    packed = torch.randn((2, 21, 12, 64), generator=g).bfloat16().cuda()
    freq = frequencies(2, 32, g)
    positions = torch.randint(0, 50, (2, 1, 21), generator=g, dtype=torch.int32)
    q = packed[:, :, 3:8]
    out = torch.zeros((2, 5, 21, 64), dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    gpu.rotate(q, positions.cuda().expand(2, 2, 21), freq.cuda(), out)
    want, off = turned(q, positions.expand(2, 2, 21), freq, False)
    ref.assert_within(out, want, want.abs() * 2.0 ** -8 + off, "strides")
    one = packed[:1, :1, :1].expand(2, 21, 5, 64)  # one row for all
    gpu.rotate(one, positions.cuda().expand(2, 2, 21), freq.cuda(), out)
    want, off = turned(one, positions.expand(2, 2, 21), freq, False)
    ref.assert_within(out, want, want.abs() * 2.0 ** -8 + off, "a broadcast row")
    before = packed.clone()
    gpu.rotate(q, positions.cuda().expand(2, 2, 21), freq.cuda(), q)  # in place, neighbours in the packed tensor stay
    assert torch.equal(packed[:, :, :3], before[:, :, :3]) and torch.equal(packed[:, :, 8:], before[:, :, 8:])


def test_turning_and_turning_back_are_adjoint(gpu):
    """<turn x, y> = <x, turn back y>, which is what makes the inverse its gradient; and it is the inverse."""
    g = torch.Generator().manual_seed(2)
    x, y = (torch.randn((2, 40, 3, 64), generator=g).bfloat16().cuda() for _ in range(2))
    positions = torch.randint(0, 100000, (1, 2, 40), generator=g, dtype=torch.int32).cuda()
    freq = frequencies(1, 32, g).cuda()
    a, b, c = (torch.empty_like(x) for _ in range(3))
    gpu.rotate(x, positions, freq, a)
    gpu.rotate(y, positions, freq, b, inverse=True)
    gpu.rotate(a, positions, freq, c, inverse=True)
    dot = lambda u, v: (u.double() * v.double()).sum().item()  # noqa: E731
    bound = 2 * 2.0 ** -8 * (x.double().abs() * 1.5 * y.double().abs().amax()).sum().item()
    assert abs(dot(a, y) - dot(x, b)) <= bound
    assert bool(((c.double() - x.double()).abs() <= 2.0 ** -8 * (x.double().abs() + 2.9 * x.double().abs().amax())).all())


def caches(kind, dt, pages, heads, page, dim, token_major=False):
    shape = (pages, page, heads) if token_major else (pages, heads, page)
    turn = lambda t: t.transpose(1, 2) if token_major else t  # noqa: E731
    if kind == "f4":
        k, v = (turn(torch.full((*shape, dim // 2), 0x77, dtype=torch.uint8, device="cuda")) for _ in range(2))
        return k, v, *(turn(torch.full((*shape, dim // 32), 255, dtype=torch.uint8, device="cuda")) for _ in range(2))
    make = lambda: turn(torch.full((*shape, dim), math.nan, device="cuda").to(TYPES["f8"] if kind == "f8" else dt))  # noqa: E731
    if kind != "f8":
        return make(), make(), None, None
    return make(), make(), *(turn(torch.full(shape, math.nan, device="cuda")) for _ in range(2))


def same_bits(a, b):
    return a is None and b is None or torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


@pytest.mark.parametrize("kind", ["same", "f8", "f4"])
@pytest.mark.parametrize("tokens,q_heads,heads,dim,pairs,axes,neighbours,page,dtype,token_major", [
    (1, 4, 2, 64, 32, 1, False, 16, "bf16", False), (48, 32, 8, 128, 64, 1, False, 64, "bf16", False), (33, 0, 3, 96, 48, 2, False, 32, "f16", True),
    (130, 7, 7, 32, 16, 3, True, 128, "bf16", False), (9, 2, 1, 256, 128, 1, False, 8, "f16", False), (2500, 6, 2, 128, 20, 1, True, 64, "bf16", True),
    (17, 3, 1, 160, 36, 1, False, 1, "bf16", False)])
def test_append(gpu, tokens, q_heads, heads, dim, pairs, axes, neighbours, page, dtype, token_major, kind):
    g = torch.Generator().manual_seed(tokens + dim)
    dt = TYPES[dtype]
    pages = -(-tokens // page) + 2
    x = (torch.randn((tokens, q_heads + 2 * heads, dim), generator=g) * 3).to(dt).cuda()
    q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
    if tokens > 4:
        slots[2], slots[3] = -1, pages * page
    positions = torch.randint(0, 500000, (axes, tokens), generator=g, dtype=torch.int32).cuda()
    freq = frequencies(axes, pairs, g).cuda()
    kc, vc, ks, vs = caches(kind, dt, pages, heads, page, dim, token_major)
    q_out = torch.full((tokens, q_heads, dim), 5.0, dtype=dt, device="cuda")
    gpu.kv_append(k, v, positions, freq, slots.cuda(), kc, vc, ks, vs, q=q if q_heads else None, q_out=q_out if q_heads else None, neighbours=neighbours)
    # queries as rotate() turns them; values as kv_store() stores them; what no slot names stays as it was
    by_itself = torch.empty((1, tokens, q_heads + heads, dim), dtype=dt, device="cuda")
    gpu.rotate(x[None, :, :q_heads + heads], positions[:, None], freq, by_itself, neighbours=neighbours)
    assert torch.equal(q_out, by_itself[0, :, :q_heads])
    k2, v2, ks2, vs2 = caches(kind, dt, pages, heads, page, dim, token_major)
    gpu.kv_store(by_itself[0, :, q_heads:], v, slots.cuda(), k2, v2, ks2, vs2)
    assert same_bits(vc, v2) and same_bits(vs, vs2)
    if kind == "same":
        assert same_bits(kc, k2)
        return
    live = (slots >= 0) & (slots < pages * page)
    where = slots[live].long()
    flat = lambda t: t.cpu().transpose(1, 2).reshape(pages * page, *t.shape[1:2], *t.shape[3:])  # noqa: E731
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[where] = False
    as_bytes = lambda t: flat(t).reshape(-1).contiguous().view(torch.uint8).reshape(pages * page, -1)[rest]  # noqa: E731
    assert torch.equal(as_bytes(kc), as_bytes(k2)) and torch.equal(as_bytes(ks), as_bytes(ks2))
    # keys against 64 bits: half a step of the codes on top of the turned elements' own error
    want, off = turned(k[None], positions[:, None], freq, neighbours)
    want, off = want[0][live], off[0][live]
    if kind == "f8":
        scale = flat(ks)[where].double()
        assert bool(((scale - want.abs().amax(-1) / 448).abs() <= scale * 2.0 ** -23 + off.amax(-1) / 448).all())
        got = flat(kc.float())[where].double() * scale[..., None]
        step = torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * scale[..., None])
    else:
        scale = 2.0 ** (flat(ks)[where].double() - 127)
        top, slack = want.reshape(*want.shape[:-1], -1, 32).abs().amax(-1), off.reshape(*off.shape[:-1], -1, 32).amax(-1)
        assert bool((top <= 6 * scale + slack).all()) and bool((top > 3 * scale - slack).all())
        got = f4_ref.values(flat(kc), flat(ks))[where]
        s = scale.repeat_interleave(32, -1)
        step = torch.where(want.abs() <= 2 * s, 0.25 * s, torch.where(want.abs() <= 4 * s, 0.5 * s, s))
    assert bool(((got - want).abs() <= step * (1 + 2.0 ** -20) + off).all())


@pytest.mark.parametrize("kind", ["same", "f8", "f4"])
def test_append_without_pairs_is_store(gpu, kind):
    g = torch.Generator().manual_seed(4)
    k, v = ((torch.randn((77, 3, 64), generator=g) * 3).bfloat16().cuda() for _ in range(2))
    slots = torch.randperm(96, generator=g)[:77].to(torch.int32).cuda()
    a, b = (caches(kind, torch.bfloat16, 3, 3, 32, 64) for _ in range(2))
    empty = torch.zeros((1, 0), dtype=torch.float64, device="cuda")
    gpu.kv_append(k, v, torch.zeros((1, 77), dtype=torch.int32, device="cuda"), empty, slots, *a)
    gpu.kv_store(k, v, slots, *b)
    assert all(same_bits(x, y) for x, y in zip(a, b))


def test_nothing_to_turn(gpu):
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)):
        x = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
        gpu.rotate(x, torch.zeros((1, *shape[:2]), dtype=torch.int32, device="cuda"), torch.zeros((1, 32), dtype=torch.float64, device="cuda"), x)
    kc, vc, _, _ = caches("same", torch.bfloat16, 2, 2, 16, 64)
    k = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    gpu.kv_append(k, k, torch.zeros((1, 0), dtype=torch.int32, device="cuda"), torch.zeros((1, 32), dtype=torch.float64, device="cuda"),
                  torch.zeros(0, dtype=torch.int32, device="cuda"), kc, vc)
    torch.cuda.synchronize()
    assert bool(torch.isnan(kc).all())


def test_rows_past_32_bits(gpu):
    """Rows beyond 2^31 elements and 4 GB, of x and of out."""
    x = torch.zeros((1, 140000, 16, 1024), dtype=torch.bfloat16, device="cuda")[..., :128]  # 4.6 GB between the first row and the last
    x[0, -3:] = torch.randn((3, 16, 128)).bfloat16().cuda()
    positions = torch.arange(140000, dtype=torch.int32, device="cuda")[None, None]
    freq = frequencies(1, 64, torch.Generator().manual_seed(5)).cuda()
    last = torch.empty((1, 3, 16, 128), dtype=torch.bfloat16, device="cuda")
    gpu.rotate(x[:, -3:].contiguous(), positions[..., -3:], freq, last)
    gpu.rotate(x, positions, freq, x)
    assert torch.equal(x[:, -3:], last) and not bool(x[:, :-3].any())


def test_other_streams_and_graphs(gpu):
    g = torch.Generator().manual_seed(6)
    x = torch.randn((1, 300, 4, 64), generator=g).bfloat16().cuda()
    positions, freq = torch.arange(300, dtype=torch.int32, device="cuda")[None, None], frequencies(1, 32, g).cuda()
    want, off = turned(x, positions, freq, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(x)
    side.wait_stream(torch.cuda.current_stream())
    gpu.rotate(x, positions, freq, out, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    ref.assert_within(out, want, want.abs() * 2.0 ** -8 + off, "another stream")
    kc, vc, ks, vs = caches("f4", torch.bfloat16, 20, 2, 16, 64)
    slots = torch.arange(300, dtype=torch.int32, device="cuda")
    moved = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.kv_append(x[0, :, :2], x[0, :, 2:], positions[0], freq, slots, kc, vc, ks, vs, q=x[0], q_out=moved[0])
    for shift in (0, 1000, 5):
        positions.copy_(torch.arange(300, dtype=torch.int32, device="cuda") + shift)
        moved.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        gpu.rotate(x, positions, freq, out)
        again = caches("f4", torch.bfloat16, 20, 2, 16, 64)
        gpu.kv_append(x[0, :, :2], x[0, :, 2:], positions[0], freq, slots, *again)
        assert torch.equal(moved, out)
        assert all(same_bits(a.reshape(20, 2, 16, -1)[:18], b.reshape(20, 2, 16, -1)[:18]) for a, b in zip((kc, vc, ks, vs), again))
