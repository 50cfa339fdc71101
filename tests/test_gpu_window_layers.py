"""Turned positions, windows and small caches put together: a layer's gradients, and answers token by token."""
import pytest
import torch

import attention_ref as ref
import f4_ref
from test_gpu_rotate import turned
from test_gpu_window_attention import mask_of

pytestmark = pytest.mark.gpu


@pytest.fixture()
def attention(gpu):
    from lapis_amd import attention
    return attention


def frequencies(axes, pairs):
    f = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    return torch.where(torch.arange(pairs) % axes == torch.arange(axes)[:, None], f, 0.0)


@pytest.mark.parametrize("neighbours", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("batch,tokens,heads,kv_heads,dim,window,sink,dtype", [
    (1, 1, 1, 1, 32, 1, 0, torch.bfloat16), (2, 150, 4, 2, 64, 40, 5, torch.bfloat16), (1, 333, 6, 1, 128, 100, 0, torch.float16),
    (1, 700, 8, 4, 96, 130, 70, torch.bfloat16)])
def test_gradients_of_a_layer(attention, batch, tokens, heads, kv_heads, dim, window, sink, dtype, neighbours):
    """One row of keys for all key-value heads and one row of values for all batch entries: gradients of broadcast inputs."""
    g = torch.Generator().manual_seed(tokens)
    r = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()  # noqa: E731
    q, k, v = (x.requires_grad_() for x in (r(batch, tokens, heads, dim), r(batch, tokens, 1, dim), r(1, tokens, kv_heads, dim)))
    positions = torch.randint(0, 100000, (2, 1, tokens), generator=g, dtype=torch.int32).cuda().expand(2, batch, tokens)
    freq = frequencies(2, dim // 4)
    turn = lambda x: attention.rotate(x, positions, freq.cuda(), neighbours)  # noqa: E731
    qr, kr, vr = turn(q), turn(k.expand(-1, -1, kv_heads, -1)), v.expand(batch, -1, -1, -1)
    for x in (qr, kr, vr):
        x.retain_grad()
    for got, x in ((qr, q), (kr, k.expand(-1, -1, kv_heads, -1))):
        want, off = turned(x.detach(), positions, freq, neighbours)
        ref.assert_within(got, want, want.abs() * ref.HALF_ULP[dtype] + off + ref.HALF_STEP.get(dtype, 0.0), "turned")
    out = attention.attend_window(qr, kr, vr, window, sink)
    dout = r(batch, tokens, dim, heads).transpose(2, 3)  # not contiguous
    (out * dout).sum().backward()
    w, scale = mask_of(batch, kv_heads, tokens, tokens, window, sink), dim ** -0.5
    want, lse, bound, _ = ref.forward(qr, kr, vr, w, scale)
    ref.assert_within(out, want, bound, "out")
    wants, bounds = ref.backward(dout, qr, kr, vr, out, lse.float().cuda(), w, scale)
    for name, x, y, z in zip(("dq turned", "dk turned", "dv of each entry"), (qr, kr, vr), wants, bounds):
        ref.assert_within(x.grad, y, z, name)
    # turning back, from the gradients there were; a sum over heads or entries in 32 bits, rounded once
    dq, off = turned(qr.grad, positions, freq, neighbours, inverse=True)
    ref.assert_within(q.grad, dq, dq.abs() * ref.HALF_ULP[dtype] + off + ref.HALF_STEP.get(dtype, 0.0), "dq")
    dk, off = turned(kr.grad, positions, freq, neighbours, inverse=True)
    u, step = ref.HALF_ULP[dtype], ref.HALF_STEP.get(dtype, 0.0)
    each = (dk.abs() * (u + 2.0 ** -20) + off + step).sum(2, keepdim=True)  # each head's turned row is rounded, then the sum
    dk = dk.sum(2, keepdim=True)
    ref.assert_within(k.grad, dk, (dk.abs() + each) * u + each + step, "dk")
    dv = vr.grad.cpu().double()
    each = dv.abs().sum(0, keepdim=True) * 2.0 ** -20
    dv = dv.sum(0, keepdim=True)
    ref.assert_within(v.grad, dv, dv.abs() * u + each + step, "dv")
    # a sum's gradient is a broadcast one
    q.grad = None
    attention.attend_window(turn(q), kr.detach(), vr.detach(), window, sink).sum().backward()
    assert bool(torch.isfinite(q.grad).all())


@pytest.mark.parametrize("neighbours", [False, True], ids=["halves", "neighbours"])
def test_gradient_of_turning_against_differences(attention, neighbours):
    g = torch.Generator().manual_seed(4)
    x = torch.randint(-60, 61, (1, 40, 3, 64), generator=g).to(torch.bfloat16).cuda().requires_grad_()
    d = torch.randint(-1, 2, x.shape, generator=g).to(torch.bfloat16).cuda()
    w = torch.randn(x.shape, generator=g).to(torch.bfloat16).cuda()
    positions, freq = torch.arange(40, dtype=torch.int32).cuda().expand(1, 1, 40), frequencies(1, 24).cuda()
    attention.rotate(x, positions, freq, neighbours).backward(w)
    with torch.no_grad():  # integers: steps ahead and behind are exact
        ahead, behind = (attention.rotate(x + s * d, positions, freq, neighbours).double() for s in (1, -1))
    slope = ((ahead - behind) / 2 * w.double()).sum()
    bound = ((ahead.abs() + behind.abs()) / 2 * w.double().abs()).sum() + (x.grad.double() * d.double()).abs().sum()
    assert abs(slope - (x.grad.double() * d.double()).sum()) <= bound * 2.0 ** -8


def held(cache, kind, s):
    """What the cache holds of a sequence, in 64 bits: keys and values, tokens x heads x dim."""
    n, page = cache.lengths[s], cache.page
    pages = torch.tensor(cache.held[s][:-(-n // page)])
    rows = []
    for x, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = x[pages.cuda()].cpu()
        if kind == "f4":
            x = f4_ref.values(x, scale[pages.cuda()])
        elif kind == "f8":
            x = x.double() * scale[pages.cuda()].cpu().double()[..., None]
        rows.append(x.double().transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n])
    return rows


def half_step(kind, x):
    """The most by which storing rows x (64 bits) may change them."""
    if kind == "f4":
        s = 2.0 ** (f4_ref.scale_bytes(x, torch.bfloat16).double() - 127)
        return s.repeat_interleave(32, -1)  # neighbouring codes are at most 2 apart
    if kind == "f8":  # 2^-4 of the value, or half of 2^-9 of the scale; the scale and the quotient are 32-bit numbers
        return x.abs() * (2.0 ** -4 + 2.0 ** -20) + x.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10
    return x.abs() * 2.0 ** -8


@pytest.mark.parametrize("kind", ["bf16", "f8", "f4"])
@pytest.mark.parametrize("page,window,sink,given,neighbours", [(16, 40, 0, False, False), (32, 25, 5, True, False), (64, 1000, 3, False, True), (1, 3, 1, False, False)])
def test_answers_token_by_token(attention, gpu, kind, page, window, sink, given, neighbours):
    """Three sequences of different lengths, one of them empty at first, turned on their way into the cache; steps over a window and
    steps over all pages in turn."""
    g = torch.Generator().manual_seed(page)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    freq = frequencies(3, 28)
    cache = attention.PagedCache(3, 3 * -(-120 // page), 120, 2, 64, page=page, f8=kind == "f8", f4=kind == "f4", frequencies=freq.cuda(), neighbours=neighbours)
    numbers = lambda t: (torch.tensor([[t], [t * 7 % 50], [t + 3]]) if given else torch.tensor([[t]] * 3)).to(torch.int32)  # noqa: E731
    history = [[], [], []]
    for s, n in enumerate((37, 0, 64)):
        if n:
            q, k, v = r(n, 4, 64), r(n, 2, 64), r(n, 2, 64)
            positions = torch.cat([numbers(t) for t in range(n)], 1)
            got = cache.prefill(s, k, v, q, positions.cuda() if given else None)
            assert torch.equal(got, gpu.rotate(q[None], positions[:, None].cuda(), freq.cuda(), torch.empty_like(q)[None], neighbours)[0])
            history[s] += [(k[t], v[t], positions[:, t]) for t in range(n)]
    for step in range(40):
        q, k, v = r(3, 4, 64), r(3, 2, 64), r(3, 2, 64)
        positions = torch.cat([numbers(n) for n in cache.lengths], 1)
        at = positions.cuda() if given else None
        whole = step % 5 == 4
        out = cache.step(q, k, v, 120, positions=at) if whole else cache.step_window(q, k, v, window, sink, positions=at)
        for s in range(3):
            history[s].append((k[s], v[s], positions[:, s]))
            if step not in (0, 14, 27, 39):
                continue
            hk, hv = held(cache, kind, s)
            keys = torch.stack([h[0] for h in history[s]]).cpu()
            where = torch.stack([h[2] for h in history[s]], 1)[:, None]
            want, off = turned(keys[None], where, freq, neighbours)
            values = torch.stack([h[1] for h in history[s]]).cpu().double()
            # a scale or a code that stands at the edge between two may be either's
            off = off[0] * 2 if kind == "bf16" else off[0].amax(-1, keepdim=True) * 2
            assert bool(((hk - want[0]).abs() <= half_step(kind, want[0]) * (2 if kind == "f4" else 1) + off).all()), (step, s)
            assert bool(((hv - values).abs() <= half_step(kind, values)).all()), (step, s)
            qt = gpu.rotate(q[s][None, None], where[..., -1:].cuda(), freq.cuda(), torch.empty_like(q[s])[None, None], neighbours)
            n = len(history[s])
            w = torch.ones((1, 2, 1, n), dtype=torch.float64) if whole else mask_of(1, 2, 1, n, window, sink)
            want, _, bound, _ = ref.forward(qt, hk[None], hv[None], w, 64 ** -0.5)
            # weights times the scales of values are rounded once more than weights
            ref.assert_within(out[s][None, None], want, bound if kind == "bf16" else 2 * bound, "step %d, sequence %d" % (step, s))
    assert cache.lengths == [77, 40, 104] == cache.length.tolist()


def test_steps_give_what_one_pass_gives(attention):
    """Of a cache that keeps all bits: a prompt in one pass, then tokens one at a time, against one pass over all of them."""
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(s, generator=g).to(torch.bfloat16).cuda() for s in ((200, 8, 128), (200, 2, 128), (200, 2, 128)))
    freq = frequencies(1, 64).cuda()
    turn = lambda x: attention.rotate(x[None], torch.arange(200, dtype=torch.int32).cuda()[None, None], freq)  # noqa: E731
    whole = attention.attend_window(turn(q), turn(k), v[None], 50, 4)
    want, _, bound, _ = ref.forward(turn(q), turn(k), v[None], mask_of(1, 2, 200, 200, 50, 4), 128 ** -0.5)
    ref.assert_within(whole, want, bound, "one pass")
    cache = attention.PagedCache(1, 13, 208, 2, 128, page=16, frequencies=freq)
    assert torch.equal(cache.prefill(0, k[:150], v[:150], q[:150]), turn(q)[0, :150])
    steps = torch.cat([cache.step_window(q[t:t + 1], k[t:t + 1], v[t:t + 1], 50, 4) for t in range(150, 200)])
    assert torch.equal(held(cache, "bf16", 0)[0], turn(k)[0].cpu().double())
    ref.assert_within(steps, want[0, 150:], bound[0, 150:], "steps")


def test_a_captured_layer(attention):
    """Forward and backward pass in one graph, replayed between eager passes over other tokens."""
    g = torch.Generator().manual_seed(2)
    make = lambda: [torch.randn(s, generator=g).to(torch.bfloat16).cuda() for s in ((1, 300, 8, 64), (1, 300, 2, 64), (1, 300, 2, 64))]  # noqa: E731
    positions, freq = torch.arange(300, dtype=torch.int32).cuda()[None, None], frequencies(1, 32).cuda()

    def layer(q, k, v):
        out = attention.attend_window(attention.rotate(q, positions, freq), attention.rotate(k, positions, freq), v, 70, 5)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), torch.ones_like(out))

    def eager(tensors):
        return [x.clone() for x in layer(*(x.clone().requires_grad_() for x in tensors))]

    inputs = [x.requires_grad_() for x in make()]
    eager(make())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = layer(*inputs)
    for turn in range(3):
        fresh = make()
        with torch.no_grad():
            for x, y in zip(inputs, fresh):
                x.copy_(y)
        for x in results:
            x.fill_(3.0)
        graph.replay()
        want = eager(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, want)), turn


def test_second_derivatives_are_refused(attention):
    q, k, v = (torch.randn((1, 64, 2, 64), device="cuda").to(torch.bfloat16).requires_grad_() for _ in range(3))
    positions, freq = torch.zeros((1, 1, 64), dtype=torch.int32, device="cuda"), frequencies(1, 32).cuda()
    for f in (lambda x: attention.rotate(x, positions, freq), lambda x: attention.attend_window(x, k, v, 9)):
        dq, = torch.autograd.grad(f(q).float().square().sum(), q, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dq.float().square().sum().backward()


def test_positions_that_are_overwritten_before_the_gradient_are_noticed(attention):
    x = torch.randn((1, 8, 2, 64), device="cuda").to(torch.bfloat16).requires_grad_()
    positions = torch.zeros((1, 1, 8), dtype=torch.int32, device="cuda")
    out = attention.rotate(x, positions, frequencies(1, 32).cuda())
    positions.fill_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_refusals(attention, gpu):
    make = lambda **more: attention.PagedCache(2, 14, 96, 2, 64, page=16, **more)  # noqa: E731
    with pytest.raises(ValueError, match="codes of 8 bits and of 4 bits"):
        make(f8=True, f4=True)
    with pytest.raises(ValueError, match="rows of 40 elements"):
        attention.PagedCache(2, 14, 96, 2, 40, page=16, f4=True)
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    plain = make()
    positions = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    for call in (plain.step_window, plain.step):
        with pytest.raises(ValueError, match="positions, and no frequencies"):
            call(r(2, 4, 64), r(2, 2, 64), r(2, 2, 64), 3, positions=positions)
    with pytest.raises(ValueError, match="positions, and no frequencies"):
        plain.prefill(0, r(2, 2, 64), r(2, 2, 64), positions=positions)
    # two caches take the same tokens; one is asked for steps in between that are refused, just before a page is full and after
    caches = [make(f4=True, frequencies=frequencies(2, 32).cuda()) for _ in range(2)]
    for s, n in enumerate((31, 14)):
        k, v = r(n, 2, 64), r(n, 2, 64)
        for c in caches:
            c.prefill(s, k, v)
    for step in range(4):
        other = r(2, 4, 64), r(2, 2, 64), r(2, 2, 64)
        before = list(caches[0].lengths), caches[0].length.tolist()
        for error, call in (
                ((ValueError, gpu.LapisHipError), lambda: caches[0].step_window(*other, 0)), ((ValueError, gpu.LapisHipError), lambda: caches[0].step_window(*other, 5, -1)),
                (TypeError, lambda: caches[0].step_window(other[0].half(), *other[1:], 5)), (gpu.LapisHipError, lambda: caches[0].step_window(other[0][:, :3], *other[1:], 5)),
                (ValueError, lambda: caches[0].step_window(other[0], other[1], other[2][:1], 5)),
                (ValueError, lambda: caches[0].step_window(*other, 5, positions=positions)),  # one axis for two
                (ValueError, lambda: caches[0].step(other[0][:, :3], *other[1:], 4))):
            with pytest.raises(error):
                call()
        assert before == (caches[0].lengths, caches[0].length.tolist())
        q, k, v = r(2, 4, 64), r(2, 2, 64), r(2, 2, 64)
        out = [c.step(q, k, v, 4) if step % 2 else c.step_window(q, k, v, 20, 3) for c in caches]
        assert torch.equal(*out)
    assert caches[0].lengths == caches[1].lengths == [35, 18] == caches[0].length.tolist()


def test_every_output_counts_its_writes(gpu):
    b = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    u = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")  # noqa: E731
    x, out, lse, grads = b(1, 32, 1, 64), b(1, 32, 1, 64), torch.zeros((1, 1, 32), device="cuda"), [b(1, 32, 1, 64) for _ in range(3)]
    kc, vc, ks, vs = u(2, 1, 16, 32), u(2, 1, 16, 32), u(2, 1, 16, 2), u(2, 1, 16, 2)
    rows, q, one, sums, freq = [b(3, 1, 64) for _ in range(2)], b(3, 2, 64), b(1, 2, 64), torch.zeros((1, 2), device="cuda"), frequencies(1, 32).cuda()
    calls = [
        (lambda: gpu.rotate(x, i(1, 1, 32), freq, out), [out]),
        (lambda: gpu.kv_append(*rows, i(1, 3), freq, torch.arange(3, dtype=torch.int32).cuda(), kc, vc, ks, vs, q, q), [kc, vc, ks, vs, q]),
        (lambda: gpu.paged_window_attention(b(1, 2, 64), kc, vc, i(1, 1), i(1) + 3, one, 2, 1, sums, None, ks, vs), [one, sums]),
        (lambda: gpu.window_attention(x, x, x, out, 4, 1, lse), [out, lse]),
        (lambda: gpu.window_attention_backward(x, x, x, x, out, lse, *grads, 4, 1), grads)]
    for call, written in calls:
        before = [t._version for t in written]
        call()
        assert all(t._version > n for t, n in zip(written, before))
