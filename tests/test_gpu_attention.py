"""The operators of block-sparse attention put together: gradients through chosen blocks, a cache that grows token by token."""
import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture()
def attention(gpu):
    from lapis_amd import attention
    return attention


def test_gradients_through_chosen_blocks(attention):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(s, generator=g).to(torch.bfloat16).cuda().requires_grad_() for s in ((2, 200, 4, 64), (2, 200, 2, 64), (2, 200, 2, 64)))
    blocks = attention.choose_blocks(q, k, 4, 32, 16)
    out = attention.attend(q, k, v, blocks, 0.2)
    weight = torch.randn((2, 200, 64, 4), generator=g).to(torch.bfloat16).cuda().transpose(2, 3)  # a gradient that is not contiguous
    (out * weight).sum().backward()
    w = ref.pair_weights(blocks.pos, blocks.crd, 2, 2, 200, 200, 32, 16, True)
    assert int(w.amax()) == 1 and bool((w[:, :, torch.arange(200), torch.arange(200)] == 1).all())  # a query's own block is listed
    want, lse, bound, _ = ref.forward(q, k, v, w, 0.2)
    ref.assert_within(out, want, bound, "out")
    lse = lse.float().cuda()
    wants, bounds = ref.backward(weight, q, k, v, out, lse, w, 0.2)
    for name, x, y, z in zip(("dq", "dk", "dv"), (q, k, v), wants, bounds):
        ref.assert_within(x.grad, y, z, name)
    # a sum's gradient is a broadcast one
    q.grad = None
    attention.attend(q, k, v, blocks).sum().backward()
    assert bool(torch.isfinite(q.grad).all())


@pytest.mark.parametrize("f8", [False, True], ids=["bf16", "f8"])
def test_a_cache_that_grows(attention, f8):
    """Three sequences of different lengths, one of them empty at first; all pages are read, so that the answer is that of
    attention over everything."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    cache = attention.PagedCache(3, 30, 160, 2, 64, page=16, f8=f8)
    history = []
    for s, n in enumerate((37, 0, 64)):
        k, v = r(n, 2, 64), r(n, 2, 64)
        if n:
            cache.prefill(s, k, v)
        history.append([k, v])
    for step in range(40):
        q, k, v = r(3, 4, 64), r(3, 2, 64), r(3, 2, 64)
        out = cache.step(q, k, v, count=10)
        for s in range(3):
            history[s] = [torch.cat([history[s][0], k[s:s + 1]]), torch.cat([history[s][1], v[s:s + 1]])]
            if step % 13 == 0 or step == 39:
                hk, hv = history[s]
                if f8:
                    hk, hv = (codes(x) for x in (hk, hv))
                keys = hk.shape[0]
                want, _, bound, _ = ref.forward(q[s:s + 1, None], hk[None], hv[None], torch.ones((1, 2, 1, keys), dtype=torch.float64), 64 ** -0.5)
                ref.assert_within(out[s:s + 1, None], want, bound, "step %d, sequence %d" % (step, s))
    assert cache.lengths == [77, 40, 104] == cache.length.tolist()


def codes(x):
    """What an e4m3 cache holds of x; on the CPU, whose division by a number is a division."""
    x = x.cpu()
    scale = x.float().abs().amax(-1, keepdim=True) / 448.0
    return (x.float() / scale).to(torch.float8_e4m3fn).double() * scale.double()


def test_few_pages_of_a_long_sequence(attention):
    """The page a query is made for is found, and what it reads is attention over the chosen pages."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    cache = attention.PagedCache(1, 70, 1100, 1, 64, page=16)
    k, v = r(1001, 1, 64) * 0.1, r(1001, 1, 64)
    k[320:336] += 3.0 * r(1, 1, 64)
    cache.prefill(0, k, v)
    q = (k[325:326] * 2).expand(1, 2, 64).contiguous()
    nk, nv = r(1, 1, 64), r(1, 1, 64)
    out = cache.step(q, nk, nv, count=1 + 2 + 1)
    k, v = torch.cat([k, nk]), torch.cat([v, nv])
    # the first page, page 20 and the last two (the last holds 10 tokens)
    listed = torch.cat([torch.arange(16), torch.arange(320, 336), torch.arange(976, 1002)])
    w = torch.zeros((1, 1, 1, 1002), dtype=torch.float64)
    w[..., listed] = 1
    want, _, bound, _ = ref.forward(q[:, None], k[None], v[None], w, 64 ** -0.5)
    ref.assert_within(out[:, None], want, bound, "four pages")


def test_pages_run_out_and_come_back(attention):
    cache = attention.PagedCache(2, 4, 64, 1, 64, page=16)
    x = torch.ones((33, 1, 64), dtype=torch.bfloat16, device="cuda")
    cache.prefill(0, x, x)
    with pytest.raises(ValueError, match="holds 33 tokens"):
        cache.prefill(0, x, x)
    with pytest.raises(RuntimeError, match="2 more pages for sequence 1, 1 are free"):
        cache.prefill(1, x[:17], x[:17])
    assert cache.lengths == [33, 0] and len(cache.free) == 1
    cache.release(0)
    cache.prefill(1, x, x)
    assert len(cache.free) == 1 and cache.lengths == [0, 33]
    with pytest.raises(ValueError, match="local = 0"):
        cache.step(x[:2], x[:2], x[:2], 2, local=0)


def test_the_example(attention):
    lines = []
    losses, difference, answered = attention.main(tokens=1024, asked=64, steps=12, count=16, log=lines.append)
    assert losses[-1] < losses[0] and lines
    # both sides round to bf16 once or twice, of answers below 8 in size
    assert difference < (8 * 2.0 ** -8) ** 2 and answered == answered


def test_a_step_that_is_refused_changes_nothing(attention):
    """Two caches take the same tokens; one is asked for steps in between that are refused, just before a page is full and after."""
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    caches = [attention.PagedCache(2, 14, 96, 2, 64, page=16) for _ in range(2)]
    for s, n in enumerate((31, 14)):
        k, v = r(n, 2, 64), r(n, 2, 64)
        for c in caches:
            c.prefill(s, k, v)
    for step in range(4):
        other = r(2, 4, 64), r(2, 2, 64), r(2, 2, 64)
        before = list(caches[0].lengths), caches[0].length.tolist()
        with pytest.raises(ValueError, match="2 pages, the first 1 and the last 2"):
            caches[0].step(*other, count=2)
        with pytest.raises(ValueError, match="the first -1"):
            caches[0].step(*other, count=4, sink=-1)
        with pytest.raises(TypeError):
            caches[0].step(other[0].half(), *other[1:], count=4)       # queries of another type than the cache
        with pytest.raises(TypeError):
            caches[0].step(other[0], other[1].half(), other[2].half(), count=4)
        with pytest.raises(ValueError):
            caches[0].step(other[0], other[1], other[2][:1], count=4)
        with pytest.raises(ValueError):
            caches[0].step(other[0][:, :3], *other[1:], count=4)       # three heads over two
        assert before == (caches[0].lengths, caches[0].length.tolist())
        q, k, v = r(2, 4, 64), r(2, 2, 64), r(2, 2, 64)
        out = [c.step(q, k, v, count=4) for c in caches]
        assert torch.equal(*out)
    assert caches[0].lengths == caches[1].lengths == [35, 18] == caches[0].length.tolist()


def test_a_step_without_pages_gives_none_out(attention):
    cache = attention.PagedCache(3, 4, 64, 1, 64, page=16)
    x = torch.ones((16, 1, 64), dtype=torch.bfloat16, device="cuda")
    for s in range(3):
        cache.prefill(s, x, x)
    with pytest.raises(RuntimeError, match="1 more pages for sequence 1, 0 are free"):
        cache.step(x[:3], x[:3], x[:3], 4)
    assert len(cache.free) == 1 and cache.lengths == [16, 16, 16] and [len(h) for h in cache.held] == [1, 1, 1]
    # a released one gives its page back and begins anew with its next token
    cache.release(2)
    with pytest.raises(RuntimeError, match="1 more pages for sequence 2, 0 are free"):
        cache.step(x[:3], x[:3], x[:3], 4)
    assert len(cache.free) == 2 and cache.lengths == [16, 16, 0]
    cache.release(1)
    cache.step(x[:3], x[:3], x[:3], 4)
    assert cache.lengths == [17, 1, 1] == cache.length.tolist() and len(cache.free) == 0


def test_second_derivatives_are_refused(attention):
    q, k, v = (torch.randn((1, 64, 2, 64), device="cuda").to(torch.bfloat16).requires_grad_() for _ in range(3))
    out = attention.attend(q, k, v, attention.choose_blocks(q, k, 4, 16, 16))
    dq, = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dq.float().square().sum().backward()


def test_a_structure_that_is_overwritten_before_the_gradient_is_noticed(attention):
    from lapis_amd import hip
    q, k, v = (torch.randn((1, 64, 2, 64), device="cuda").to(torch.bfloat16).requires_grad_() for _ in range(3))
    codes, scales = torch.empty((1, 2, 4, 64), dtype=torch.int8, device="cuda"), torch.empty((1, 2, 4), device="cuda")
    hip.block_pool(k.detach(), 16, codes, scales)
    select = lambda b: hip.block_select(codes, codes, scales, 2, b.pos, b.crd, 64, 64, 16, 16)  # noqa: E731
    for late in (False, True):
        blocks = attention.choose_blocks(q, k, 2, 16, 16, sink=0, local=1)
        out = attention.attend(q, k, v, blocks)
        if not late:
            out.sum().backward()
            continue
        select(blocks)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_every_output_counts_its_writes(attention):
    from lapis_amd import hip
    b = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    codes, more = torch.zeros((1, 1, 2, 64), dtype=torch.int8, device="cuda"), f(1, 1, 2)
    q, out, lse, pos, crd, grads = b(1, 32, 1, 64), b(1, 32, 1, 64), f(1, 1, 32), i(3), i(4), [b(1, 32, 1, 64) for _ in range(3)]
    caches, scales, rows = [b(2, 1, 16, 64).to(torch.float8_e4m3fn) for _ in range(2)], [f(2, 1, 16) for _ in range(2)], [b(3, 1, 64) for _ in range(2)]
    one, sums = b(1, 1, 64), f(1, 1)
    calls = [
        (lambda: hip.block_pool(q, 16, codes, more), [codes, more]),
        (lambda: hip.block_select(codes, codes, more, 2, pos, crd, 32, 32, 16, 16), [pos, crd]),
        (lambda: hip.block_attention(q, q, q, pos, crd, out, lse, 16, 16), [out, lse]),
        (lambda: hip.block_attention_backward(q, q, q, q, out, lse, pos, crd, *grads, 16, 16), grads),
        (lambda: hip.kv_store(rows[0], rows[0], i(3) + torch.arange(3, dtype=torch.int32, device="cuda"), *caches, *scales), caches + scales),
        (lambda: hip.kv_load(*caches, i(3), *rows, *scales), rows),
        (lambda: hip.paged_attention(one, *caches, i(2), i(0), i(1), out[:1, :1, 0], sums, None, *scales), [sums])]
    for call, outputs in calls:
        before = [x._version for x in outputs]
        call()
        assert all(x._version == n + 1 for x, n in zip(outputs, before))
    with torch.inference_mode():
        kept = b(1, 32, 1, 64)
    hip.block_attention(q, q, q, pos, crd, kept, lse, 16, 16)  # a tensor without a version is written as any other
    torch.cuda.synchronize()
