"""Attention over a window and the first keys, forward and backward, against 64 bits."""
import math

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def mask_of(batch, kv_heads, queries, keys, window, sink):
    p, j = torch.arange(queries)[:, None] + keys - queries, torch.arange(keys)
    seen = (j <= p) & ((j > p - window) | (j < sink))
    return seen.double().expand(batch, kv_heads, queries, keys)


def inputs(batch, queries, keys, heads, kv_heads, dim, dtype, seed=0, packed=False, spread=1.0):
    g = torch.Generator().manual_seed(seed + queries + keys + dim)
    dt = TYPES[dtype]
    if packed:
        x = (torch.randn((batch, queries, heads + 2 * kv_heads, dim), generator=g) * spread).to(dt).cuda()
        return x[:, :, :heads], x[:, :, heads:heads + kv_heads], x[:, :, heads + kv_heads:]
    make = lambda n, h: (torch.randn((batch, n, h, dim), generator=g) * spread).to(dt).cuda()  # noqa: E731
    return make(queries, heads), make(keys, kv_heads), make(keys, kv_heads)


def forward(gpu, q, k, v, window, sink, scale=None):
    out = torch.full(q.shape, 9.0, dtype=q.dtype, device="cuda")
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), 9.0, device="cuda")
    got = gpu.window_attention(q, k, v, out, window, sink, lse=lse, scale=scale)
    assert got[0] is out and got[1] is lse
    return out, lse


def backward(gpu, dout, q, k, v, out, lse, window, sink, scale=None):
    grads = [torch.full(x.shape, 9.0, dtype=x.dtype, device="cuda") for x in (q, k, v)]
    gpu.window_attention_backward(dout, q, k, v, out, lse, *grads, window, sink, scale=scale)
    return grads


SIZES = [  # batch, queries, keys, heads, kv_heads, dim, window, sink, dtype, packed
    (1, 1, 1, 1, 1, 8, 1, 0, "bf16", False), (1, 1, 700, 4, 2, 64, 100, 3, "f16", False), (2, 33, 33, 4, 2, 64, 1, 0, "bf16", True),
    (1, 130, 130, 3, 1, 72, 16, 1, "bf16", False), (2, 100, 333, 6, 2, 128, 64, 5, "f16", False), (1, 257, 257, 2, 2, 128, 1000, 0, "bf16", True),
    (1, 300, 300, 8, 8, 40, 65, 64, "bf16", False), (1, 513, 640, 5, 1, 96, 128, 200, "f16", False), (1, 200, 90, 4, 2, 64, 30, 7, "bf16", False),
    (1, 1000, 1000, 4, 1, 128, 127, 33, "bf16", True), (3, 65, 129, 40, 1, 64, 50, 16, "f16", False), (1, 64, 64, 140, 1, 32, 20, 2, "bf16", False),
    (1, 40, 500, 2, 1, 80, 10, 5000, "bf16", False), (1, 2100, 2100, 16, 8, 128, 300, 17, "bf16", False), (2, 1500, 2000, 8, 4, 64, 257, 0, "f16", False),
    (1, 3000, 3000, 8, 8, 64, 3000, 0, "bf16", False),
    (1, 1700, 1800, 12, 12, 104, 100, 40, "f16", False)]


@pytest.mark.parametrize("batch,queries,keys,heads,kv_heads,dim,window,sink,dtype,packed", SIZES)
def test_forward_and_backward(gpu, batch, queries, keys, heads, kv_heads, dim, window, sink, dtype, packed):
    q, k, v = inputs(batch, queries, keys, heads, kv_heads, dim, dtype, packed=packed)
    out, lse = forward(gpu, q, k, v, window, sink)
    w, scale = mask_of(batch, kv_heads, queries, keys, window, sink), dim ** -0.5
    want, want_lse, bound, lse_bound = ref.forward(q, k, v, w, scale)
    ref.assert_within(out, want, bound, "out")
    ref.assert_within(lse, want_lse, lse_bound, "lse")
    dout = inputs(batch, queries, keys, heads, kv_heads, dim, dtype, seed=5)[0]
    grads = backward(gpu, dout, q, k, v, out, lse, window, sink)
    want, bounds = ref.backward(dout, q, k, v, out, lse, w, scale)
    for name, got, x, b in zip(("dq", "dk", "dv"), grads, want, bounds):
        ref.assert_within(got, x, b, name)
    again = backward(gpu, dout, q, k, v, out, lse, window, sink)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(gpu, scale):
    q, k, v = inputs(1, 150, 150, 4, 2, 64, "bf16")
    out, lse = forward(gpu, q, k, v, 40, 3, scale)
    w = mask_of(1, 2, 150, 150, 40, 3)
    want, want_lse, bound, lse_bound = ref.forward(q, k, v, w, scale)
    ref.assert_within(out, want, bound, "out")
    ref.assert_within(lse, want_lse, lse_bound, "lse")
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    grads = backward(gpu, dout, q, k, v, out, lse, 40, 3, scale)
    for name, got, x, b in zip(("dq", "dk", "dv"), grads, *ref.backward(dout, q, k, v, out, lse, w, scale)):
        ref.assert_within(got, x, b, name)


def test_gradient_against_differences(gpu):
    """A step along each gradient's own direction, the output in 64 bits from the formulas."""
    q, k, v = inputs(1, 90, 90, 4, 2, 64, "bf16", spread=0.5)
    w, scale = mask_of(1, 2, 90, 90, 25, 6), 0.125
    out, lse = forward(gpu, q, k, v, 25, 6)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    grads = backward(gpu, dout, q, k, v, out, lse, 25, 6)

    def value(*x):
        Q, K, V = (t.double().cpu().transpose(1, 2) for t in x)
        K, V = K.repeat_interleave(2, 1), V.repeat_interleave(2, 1)
        s = torch.where(w.repeat_interleave(2, 1) > 0, scale * Q @ K.transpose(2, 3), -math.inf)
        return ((torch.softmax(s, -1) @ V) * dout.double().cpu().transpose(1, 2)).sum()

    x = [t.double().cpu() for t in (q, k, v)]
    for i, grad in enumerate(grads):
        d = grad.double().cpu()
        d = d / d.norm()
        h = 1e-4
        ahead, behind = ([t + (sign * h * d if j == i else 0.0) for j, t in enumerate(x)] for sign in (1, -1))
        slope = ((value(*ahead) - value(*behind)) / (2 * h)).item()
        # the gradient's own rounding (2^-8 of its norm) and that of weights and score gradients in 16 bits (2 * 2^-8)
        assert abs(slope - grad.double().norm().item()) <= 3 * 2.0 ** -8 * grad.double().norm().item()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("sizes", [(60, 2), (1100, 16)], ids=["few", "many"])
def test_values_that_are_not_finite_stay_with_who_sees_them(gpu, sizes, bad):
    """One key's value element, one key element, and one element of dout."""
    n, heads = sizes
    window, sink, at = 20, 3, n // 2
    q, k, v = inputs(1, n, n, heads, heads, 64, "bf16")
    p = torch.arange(n)
    sees = (p >= at) & (p < at + window)
    clean, clean_lse = forward(gpu, q, k, v, window, sink)
    v[0, at, 0, 5] = bad
    out, lse = forward(gpu, q, k, v, window, sink)
    want = clean.clone()
    assert not bool(torch.isfinite(out[0, sees, 0, 5]).any())
    want[0, sees, 0, 5] = out[0, sees, 0, 5]
    assert torch.equal(out.nan_to_num(), want.nan_to_num()) and torch.equal(lse, clean_lse)
    v[0, at, 0, 5] = 1.0
    out, lse = forward(gpu, q, k, v, window, sink)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    plain = backward(gpu, dout, q, k, v, out, lse, window, sink)
    dout[0, at, 0, 7] = bad  # of one query: to its own dq, to dv of the keys it sees in this element, to dk of those keys
    grads = backward(gpu, dout, q, k, v, out, lse, window, sink)
    seen = (p <= at) & ((p > at - window) | (p < sink))
    for name, got, was in zip(("dq", "dk", "dv"), grads, plain):
        touched = torch.zeros(got.shape, dtype=torch.bool)
        if name == "dq":
            touched[0, at, 0] = True
        elif name == "dk":
            touched[0, seen, 0] = True
        else:
            touched[0, seen, 0, 7] = True
        assert torch.equal(got.cpu()[~touched], was.cpu()[~touched]), name
        if name == "dv":
            assert not bool(torch.isfinite(got.cpu()[touched]).any())


def test_keys_that_are_not_finite_behind_every_mask(gpu):
    """Infinities and NaN in keys and values that no query sees: between the first keys and the windows."""
    for n, keys, heads in ((30, 400, 2), (1200, 1700, 16)):
        q, k, v = inputs(1, n, keys, heads, heads, 128, "bf16")
        out, lse = forward(gpu, q, k, v, 40, 10)
        dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
        grads = backward(gpu, dout, q, k, v, out, lse, 40, 10)
        unseen = slice(10, keys - n - 40 + 1)
        assert unseen.stop > 50
        k[:, unseen], v[:, unseen] = math.nan, math.inf
        out2, lse2 = forward(gpu, q, k, v, 40, 10)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        grads2 = backward(gpu, dout, q, k, v, out, lse, 40, 10)
        assert torch.equal(grads[0], grads2[0])
        for a, b in zip(grads[1:], grads2[1:]):
            assert torch.equal(a, b) and not bool(b[:, unseen].any())


def test_lse_is_optional_and_neighbouring_memory_stays(gpu):
    q, k, v = inputs(2, 77, 77, 4, 2, 64, "bf16")
    want, _ = forward(gpu, q, k, v, 30, 2)
    wide = torch.full((2, 77, 6, 80), 4.0, dtype=torch.bfloat16, device="cuda")
    assert gpu.window_attention(q, k, v, wide[:, :, 1:5, 8:72], 30, 2)[1] is None
    assert torch.equal(wide[:, :, 1:5, 8:72], want)
    wide[:, :, 1:5, 8:72] = 4.0
    assert bool((wide == 4.0).all())


def test_keys_and_values_of_one_row(gpu):
    """Broadcast inputs: one key for all places, one query for all heads."""
    g = torch.Generator().manual_seed(11)
    q = torch.randn((1, 50, 1, 64), generator=g).bfloat16().cuda().expand(1, 50, 4, 64)
    k = torch.randn((1, 1, 2, 64), generator=g).bfloat16().cuda().expand(1, 50, 2, 64)
    v = torch.randn((1, 50, 1, 64), generator=g).bfloat16().cuda().expand(1, 50, 2, 64)
    out, lse = forward(gpu, q, k, v, 9, 2)
    want = forward(gpu, q.contiguous(), k.contiguous(), v.contiguous(), 9, 2)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_a_long_context(gpu):
    """Offsets beyond 4 GB in keys and queries; the last queries against a short call on the same rows."""
    n = 300000
    x = torch.zeros((1, n, 8, 1024), dtype=torch.bfloat16, device="cuda")  # 4.9 GB; rows of 128 out of it
    g = torch.Generator().manual_seed(12)
    x[0, -400:, :, :128] = torch.randn((400, 8, 128), generator=g).bfloat16().cuda()
    x[0, :4, :, :128] = torch.randn((4, 8, 128), generator=g).bfloat16().cuda()
    q, k, v = x[..., :128], x[:, :, :2, :128], x[:, :, 2:4, :128]
    out, lse = forward(gpu, q, k, v, 200, 4)
    few = torch.cat([x[:, :4], x[:, -400:]], 1)
    part, part_lse = forward(gpu, few[:, -100:, :, :128], few[:, :, :2, :128], few[:, :, 2:4, :128], 200, 4)
    # the first keys stand elsewhere among the tiles, so sums differ in their order; weights in 16 bits of another maximum
    assert bool(((out[:, -100:].double() - part.double()).abs() <= 2.0 ** -6 * (part.double().abs() + 1)).all())
    assert bool(((lse[..., -100:] - part_lse).abs() <= 2.0 ** -18 * (1 + part_lse.abs())).all())


def test_two_graphs_and_streams(gpu):
    """Captured backward passes replayed in turn with eager ones, and calls on two streams at once."""
    q, k, v = inputs(1, 300, 300, 8, 2, 64, "bf16")
    douts = [torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(2)]
    out, lse = forward(gpu, q, k, v, 70, 5)
    eager = [backward(gpu, d, q, k, v, out, lse, 70, 5) for d in douts]
    graphs, results = [], []
    for d in douts:
        held = [torch.empty_like(x.contiguous()) for x in (q, k, v)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gpu.window_attention_backward(d, q, k, v, out, lse, *held, 70, 5)
        graphs.append(graph)
        results.append(held)
    for turn in range(3):
        for held in results:
            for x in held:
                x.fill_(3.0)
        for graph in graphs:
            graph.replay()
        backward(gpu, douts[0], q, k, v, out, lse, 70, 5)
        torch.cuda.synchronize()
        for held, want in zip(results, eager):
            assert all(torch.equal(a, b) for a, b in zip(held, want)), turn
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [[torch.empty_like(x.contiguous()) for x in (q, k, v)] for _ in range(2)]
    side.wait_stream(torch.cuda.current_stream())
    for i in range(2):
        gpu.window_attention_backward(douts[i], q, k, v, out, lse, *got[i], 70, 5, stream=side if i else None)
    torch.cuda.synchronize()
    for a, b in zip(got, eager):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("batch,queries,keys,heads", [(1, 9, 0, 2), (2, 0, 70, 2), (0, 5, 5, 2), (2, 4, 5, 0)])
def test_no_keys_or_no_queries(gpu, batch, queries, keys, heads):
    q, k, v = inputs(batch, queries, keys, heads, 1, 64, "bf16")
    out, lse = forward(gpu, q, k, v, 4, 4)
    grads = backward(gpu, torch.ones_like(q), q, k, v, out, lse, 4, 4)
    for x in grads + ([out] if keys == 0 else []):
        assert not bool(x.any())
    assert keys or bool((lse == -math.inf).all())
