"""Block-sparse attention, forward and backward, against its formulas in 64 bits: sizes around the tiles, lists that are
empty, unordered or point outside, masks that leave rows empty, strides, non-finite values where nothing is listed."""
import math

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def make(batch, queries, keys, heads, kv_heads, dim, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(s, generator=g) * spread).to(dtype).cuda()  # noqa: E731
    return r(batch, queries, heads, dim), r(batch, keys, kv_heads, dim), r(batch, keys, kv_heads, dim), r(batch, queries, heads, dim)


def random_lists(lists, rows, columns, most, seed, empty=0.1, ordered=True):
    g = torch.Generator().manual_seed(seed)
    pos, crd = [0], []
    for _ in range(lists * rows):
        n = 0 if torch.rand(1, generator=g) < empty or columns == 0 else int(torch.randint(1, min(most, columns) + 1, (1,), generator=g))
        c = torch.randperm(columns, generator=g)[:n]
        crd += (c.sort().values if ordered else c).tolist()
        pos.append(len(crd))
    return torch.tensor(pos, dtype=torch.int32).cuda(), torch.tensor(crd, dtype=torch.int32).cuda()


def run_forward(gpu, q, k, v, pos, crd, **sizes):
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), 7.0, device="cuda")
    gpu.block_attention(q, k, v, pos, crd, out, lse, **sizes)
    return out, lse


def run_backward(gpu, dout, q, k, v, out, lse, pos, crd, **sizes):
    grads = [torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda") for x in (q, k, v)]
    gpu.block_attention_backward(dout, q, k, v, out, lse, pos, crd, *grads, **sizes)
    return grads


def check(gpu, what, tensors, pos, crd, block_m, block_n, causal, scale=None, gradient=True):
    q, k, v, dout = tensors
    print("case", what, flush=True)
    sizes = dict(block_m=block_m, block_n=block_n, causal=causal, scale=scale)
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    torch.cuda.synchronize()
    scale = q.shape[3] ** -0.5 if scale is None else scale
    w = ref.pair_weights(pos, crd, q.shape[0], k.shape[2], q.shape[1], k.shape[1], block_m, block_n, causal)
    want, want_lse, bound, lse_bound = ref.forward(q, k, v, w, scale)
    ref.assert_within(out, want, bound, what + ": out")
    ref.assert_within(lse, want_lse, lse_bound, what + ": lse")
    if gradient:
        grads = run_backward(gpu, dout, q, k, v, out, lse, pos, crd, **sizes)
        torch.cuda.synchronize()
        wants, bounds = ref.backward(dout, q, k, v, out, lse, w, scale)
        for name, g, x, y in zip(("dq", "dk", "dv"), grads, wants, bounds):
            ref.assert_within(g, x, y, what + ": " + name)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("queries,keys,block_m,block_n,causal", [
    (1, 1, 1, 16, True), (1, 300, 1, 32, True), (2, 65, 64, 64, False), (17, 17, 16, 16, True), (63, 64, 64, 64, True),
    (65, 65, 64, 64, True), (127, 129, 128, 128, True), (200, 200, 37, 16, True), (130, 515, 50, 128, True),
    (96, 500, 128, 256, False), (257, 100, 64, 32, False), (100, 60, 16, 16, True), (33, 1, 8, 16, False)])
def test_sizes_around_the_tiles(gpu, dtype, queries, keys, block_m, block_n, causal):
    # 100 queries and 60 keys, causal: the first 40 queries see no key
    rows, columns = -(-queries // block_m), -(-keys // block_n)
    t = make(2, queries, keys, 4, 2, 64, TYPES[dtype], queries + keys)
    pos, crd = random_lists(4, rows, columns, 6, queries, empty=0.1)
    check(gpu, "%s %d x %d, blocks %d x %d" % (dtype, queries, keys, block_m, block_n), t, pos, crd, block_m, block_n, causal)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 80, 96, 104, 120, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_row_lengths(gpu, dim, dtype):
    t = make(1, 70, 150, 2, 1, dim, TYPES[dtype], dim)
    pos, crd = random_lists(1, 3, 5, 5, dim)
    check(gpu, "dim %d %s" % (dim, dtype), t, pos, crd, 32, 32, True)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (5, 1), (6, 2), (7, 1), (16, 1), (17, 1), (40, 2), (64, 1)])
@pytest.mark.parametrize("block_m", [1, 5, 64])
def test_groups_of_heads(gpu, heads, kv_heads, block_m):
    t = make(1, 45, 90, heads, kv_heads, 32, torch.bfloat16, heads)
    pos, crd = random_lists(kv_heads, -(-45 // block_m), 6, 4, heads + block_m)
    check(gpu, "%d heads over %d, %d queries a row" % (heads, kv_heads, block_m), t, pos, crd, block_m, 16, True)


@pytest.mark.parametrize("block_n", [16, 64, 256])
def test_full_lists_equal_dense_attention(gpu, block_n):
    t = make(1, 300, 300, 2, 2, 64, torch.bfloat16, 5)
    rows, columns = 5, -(-300 // block_n)
    pos = torch.arange(2 * rows + 1, dtype=torch.int32).cuda() * columns
    crd = torch.arange(columns, dtype=torch.int32).repeat(2 * rows).cuda()
    check(gpu, "all blocks of %d" % block_n, t, pos, crd, 64, block_n, True)


def test_nothing_listed_at_all(gpu):
    q, k, v, dout = make(1, 100, 100, 2, 1, 64, torch.bfloat16, 1)
    pos, crd = torch.zeros(3, dtype=torch.int32).cuda(), torch.zeros(0, dtype=torch.int32).cuda()
    check(gpu, "empty structure", (q, k, v, dout), pos, crd, 64, 64, True)


def test_no_queries_and_no_keys(gpu):
    for queries, keys in ((0, 50), (50, 0), (0, 0)):
        q, k, v, dout = make(1, queries, keys, 2, 1, 64, torch.bfloat16, 1)
        pos = torch.zeros(-(-queries // 16) + 1, dtype=torch.int32).cuda()
        crd = torch.zeros(0, dtype=torch.int32).cuda()
        out, lse = run_forward(gpu, q, k, v, pos, crd, block_m=16, block_n=16, causal=False)
        grads = run_backward(gpu, dout, q, k, v, out, lse, pos, crd, block_m=16, block_n=16, causal=False)
        torch.cuda.synchronize()
        assert all(bool((x == 0).all()) for x in (out, *grads)) and bool((lse == -math.inf).all())


def test_lists_out_of_order_twice_over_and_outside(gpu):
    t = make(1, 96, 200, 2, 1, 64, torch.float16, 3)
    # columns 0..6; the last one is cut at 200 keys
    pos = torch.tensor([0, 5, 5, 11], dtype=torch.int32).cuda()
    crd = torch.tensor([6, 0, 3, 0, -1, 2, 7, 1 << 30, -2147483648, 6, 2], dtype=torch.int32).cuda()
    check(gpu, "disorder", t, pos, crd, 32, 32, False)


def test_positions_that_start_past_the_first_entry_and_end_before_the_last(gpu):
    """Only what the rows name counts of a coordinate buffer that holds more; many entries in front, so that units of work
    come before the first column's."""
    t = make(1, 96, 200, 32, 1, 64, torch.float16, 3)
    front = 3000
    pos = (torch.tensor([0, 2, 2, 5], dtype=torch.int32) + front).cuda()
    crd = torch.zeros(front + 5 + 700, dtype=torch.int32)
    crd[front:front + 5] = torch.tensor([1, 4, 0, 3, 6])
    check(gpu, "positions from 3000", t, pos, crd.cuda(), 32, 32, False)


def test_positions_that_make_no_sense_are_not_followed(gpu):
    t = make(1, 96, 200, 2, 1, 64, torch.float16, 3)
    pos = torch.tensor([-5, 2, 1, 1000], dtype=torch.int32).cuda()  # rows [0, 2), nothing, [1, 4)
    crd = torch.tensor([0, 3, 5, 6], dtype=torch.int32).cuda()
    check(gpu, "positions", t, pos, crd, 32, 32, False)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("block_n", [16, 64, 128])
def test_what_no_query_attends_to_may_be_anything(gpu, bad, block_n):
    """Keys and values of unlisted blocks, and of listed blocks past every query's position."""
    queries = keys = 160
    q, k, v, dout = make(1, queries, keys, 2, 1, 64, torch.bfloat16, 9)
    rows, columns = 5, -(-keys // block_n)
    rows_listed = [[c for c in range(columns) if c * block_n <= 32 * r + 31] for r in range(rows)]
    pos = torch.tensor([0] + [sum(len(x) for x in rows_listed[:r + 1]) for r in range(rows)], dtype=torch.int32).cuda()
    crd = torch.tensor(sum(rows_listed, []), dtype=torch.int32).cuda()
    for at in (150, 159, 33):
        bk, bv = k.clone(), v.clone()
        bk[:, at:], bv[:, at:] = bad, bad
        # queries from `at` on do see those keys: only the rows before are compared
        out, _ = run_forward(gpu, q, bk, bv, pos, crd, block_m=32, block_n=block_n, causal=True)
        clean, _ = run_forward(gpu, q, k, v, pos, crd, block_m=32, block_n=block_n, causal=True)
        torch.cuda.synchronize()
        w = ref.pair_weights(pos, crd, 1, 1, queries, keys, 32, block_n, True)
        want, _, bound, _ = ref.forward(q, k, v, w, 64 ** -0.5)
        ref.assert_within(out[:, :at], want[:, :at], bound[:, :at], "rows before %d, %r" % (at, bad))
        ref.assert_within(clean, want, bound, "clean rows")


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_gradients_beside_values_that_nothing_attends_to(gpu, bad):
    """Keys past the last query's position and queries in front of the first key hold anything; their rows take no part."""
    q, k, v, dout = make(1, 90, 90, 2, 1, 64, torch.bfloat16, 4)
    pos, crd = torch.tensor([0, 1, 3, 6], dtype=torch.int32).cuda(), torch.tensor([0, 0, 1, 0, 1, 2], dtype=torch.int32).cuda()
    sizes = dict(block_m=32, block_n=32, causal=True)
    # keys 70.. are seen by queries 70.. only; their dout is zero and they are left out of the comparison
    w = ref.pair_weights(pos, crd, 1, 1, 90, 90, 32, 32, True)
    w[:, :, 70:] = 0
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    bk, bv, bq, bd = k.clone(), v.clone(), q.clone(), dout.clone()
    for x in (bk, bv, bq, bd):
        x[:, 70:] = bad
    bo, bl = out.clone(), lse.clone()
    bo[:, 70:], bl[:, :, 70:] = bad, bad
    dq, dk, dv = run_backward(gpu, bd, bq, bk, bv, bo, bl, pos, crd, **sizes)
    torch.cuda.synchronize()
    lse2, out2, dout2 = lse.clone(), out.clone(), dout.clone()
    wants, bounds = ref.backward(dout2, q, k, v, out2, lse2, w, 64 ** -0.5)
    ref.assert_within(dq[:, :70], wants[0][:, :70], bounds[0][:, :70], "dq before the bad keys")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_scores_and_scales(gpu, dtype):
    t = make(1, 64, 256, 2, 2, 64, TYPES[dtype], 8, spread=4.0)
    pos, crd = random_lists(2, 2, 4, 4, 2, empty=0.0)
    check(gpu, "scores of hundreds", t, pos, crd, 32, 64, False, scale=1.0)
    check(gpu, "negative scale", t, pos, crd, 32, 64, False, scale=-0.25)
    check(gpu, "scale 0", t, pos, crd, 32, 64, False, scale=0.0)


def test_scores_of_minus_infinity(gpu):
    q, k, v, _ = make(1, 32, 64, 1, 1, 64, torch.float16, 2)
    q[:, :, :, 0], k[:, :32, :, 0] = 60000.0, -math.inf
    pos, crd = torch.tensor([0, 2], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda()
    k[:, 32:, :, 0] = 0.0
    out, _ = run_forward(gpu, q, k, v, pos, crd, block_m=32, block_n=32, causal=False)
    only, _ = run_forward(gpu, q, k[:, 32:], v[:, 32:], torch.tensor([0, 1], dtype=torch.int32).cuda(),
                          torch.zeros(1, dtype=torch.int32).cuda(), block_m=32, block_n=32, causal=False)
    torch.cuda.synchronize()
    assert torch.equal(out, only)


def test_strides_of_slices_permuted_and_broadcast_operands(gpu):
    g = torch.Generator().manual_seed(6)
    packed = torch.randn((2, 130, 4 + 2 + 2, 64), generator=g).to(torch.bfloat16).cuda()
    q, k, v = packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:]
    dout = torch.randn((2, 4, 130, 64), generator=g).to(torch.bfloat16).cuda().transpose(1, 2)
    pos, crd = random_lists(4, 3, 5, 5, 3)
    check(gpu, "slices", (q, k, v, dout), pos, crd, 64, 32, True)
    k1 = torch.randn((1, 130, 1, 64), generator=g).to(torch.bfloat16).cuda().expand(2, 130, 2, 64)
    check(gpu, "broadcast keys and values", (q, k1, k1, dout), pos, crd, 64, 32, True)
    # outputs as slices of a larger tensor leave the rest of it alone
    big = torch.full((2, 130, 9, 72), 3.0, dtype=torch.bfloat16, device="cuda")
    out = big[:, :, 2:6, :64]
    lse = torch.empty((2, 4, 130), device="cuda")
    gpu.block_attention(q, k, v, pos, crd, out, lse, block_m=64, block_n=32)
    plain, _ = run_forward(gpu, q, k, v, pos, crd, block_m=64, block_n=32, causal=True)
    torch.cuda.synchronize()
    assert torch.equal(out, plain)
    out.fill_(3.0)
    assert bool((big == 3.0).all())


def test_offsets_beyond_32_bits(gpu):
    """Keys and values 2^31 elements apart: views into one large buffer."""
    stride = 1 << 24
    big = torch.empty(160 << 24, dtype=torch.bfloat16, device="cuda")
    q, k, v, dout = make(1, 40, 160, 2, 1, 64, torch.bfloat16, 12)
    far_k = torch.as_strided(big, (1, 160, 1, 64), (0, stride, 0, 1), 0)
    far_v = torch.as_strided(big, (1, 160, 1, 64), (0, stride, 0, 1), 64)
    far_k.copy_(k)
    far_v.copy_(v)
    assert stride * 159 > 1 << 31
    pos, crd = torch.tensor([0, 5, 10], dtype=torch.int32).cuda(), torch.tensor([0, 1, 2, 3, 4] * 2, dtype=torch.int32).cuda()
    check(gpu, "far apart", (q, far_k, far_v, dout), pos, crd, 32, 32, True)


def test_the_same_bits_again_and_on_another_stream(gpu):
    q, k, v, dout = make(2, 500, 500, 8, 2, 128, torch.bfloat16, 21)
    pos, crd = random_lists(4, 8, 8, 8, 7)
    sizes = dict(block_m=64, block_n=64, causal=True)
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    grads = run_backward(gpu, dout, q, k, v, out, lse, pos, crd, **sizes)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (None, side, side.cuda_stream):
        for _ in range(3):
            again = [torch.empty_like(x) for x in (out, lse, *grads)]
            gpu.block_attention(q, k, v, pos, crd, *again[:2], stream=stream, **sizes)
            gpu.block_attention_backward(dout, q, k, v, *again[:2], pos, crd, *again[2:], stream=stream, **sizes)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(again, (out, lse, *grads)))


def test_a_captured_graph_repeats(gpu):
    q, k, v, dout = make(1, 300, 300, 4, 2, 64, torch.float16, 31)
    pos, crd = random_lists(2, 5, 5, 4, 8)
    sizes = dict(block_m=64, block_n=64, causal=True)
    want = run_forward(gpu, q, k, v, pos, crd, **sizes)
    want += tuple(run_backward(gpu, dout, q, k, v, *want, pos, crd, **sizes))
    got = [torch.empty_like(x) for x in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.block_attention(q, k, v, pos, crd, *got[:2], **sizes)
        gpu.block_attention_backward(dout, q, k, v, *got[:2], pos, crd, *got[2:], **sizes)
    for _ in range(4):
        for x in got:
            x.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("which", [0, 1, 2])
def test_gradients_against_differences(gpu, which):
    """The formula's gradient in 64 bits, to which the kernels are held above, against central differences of the forward
    formula: both sides on the CPU."""
    g = torch.Generator().manual_seed(which)
    q, k, v, dout = (torch.randn(s, generator=g).double() for s in ((1, 9, 4, 8), (1, 12, 2, 8), (1, 12, 2, 8), (1, 9, 4, 8)))
    w = (torch.rand((1, 2, 9, 12), generator=g) < 0.5).double()
    w[:, :, 3] = 0

    def loss(*x):
        s = ref._heads_first(x[0]) @ ref._expand(ref._heads_first(x[1]), 2).transpose(2, 3) * 0.3
        p = ref._expand(w, 2) * torch.exp(s)
        total = p.sum(-1, keepdim=True)
        o = (p / torch.where(total == 0, 1.0, total)) @ ref._expand(ref._heads_first(x[2]), 2)
        return (o.transpose(1, 2) * dout).sum(), o.transpose(1, 2), torch.where(total == 0, -math.inf, torch.log(total))[..., 0]

    _, out, lse = loss(q, k, v)
    ref.HALF_ULP[torch.float64], ref.TINY[torch.float64] = 0.0, 0.0
    grads, _ = ref.backward(dout, q, k, v, out, lse, w, 0.3)
    x = [q, k, v]
    h = 1e-5
    for index in range(0, x[which].numel(), 7):
        sides = []
        for sign in (1, -1):
            moved = [t.clone() for t in x]
            moved[which].view(-1)[index] += sign * h
            sides.append(loss(*moved)[0])
        slope = float((sides[0] - sides[1]) / (2 * h))
        assert abs(slope - float(grads[which].reshape(-1)[index])) <= 1e-7 * (1 + abs(slope))


def test_the_c_entries_refuse(gpu):
    q, k, v, dout = make(1, 32, 32, 2, 1, 64, torch.bfloat16, 1)
    pos, crd = torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    out, lse = torch.empty_like(q), torch.empty((1, 2, 32), device="cuda")
    for bn in (8, 24, 512):
        with pytest.raises(gpu.LapisHipError, match="INVALID_ARGUMENT"):
            gpu.block_attention(q, k, v, torch.tensor([0, 1], dtype=torch.int32).cuda(), crd, out, lse, block_m=32, block_n=bn)
    q4, k4 = q[..., :60], k[..., :60]
    with pytest.raises(gpu.LapisHipError, match="multiple of 8"):
        gpu.block_attention(q4, k4, k4, pos, crd, torch.empty((1, 32, 2, 60), dtype=q.dtype, device="cuda"), lse, block_m=32, block_n=32)
    big = torch.empty((1, 32, 2, 136), dtype=q.dtype, device="cuda")
    with pytest.raises(gpu.LapisHipError, match="up to 128"):
        gpu.block_attention(big, big[:, :, :1], big[:, :, :1], pos, crd, torch.empty_like(big), lse, block_m=32, block_n=32)
    flat = torch.empty(1 * 32 * 2 * 64 + 1, dtype=q.dtype, device="cuda")[1:].view(1, 32, 2, 64)
    with pytest.raises(gpu.LapisHipError, match="16-byte"):
        gpu.block_attention(flat, k, v, pos, crd, out, lse, block_m=32, block_n=32)
    odd = torch.empty((1, 32, 2, 65), dtype=q.dtype, device="cuda")[..., :64]
    with pytest.raises(gpu.LapisHipError, match="multiples of 8"):
        gpu.block_attention(odd, k, v, pos, crd, out, lse, block_m=32, block_n=32)


# ---- many rows: workgroups of 128 rows, units from counters, the lists of columns in three launches ---------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("queries,keys,heads,block_m,block_n,dim,causal", [
    (300, 300, 8, 40, 16, 64, True), (300, 211, 8, 64, 32, 128, True), (257, 500, 16, 64, 64, 40, True),
    (300, 300, 24, 100, 128, 104, True), (200, 700, 8, 33, 256, 128, False), (330, 90, 16, 128, 64, 72, True)])
def test_many_rows(gpu, queries, keys, heads, block_m, block_n, dim, causal, dtype):
    # 8 key-value heads times 4 batch entries times two to ten rows of blocks: more than half a workgroup to a compute unit
    t = make(4, queries, keys, heads, 8, dim, TYPES[dtype], queries + dim)
    pos, crd = random_lists(32, -(-queries // block_m), -(-keys // block_n), 9, dim, empty=0.1)
    check(gpu, "%s %d x %d, %d heads, blocks %d x %d, dim %d" % (dtype, queries, keys, heads, block_m, block_n, dim), t, pos, crd, block_m,
          block_n, causal)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("block_n", [16, 64, 128])
def test_many_rows_beside_what_nothing_attends_to(gpu, bad, block_n):
    """Keys past every compared query's position, inside listed blocks and in unlisted ones, may hold anything."""
    q, k, v, dout = make(4, 160, 160, 16, 8, 64, torch.bfloat16, 9)
    rows, columns = 5, -(-160 // block_n)
    listed = [[c for c in range(columns) if c * block_n <= 32 * r + 31] for r in range(rows)] * 32
    pos = torch.tensor([0] + [len(x) for x in listed], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    crd = torch.tensor(sum(listed, []), dtype=torch.int32).cuda()
    sizes = dict(block_m=32, block_n=block_n, causal=True)
    w = ref.pair_weights(pos, crd, 4, 8, 160, 160, 32, block_n, True)
    want, want_lse, bound, _ = ref.forward(q, k, v, w, 64 ** -0.5)
    for at in (150, 33):
        bk, bv = k.clone(), v.clone()
        bk[:, at:], bv[:, at:] = bad, bad
        out, lse = run_forward(gpu, q, bk, bv, pos, crd, **sizes)
        dq, _, _ = run_backward(gpu, dout, q, bk, bv, out, lse, pos, crd, **sizes)
        torch.cuda.synchronize()
        ref.assert_within(out[:, :at], want[:, :at], bound[:, :at], "rows before %d, %r" % (at, bad))
        seen = w.clone()
        seen[:, :, at:] = 0  # the rows from `at` on are not compared
        wants, bounds = ref.backward(dout, q, k, v, torch.where(torch.isfinite(out), out, 0.0), torch.where(torch.isfinite(lse), lse, 0.0), seen, 64 ** -0.5)
        ref.assert_within(dq[:, :at], wants[0][:, :at], bounds[0][:, :at], "dq before %d, %r" % (at, bad))


def test_lists_of_many_blocks(gpu):
    """A few hundred entries to a row, in any order: more than a wavefront looks up at a time."""
    t = make(4, 96, 4100, 8, 8, 64, torch.bfloat16, 77)
    pos, crd = random_lists(32, 2, 257, 250, 3, empty=0.0, ordered=False)
    check(gpu, "long lists", t, pos, crd, 64, 16, True)


@pytest.mark.parametrize("queries,keys,block_m,block_n", [(1100, 1100, 2, 16), (60, 16500, 4, 16), (1030, 16500, 2, 16)])
def test_more_rows_or_columns_than_one_workgroup_lists(gpu, queries, keys, block_m, block_n):
    t = make(1, queries, keys, 1, 1, 16, torch.float16, queries)
    pos, crd = random_lists(1, -(-queries // block_m), -(-keys // block_n), 30, keys, empty=0.2)
    check(gpu, "%d rows, %d columns" % (pos.numel() - 1, -(-keys // block_n)), t, pos, crd, block_m, block_n, True)


def test_one_column_that_every_row_names(gpu):
    """Its entries are several units of work, added up afterwards; most columns have none."""
    t = make(1, 4000, 640, 4, 2, 64, torch.bfloat16, 5)
    rows = 63
    g = torch.Generator().manual_seed(2)
    other = torch.randint(1, 10, (2 * rows,), generator=g)
    crd = torch.stack([torch.zeros_like(other), other], 1).reshape(-1).to(torch.int32).cuda()
    pos = (torch.arange(2 * rows + 1) * 2).to(torch.int32).cuda()
    check(gpu, "a column of 63 entries", t, pos, crd, 64, 64, False)


def test_many_rows_the_same_bits_again_and_in_a_graph(gpu):
    q, k, v, dout = make(4, 500, 500, 16, 8, 64, torch.bfloat16, 21)
    pos, crd = random_lists(32, 8, 16, 12, 7)
    sizes = dict(block_m=64, block_n=32, causal=True)
    want = run_forward(gpu, q, k, v, pos, crd, **sizes)
    want += tuple(run_backward(gpu, dout, q, k, v, *want, pos, crd, **sizes))
    torch.cuda.synchronize()
    got = [torch.empty_like(x) for x in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.block_attention(q, k, v, pos, crd, *got[:2], **sizes)
        gpu.block_attention_backward(dout, q, k, v, *got[:2], pos, crd, *got[2:], **sizes)
    for _ in range(4):
        for x in got:
            x.fill_(5.0)
        graph.replay()
        again = run_forward(gpu, q, k, v, pos, crd, **sizes)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(torch.equal(x, y) for x, y in zip(again, want))


# ---- scratch memory and streams ------------------------------------------------------------------------------------------

def side_by_side(call, outputs):
    """``call(outputs, stream)`` queued several times on the current stream and, while these run, on another one that only waits
    for the inputs: both get what a call by itself gives."""
    call(outputs, None)
    torch.cuda.synchronize()
    want = [x.clone() for x in outputs]
    here, there = ([torch.empty_like(x) for x in outputs] for _ in range(2))
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        for x in here + there:
            x.zero_()
        ready = torch.cuda.Event()
        ready.record()
        side.wait_event(ready)
        for _ in range(4):
            call(here, None)
            call(there, stream)
        torch.cuda.synchronize()
        for name, got in (("the current stream", here), ("the other stream", there)):
            assert all(torch.equal(x, y) for x, y in zip(got, want)), "results on " + name


def test_scratch_of_calls_on_two_streams_is_not_shared(gpu):
    q, k, v, dout = make(2, 2000, 2000, 8, 2, 64, torch.bfloat16, 21)
    pos, crd = random_lists(4, 32, 63, 12, 7)
    sizes = dict(block_m=64, block_n=32, causal=True)
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    side_by_side(lambda grads, stream: gpu.block_attention_backward(dout, q, k, v, out, lse, pos, crd, *grads, stream=stream, **sizes),
                 [torch.zeros_like(x) for x in (q, k, v)])


def test_scratch_on_the_default_stream_while_another_one_is_current(gpu):
    q, k, v, dout = make(2, 2000, 2000, 8, 2, 64, torch.float16, 22)
    pos, crd = random_lists(4, 32, 63, 12, 8)
    sizes = dict(block_m=64, block_n=32, causal=True)
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    want = run_backward(gpu, dout, q, k, v, out, lse, pos, crd, **sizes)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [[torch.empty_like(x) for x in want] for _ in range(2)]
        side.synchronize()
        for _ in range(4):
            for grads, stream in zip(got, (None, 0)):
                gpu.block_attention_backward(dout, q, k, v, out, lse, pos, crd, *grads, stream=stream, **sizes)
        assert torch.cuda.current_stream() == side  # the calls leave it as it was
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for grads in got for x, y in zip(grads, want))


# ---- positions that descend --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("queries,block_m,columns", [(480, 16, 12), (1100, 2, 12), (480, 16, 1100)])
def test_rows_that_overlap(gpu, queries, block_m, columns):
    """Positions that go back twice within a list and once from one list to the next, in structures that one workgroup lists and
    in larger ones: the rows share entries, and each counts."""
    rows = -(-queries // block_m)
    t = make(2, queries, columns * 16, 2, 1, 64, torch.float16, rows)
    pos, crd = random_lists(2, rows, columns, 4, rows, empty=0.1)
    pos = pos.cpu()
    third = rows // 3
    pos[third] = max(0, int(pos[third]) - 20)
    pos[2 * third] = max(0, int(pos[2 * third]) - 9)
    pos[rows] = max(0, int(pos[rows]) - 30)
    assert 1 <= int((pos[1:] < pos[:-1]).sum()) <= 16
    check(gpu, "%d rows, %d columns" % (rows, columns), t, pos.cuda(), crd, block_m, 16, False)


def test_a_block_that_too_many_rows_name_where_rows_overlap(gpu):
    """Every row names block 0, each of the others a few: the gradient of block 0 says that it was not computed."""
    rows = 500
    t = make(1, rows, 160, 1, 1, 64, torch.bfloat16, 4)
    crd = torch.stack([torch.zeros(rows, dtype=torch.int32), torch.arange(rows, dtype=torch.int32) % 9 + 1], 1).reshape(-1).cuda()
    pos = torch.arange(rows + 1, dtype=torch.int32) * 2
    pos[200] -= 8
    pos, sizes = pos.cuda(), dict(block_m=1, block_n=16, causal=False)
    q, k, v, dout = t
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    dq, dk, dv = run_backward(gpu, dout, q, k, v, out, lse, pos, crd, **sizes)
    torch.cuda.synchronize()
    w = ref.pair_weights(pos, crd, 1, 1, rows, 160, 1, 16, False)
    wants, bounds = ref.backward(dout, q, k, v, out, lse, w, 64 ** -0.5)
    ref.assert_within(dq, wants[0], bounds[0], "dq")
    for name, g, x, y in (("dk", dk, wants[1], bounds[1]), ("dv", dv, wants[2], bounds[2])):
        assert bool(torch.isnan(g[:, :16]).all()), name
        ref.assert_within(g[:, 16:], x[:, 16:], y[:, 16:], name)


def block_args(**values):
    """The C structure of the entries' operands: tensors batch x tokens x heads x dim as rows, the rest as it is."""
    import ctypes

    class Rows(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("stride", ctypes.c_int64 * 3)]

    class Args(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_int64) for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim", "block_m", "block_n", "nnz")] +
                    [("causal", ctypes.c_int), ("dtype", ctypes.c_int), ("scale", ctypes.c_float), ("pos", ctypes.c_void_p), ("crd", ctypes.c_void_p)] +
                    [(n, Rows) for n in ("q", "k", "v", "out")] + [("lse", ctypes.c_void_p)] + [(n, Rows) for n in ("dout", "dq", "dk", "dv")] +
                    [("work", ctypes.c_void_p)])
    a = Args()
    for name, x in values.items():
        if not torch.is_tensor(x):
            setattr(a, name, x)
        elif x.dim() == 4:
            getattr(a, name).data = x.data_ptr()
            getattr(a, name).stride[:] = x.stride()[:3]
        else:
            setattr(a, name, x.data_ptr())
    return a


@pytest.mark.parametrize("queries,block_m,columns,entries", [(40, 1, 8, 30), (512, 1, 8, 1 << 24), (8192, 1, 8, 1 << 20), (600, 1, 9000, 1 << 20)])
def test_positions_that_go_up_and_down_write_nothing_outside(gpu, queries, block_m, columns, entries):
    """Rows that name all entries in turn with rows that name none: more entries together than 32 bits count.  Scratch
    memory stands between bytes that nothing may change."""
    import ctypes
    q, k, v, dout = make(1, queries, columns * 16, 1, 1, 8, torch.bfloat16, 5)
    pos = torch.zeros(queries + 1, dtype=torch.int32)
    pos[1::2] = entries
    crd = (torch.arange(entries, dtype=torch.int32) % columns).cuda()
    pos = pos.cuda()
    out, lse = torch.zeros_like(q), torch.full((1, 1, queries), 20.0, device="cuda")
    dq, dk, dv = (torch.full_like(x, 7.0) for x in (q, k, v))
    a = block_args(batch=1, queries=queries, keys=columns * 16, heads=1, kv_heads=1, dim=8, block_m=block_m, block_n=16, nnz=entries, causal=0,
                   dtype=0, scale=0.3, pos=pos, crd=crd, q=q, k=k, v=v, out=out, lse=lse, dout=dout, dq=dq, dk=dk, dv=dv)
    lib, bytes_ = gpu.load(), ctypes.c_int64()
    gpu.check(lib.lapis_hip_block_attention_backward_work(ctypes.byref(a), ctypes.byref(bytes_)))
    margin = 1 << 24
    work = torch.full((bytes_.value + 2 * margin,), 0xa5, dtype=torch.uint8, device="cuda")
    a.work = work.data_ptr() + margin
    torch.cuda.synchronize()
    gpu.check(lib.lapis_hip_block_attention_backward(ctypes.byref(a), None))
    torch.cuda.synchronize()
    assert bool((work[:margin] == 0xa5).all()) and bool((work[margin + bytes_.value:] == 0xa5).all())
    assert bool(torch.isnan(dk).all()) and bool(torch.isnan(dv).all())
    assert bool(torch.isfinite(dq).all()) and bool((dq[:, 1::2] == 0).all())  # rows that name nothing


def test_a_list_whose_keys_pass_31_bits(gpu):
    """Eight million entries of blocks that do not exist, then one that does: 2^31 keys into the list."""
    q, k, v, _ = make(1, 3, 600, 1, 1, 8, torch.bfloat16, 6)
    entries = (1 << 23) + 2
    crd = torch.full((entries,), -1, dtype=torch.int32)
    crd[-1] = 1
    pos = torch.tensor([0, entries], dtype=torch.int32).cuda()
    out, lse = run_forward(gpu, q, k, v, pos, crd.cuda(), block_m=3, block_n=256, causal=False)
    only = run_forward(gpu, q, k, v, torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.ones(1, dtype=torch.int32).cuda(), block_m=3, block_n=256,
                       causal=False)
    torch.cuda.synchronize()
    w = torch.zeros((1, 1, 3, 600), dtype=torch.float64)
    w[..., 256:512] = 1
    want, want_lse, bound, lse_bound = ref.forward(q, k, v, w, 8 ** -0.5)
    for o, l in ((out, lse), only):
        ref.assert_within(o, want, bound, "out")
        ref.assert_within(l, want_lse, lse_bound, "lse")


@pytest.mark.parametrize("change,what", [
    (dict(batch=64, heads=64, kv_heads=64, keys=1 << 30, block_n=16), "4096 lists of 67108864 columns"),       # 2^38 columns: 0 in 32 bits
    (dict(batch=300, heads=300, kv_heads=300), "90000 lists"),
    (dict(queries=1 << 30, block_m=1, heads=1), "67108864|rows of the structure"),
    (dict(nnz=2147483647, block_m=1 << 20, queries=1 << 20), "2147483649 units of work")])
def test_sizes_that_numbers_do_not_hold_are_refused_before_anything_is_launched(gpu, change, what):
    import ctypes
    x, lse = torch.full((1, 8, 1, 8), 7.0, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    sizes = dict(batch=1, queries=8, keys=32, heads=1, kv_heads=1, dim=8, block_m=8, block_n=16, nnz=0, causal=0, dtype=0, scale=1.0)
    a = block_args(**dict(sizes, **change), pos=pos, crd=pos, q=x, k=x, v=x, out=x, lse=lse, dout=x, dq=x, dk=x, dv=x)
    a.work = x.data_ptr()
    gpu.init()
    lib, bytes_ = gpu.load(), ctypes.c_int64(-1)
    for call in (lambda: lib.lapis_hip_block_attention_backward_work(ctypes.byref(a), ctypes.byref(bytes_)),
                 lambda: lib.lapis_hip_block_attention_backward(ctypes.byref(a), None)):
        with pytest.raises(gpu.LapisHipError, match=what):
            gpu.check(call())
    torch.cuda.synchronize()
    assert bool((x == 7.0).all())


# ---- operands that are not finite, and all three gradients --------------------------------------------------------------------------

@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("batch,kv_heads,block_m,block_n,dim", [(1, 1, 32, 16, 64), (1, 1, 32, 64, 128), (4, 8, 40, 32, 96), (4, 8, 64, 128, 64)])
def test_gradients_beside_queries_that_see_no_key(gpu, batch, kv_heads, block_m, block_n, dim, dtype, bad):
    """More queries than keys: what the first ones, in front of the first key, hold in any operand takes no part."""
    queries, keys, none = 170, 130, 40
    q, k, v, dout = make(batch, queries, keys, 2 * kv_heads, kv_heads, dim, TYPES[dtype], dim)
    rows, columns = -(-queries // block_m), -(-keys // block_n)
    n = batch * kv_heads * rows
    pos, crd = torch.arange(n + 1, dtype=torch.int32).cuda() * columns, torch.arange(columns, dtype=torch.int32).repeat(n).cuda()
    sizes = dict(block_m=block_m, block_n=block_n, causal=True)
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    bq, bd, bo = q.clone(), dout.clone(), out.clone()
    for x in (bq, bd, bo):
        x[:, :none] = bad
    again, _ = run_forward(gpu, bq, k, v, pos, crd, **sizes)
    grads = run_backward(gpu, bd, bq, k, v, bo, lse, pos, crd, **sizes)
    torch.cuda.synchronize()
    assert torch.equal(again, out) and bool((out[:, :none] == 0).all())
    w = ref.pair_weights(pos, crd, batch, kv_heads, queries, keys, block_m, block_n, True)
    wants, bounds = ref.backward(dout, q, k, v, out, lse, w, dim ** -0.5)
    for name, g, x, y in zip(("dq", "dk", "dv"), grads, wants, bounds):
        ref.assert_within(g, x, y, name)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("batch,kv_heads,block_m,block_n,dim", [(1, 1, 32, 16, 64), (1, 1, 32, 64, 128), (4, 8, 40, 32, 96), (4, 8, 64, 128, 64)])
def test_one_element_of_a_gradient_that_is_not_finite(gpu, batch, kv_heads, block_m, block_n, dim, dtype, bad):
    """It shows in that element of dV of the keys its query sees, in all of dK of these, and in its own row of dQ; everywhere else the
    gradients are as they would be.  Queries in tiles that the diagonal cuts, and one that sees whole tiles."""
    n = 200
    q, k, v, dout = make(batch, n, n, 2 * kv_heads, kv_heads, dim, TYPES[dtype], block_n)
    rows, columns = -(-n // block_m), -(-n // block_n)
    lists = batch * kv_heads * rows
    pos, crd = torch.arange(lists + 1, dtype=torch.int32).cuda() * columns, torch.arange(columns, dtype=torch.int32).repeat(lists).cuda()
    sizes = dict(block_m=block_m, block_n=block_n, causal=True)
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    w = ref.pair_weights(pos, crd, batch, kv_heads, n, n, block_m, block_n, True)
    for query, element in ((7, 3), (70, dim - 1), (150, 33)):
        there, zeroed = dout.clone(), dout.clone()
        there[:, query, 0, element], zeroed[:, query, 0, element] = bad, 0.0
        dq, dk, dv = (x.cpu() for x in run_backward(gpu, there, q, k, v, out, lse, pos, crd, **sizes))
        wants, bounds = ref.backward(zeroed, q, k, v, out, lse, w, dim ** -0.5)
        # dQ: all of the query's row of that head, and nothing else
        hit = torch.zeros(dq.shape, dtype=torch.bool)
        hit[:, query, 0] = True
        assert not bool(torch.isfinite(dq[hit]).any())  # dO v^T and the row sum, one from the other: NaN or infinite
        ref.assert_within(torch.where(hit, 0.0, dq.float()).to(dq.dtype), torch.where(hit, 0.0, wants[0]), bounds[0], "dq, query %d" % query)
        # dK: keys up to the query of that group; dV: that element of them
        hit = torch.zeros(dk.shape, dtype=torch.bool)
        hit[:, :query + 1, 0] = True
        assert not bool(torch.isfinite(dk[hit]).any())  # dO v^T and the row sum, one from the other: NaN or infinite
        ref.assert_within(torch.where(hit, 0.0, dk.float()).to(dk.dtype), torch.where(hit, 0.0, wants[1]), bounds[1], "dk, query %d" % query)
        hit = torch.zeros(dv.shape, dtype=torch.bool)
        hit[:, :query + 1, 0, element] = True
        want = torch.full(dv[hit].shape, bad, dtype=dv.dtype)
        assert torch.equal(dv[hit].nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))
        ref.assert_within(torch.where(hit, 0.0, dv.float()).to(dv.dtype), torch.where(hit, 0.0, wants[2]), bounds[2], "dv, query %d" % query)


@pytest.mark.parametrize("queries", [16, 4000])
def test_a_scale_that_is_not_a_number_shows(gpu, queries):
    q, k, v, dout = make(1, queries, 300, 2, 1, 64, torch.bfloat16, 3)
    rows = -(-queries // 16)
    pos, crd = torch.arange(rows + 1, dtype=torch.int32).cuda() * 2, torch.tensor([0, 3], dtype=torch.int32).repeat(rows).cuda()
    sizes = dict(block_m=16, block_n=64, causal=False, scale=math.nan)
    out, lse = run_forward(gpu, q, k, v, pos, crd, **sizes)
    grads = run_backward(gpu, dout, q, k, v, out, lse, pos, crd, **sizes)
    torch.cuda.synchronize()
    assert all(bool(torch.isnan(x).all()) for x in (out, lse, grads[0]))
    seen = [*range(64), *range(192, 256)]
    assert all(bool(torch.isnan(x[:, seen]).all()) for x in grads[1:])


def test_scratch_of_more_queries_times_entries_than_31_bits(gpu):
    """2^30 entries of 512 queries: sixteen to a unit of work."""
    import ctypes
    x, pos = torch.zeros((1, 8, 1, 8), dtype=torch.bfloat16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    a = block_args(batch=1, queries=512, keys=32, heads=1, kv_heads=1, dim=8, block_m=512, block_n=16, nnz=1 << 30, causal=0, dtype=0, scale=1.0,
                   pos=pos, crd=pos, q=x, k=x, v=x, out=x, lse=x.view(-1), dout=x, dq=x, dk=x, dv=x)
    gpu.init()
    bytes_ = ctypes.c_int64(-1)
    gpu.check(gpu.load().lapis_hip_block_attention_backward_work(ctypes.byref(a), ctypes.byref(bytes_)))
    partial, rows, units = 2 * (1 << 26) * 2 * 16 * 64 * 4, 4 << 30, 4 * ((1 << 26) + 2)
    assert partial + rows + units <= bytes_.value <= partial + rows + units + (1 << 20)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("batch,kv_heads,block_m,block_n,dim", [(1, 1, 16, 16, 64), (1, 1, 32, 64, 128), (4, 8, 40, 32, 96), (4, 8, 64, 128, 64)])
def test_keys_of_minus_infinity(gpu, batch, kv_heads, block_m, block_n, dim, dtype):
    """A key whose score is -infinity has no weight; in the one element it has infinite, dS k is 0 times infinity for the queries that see
    it, whether a mask cuts their tile or not, and everything else is as without the key."""
    n, element = 200, 5
    q, k, v, dout = make(batch, n, n, 2 * kv_heads, kv_heads, dim, TYPES[dtype], block_n + 1)
    q[..., element] = q[..., element].abs() + 1.0
    rows, columns = -(-n // block_m), -(-n // block_n)
    lists = batch * kv_heads * rows
    pos, crd = torch.arange(lists + 1, dtype=torch.int32).cuda() * columns, torch.arange(columns, dtype=torch.int32).repeat(lists).cuda()
    sizes = dict(block_m=block_m, block_n=block_n, causal=True)
    w = ref.pair_weights(pos, crd, batch, kv_heads, n, n, block_m, block_n, True)
    for key in (1, 77, 130):
        there, without, zeroed = k.clone(), w.clone(), k.clone()
        there[:, key, :, element], zeroed[:, key, :, element] = -math.inf, 0.0
        without[..., key] = 0
        out, lse = run_forward(gpu, q, there, v, pos, crd, **sizes)
        grads = run_backward(gpu, dout, q, there, v, out, lse, pos, crd, **sizes)
        torch.cuda.synchronize()
        want, want_lse, bound, lse_bound = ref.forward(q, zeroed, v, without, dim ** -0.5)
        ref.assert_within(out, want, bound, "out, key %d" % key)
        ref.assert_within(lse, want_lse, lse_bound, "lse, key %d" % key)
        wants, bounds = ref.backward(dout, q, zeroed, v, out, lse, without, dim ** -0.5)
        dq = grads[0].cpu()
        hit = torch.zeros(dq.shape, dtype=torch.bool)
        hit[:, key:, :, element] = True
        assert bool(torch.isnan(dq[hit]).all()), "key %d" % key
        ref.assert_within(torch.where(hit, 0.0, dq.float()).to(dq.dtype), torch.where(hit, 0.0, wants[0]), bounds[0], "dq, key %d" % key)
        for name, g, x, y in zip(("dk", "dv"), grads[1:], wants[1:], bounds[1:]):
            ref.assert_within(g, x, y, "%s, key %d" % (name, key))


@pytest.mark.parametrize("queries,block_m", [(96, 16), (1100, 2)])
def test_positions_outside_the_entries(gpu, queries, block_m):
    """Ascending ones in front of the first entry and behind the last: as if they were at the ends."""
    rows = -(-queries // block_m)
    t = make(1, queries, 200, 2, 1, 64, torch.float16, 3)
    pos, crd = random_lists(1, rows, 7, 4, rows, empty=0.1)
    pos = pos.cpu()
    pos[:2] -= 7
    pos[-2:] += 1000
    pos[0] = -2 ** 31
    pos[-1] = 2 ** 31 - 1
    check(gpu, "%d rows" % rows, t, pos.cuda(), crd, block_m, 32, True)


def test_scratch_that_is_not_on_a_boundary_is_refused(gpu):
    import ctypes
    x, lse = torch.full((1, 8, 1, 8), 7.0, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, device="cuda")
    pos, work = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    a = block_args(batch=1, queries=8, keys=32, heads=1, kv_heads=1, dim=8, block_m=8, block_n=16, nnz=0, causal=0, dtype=0, scale=1.0, pos=pos, crd=pos,
                   q=x, k=x, v=x, out=x, lse=lse, dout=x, dq=x, dk=x, dv=x)
    gpu.init()
    for at in (0, work.data_ptr() + 8):
        a.work = at
        with pytest.raises(gpu.LapisHipError, match="16-byte boundary"):
            gpu.check(gpu.load().lapis_hip_block_attention_backward(ctypes.byref(a), None))
    torch.cuda.synchronize()
    assert bool((x == 7.0).all())
