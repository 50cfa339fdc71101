"""8-bit block means and the selection of blocks: exact, ties to the lowest block."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,tokens,heads,groups,dim,block", [
    (1, 1, 1, 1, 8, 1), (2, 100, 4, 2, 64, 16), (1, 333, 3, 3, 72, 100), (1, 64, 16, 1, 128, 64), (3, 17, 6, 2, 128, 1), (1, 40, 1, 1, 128, 1),
    (1, 50, 8, 8, 256, 64), (1, 1000, 5, 1, 136, 1000), (2, 90, 2, 2, 40, 7), (1, 9, 70, 2, 64, 4)])
def test_pool(gpu, batch, tokens, heads, groups, dim, block, dtype):
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn((batch, tokens, heads, dim), generator=g).to(dtype)
    blocks = -(-tokens // block)
    codes = torch.full((batch, groups, blocks, dim), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((batch, groups, blocks), 7.0, device="cuda")
    print("case", batch, tokens, heads, groups, dim, block, flush=True)
    gpu.block_pool(x.cuda(), block, codes, scales)
    torch.cuda.synchronize()
    for j in range(blocks):
        part = x[:, j * block:(j + 1) * block].double()
        n = part.shape[1] * heads // groups
        mean = part.reshape(batch, -1, groups, heads // groups, dim).mean((1, 3))
        size = part.abs().reshape(batch, -1, groups, heads // groups, dim).mean((1, 3))
        err = n * 2.0 ** -23 * size                     # of an fp32 sum of n terms
        s = scales[:, :, j].cpu().double()
        top = mean.abs().amax(-1) / 127
        assert bool(((s - top).abs() <= err.amax(-1) / 127 + 2.0 ** -22 * top).all())
        got = codes[:, :, j].cpu().double() * s[..., None]
        # half a code, the sum's error, and what the division may turn over at a tie
        assert bool(((got - mean).abs() <= s[..., None] * (0.5 + 1e-4) + 2 * err).all())
        assert int(codes[:, :, j].cpu().abs().amax()) in (0, 127)


def test_pool_of_zeros_and_of_values_that_are_not_finite(gpu):
    x = torch.ones((1, 4 * 16, 1, 64), dtype=torch.bfloat16, device="cuda")
    x[:, :16] = 0.0
    x[:, 20, :, 3] = math.nan
    x[:, 40, :, 3] = math.inf
    codes, scales = torch.full((1, 1, 4, 64), 9, dtype=torch.int8, device="cuda"), torch.empty((1, 1, 4), device="cuda")
    gpu.block_pool(x, 16, codes, scales)
    s = scales.cpu()[0, 0]
    assert s[0] == 0 and math.isnan(s[1]) and math.isnan(s[2]) and abs(float(s[3]) - 1 / 127) < 1e-8
    assert not bool(codes[0, 0, :3].any()) and bool((codes[0, 0, 3] == 127).all())


def reference(q, k, s, count, seen, sink, local):
    """Columns of one row: q (dim), k (columns x dim), s (columns), on the CPU."""
    score = np.where(np.isnan(s[:seen]), -np.inf, (k[:seen].astype(np.int64) @ q.astype(np.int64)).astype(np.float32) * s[:seen]) if seen else np.zeros(0)
    nan = np.isnan(s[:seen])
    rank = sorted(range(seen), key=lambda j: (0 if j < sink or j >= seen - local else 1, 0 if j < sink or j >= seen - local else int(nan[j]),
                                              0.0 if j < sink or j >= seen - local or nan[j] else -float(score[j]), j))
    return sorted(rank[:count])


def run_select(gpu, q, k, s, count, queries, keys, m, n, causal, sink, local):
    batch, heads, rows, _ = q.shape
    pos = torch.full((batch * heads * rows + 1,), -9, dtype=torch.int32, device="cuda")
    crd = torch.full((batch * heads * rows * min(count, k.shape[2]) + 5,), -9, dtype=torch.int32, device="cuda")
    gpu.block_select(q.cuda(), k.cuda(), s.cuda(), count, pos, crd, queries=queries, keys=keys, block_m=m, block_n=n, causal=causal,
                     sink=sink, local=local)
    torch.cuda.synchronize()
    return pos.cpu().numpy(), crd.cpu().numpy()


@pytest.mark.parametrize("queries,keys,m,n,count,causal,sink,local,dim", [
    (1, 1, 1, 16, 1, True, 0, 1, 8), (100, 100, 1, 4, 5, True, 1, 1, 64), (100, 130, 16, 8, 4, True, 1, 2, 72), (64, 2000, 8, 4, 7, False, 0, 0, 128),
    (300, 300, 7, 3, 9, True, 0, 1, 128), (40, 700, 3, 2, 64, False, 1, 1, 256), (90, 50, 4, 4, 3, True, 1, 1, 16), (33, 9000, 33, 1, 100, False, 2, 2, 40),
    (50, 5000, 10, 1, 17, True, 0, 1, 128), (20, 100, 5, 10, 50, True, 3, 4, 1024), (17, 64, 1, 1, 64, False, 0, 0, 8)])
def test_selection_is_exact(gpu, queries, keys, m, n, count, causal, sink, local, dim):
    rng = np.random.default_rng(queries + keys)
    rows, columns = -(-queries // m), -(-keys // n)
    q = rng.integers(-127, 128, (2, 3, rows, dim)).astype(np.int8)
    k = rng.integers(-127, 128, (2, 3, columns, dim)).astype(np.int8)
    s = rng.uniform(0, 0.1, (2, 3, columns)).astype(np.float32)
    s[:, 0] = np.float32(0.01)
    k[:, 0] = rng.integers(-1, 2, k[:, 0].shape) * (rng.random(k[:, 0].shape) < 4 / dim)      # scores full of ties
    q[:, 0] = rng.integers(-1, 2, q[:, 0].shape)
    s[0, 1, rng.random(columns) < 0.2] = np.nan
    print("case", queries, keys, m, n, count, flush=True)
    pos, crd = run_select(gpu, *(torch.from_numpy(x) for x in (q, k, s)), count, queries, keys, m, n, causal, sink, local)
    at = 0
    for b in range(2):
        for h in range(3):
            for r in range(rows):
                last = min((r + 1) * m, queries) - 1
                seen = min(max((last + keys - queries) // n + 1, 0), columns) if causal else columns
                want = reference(q[b, h, r], k[b, h], s[b, h], count, seen, sink, local)
                row = (b * 3 + h) * rows + r
                assert pos[row] == at
                assert crd[at:at + len(want)].tolist() == want, (b, h, r)
                at += len(want)
    assert pos[-1] == at and bool((crd[at:] == -9).all())


def test_scores_at_the_ends(gpu):
    """Scales of 0, -0, infinity and negative ones: equal scores go to the lowest block, NaN (0 times infinity) last."""
    q = torch.full((1, 1, 1, 8), 1, dtype=torch.int8)
    k = torch.zeros((1, 1, 12, 8), dtype=torch.int8)
    k[..., 0] = torch.tensor([1, -1, 0, 1, 1, 0, -1, 1, 5, 0, 1, -1], dtype=torch.int8)
    s = torch.tensor([[[0.0, 0.0, 3.0, -0.0, 1e-30, math.inf, math.inf, math.inf, -1.0, 2.0, 1e-30, 1e-45]]])
    for count in range(1, 13):
        _, crd = run_select(gpu, q, k, s, count, 1, 12, 1, 1, False, 0, 0)
        # 7: inf; 4, 10: 1e-30; zeros of either sign 0 1 2 3 9; 11: -1e-45; 8: -5; 6: -inf; 5: NaN
        assert crd[:count].tolist() == sorted([7, 4, 10, 0, 1, 2, 3, 9, 11, 8, 6, 5][:count])


def test_no_rows_and_no_columns(gpu):
    for queries, keys in ((0, 64), (64, 0)):
        q = torch.zeros((2, 2, queries // 16, 64), dtype=torch.int8)
        k, s = torch.zeros((2, 2, keys // 16, 64), dtype=torch.int8), torch.zeros((2, 2, keys // 16))
        pos, _ = run_select(gpu, q, k, s, 4, queries, keys, 16, 16, False, 0, 0)
        assert bool((pos == 0).all())


def test_selection_over_a_cache(gpu):
    rng = np.random.default_rng(4)
    pages, heads, dim, width, count = 40, 3, 64, 20, 6
    blocks = np.array([20, 0, 3, 7, 25, 1, -2], dtype=np.int32)  # 25 and -2: as many as the table is wide, none
    table = rng.integers(0, pages, (7, width)).astype(np.int32)
    table[3, 2] = -1
    table[0, 5] = pages
    q = rng.integers(-127, 128, (7, heads, 1, dim)).astype(np.int8)
    k = rng.integers(-127, 128, (pages, heads, dim)).astype(np.int8)
    s = rng.uniform(0, 1, (pages, heads)).astype(np.float32)
    pos = torch.full((7 * heads + 1,), -9, dtype=torch.int32, device="cuda")
    crd = torch.full((7 * heads * count,), -9, dtype=torch.int32, device="cuda")
    gpu.block_select(*(torch.from_numpy(x).cuda() for x in (q, k, s)), count, pos, crd, queries=1, keys=width, block_m=1, block_n=1,
                     causal=False, sink=1, local=1, table=torch.from_numpy(table).cuda(), blocks=torch.from_numpy(blocks).cuda())
    pos, crd = pos.cpu().numpy(), crd.cpu().numpy()
    at = 0
    for b in range(7):
        for h in range(heads):
            seen = min(max(int(blocks[b]), 0), width)
            page = np.clip(table[b], 0, pages - 1)
            scale = np.where((table[b] >= 0) & (table[b] < pages), s[page, h], np.nan).astype(np.float32)
            want = reference(q[b, h, 0], k[page, h], scale, count, seen, 1, 1)
            assert pos[b * heads + h] == at
            assert crd[at:at + len(want)].tolist() == [int(table[b, j]) for j in want], (b, h)
            at += len(want)
    assert pos[-1] == at and bool((crd[at:] == -9).all())


def test_the_c_entries_refuse(gpu):
    z8 = lambda *s: torch.zeros(s, dtype=torch.int8, device="cuda")  # noqa: E731
    pos, crd = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(20, dtype=torch.int32, device="cuda")
    good = dict(queries=2, keys=4, block_m=1, block_n=1, causal=False, sink=0, local=0)
    call = lambda dim, count, **more: gpu.block_select(z8(1, 1, 2, dim), z8(1, 1, 4, dim), torch.zeros((1, 1, 4), device="cuda"), count, pos, crd,  # noqa: E731
                                                       **dict(good, **more))
    call(8, 1)
    for dim, count, more in ((12, 1, {}), (1032, 1, {}), (8, 0, {}), (8, 1, {"sink": 1, "local": 1}), (8, 1, {"sink": -1})):
        with pytest.raises(gpu.LapisHipError, match="INVALID_ARGUMENT"):
            call(dim, count, **more)


def best_on_the_device(q, k, s, count, sink, local):
    """Columns of each row (rows x dim against columns x dim, every row sees all) by a stable sort: whole-number products are exact."""
    best = []
    for part in q.split(max(1, (1 << 27) // k.shape[0])):
        score = (part.float() @ k.float().T.contiguous()) * s
        score[:, :sink], score[:, k.shape[0] - local:] = math.inf, math.inf
        best.append(score.sort(dim=1, descending=True, stable=True).indices[:, :count].sort(dim=1).values)
    return torch.cat(best)


@pytest.mark.parametrize("rows,columns,dim,count", [(2000, 70001, 64, 5), (9_700_000, 7, 264, 3)])
def test_rows_whose_scores_take_several_launches(gpu, rows, columns, dim, count):
    """256 MB of scores at a time: rows of the second and third launch; and launches of so many rows that their grid is rounded up,
    with bytes behind the scratch memory that nothing may change."""
    import ctypes
    from test_block_attention_binding import SelectArgs
    assert rows * columns * 4 > 1 << 28
    g = torch.Generator(device="cuda").manual_seed(rows)
    q = torch.randint(-127, 128, (rows, dim), dtype=torch.int8, device="cuda", generator=g)
    k = torch.randint(-127, 128, (columns, dim), dtype=torch.int8, device="cuda", generator=g)
    s = torch.rand(columns, device="cuda", generator=g) + 0.01
    pos = torch.full((rows + 1,), -9, dtype=torch.int32, device="cuda")
    crd = torch.full((rows * count,), -9, dtype=torch.int32, device="cuda")
    a = SelectArgs(batch=1, heads=1, queries=rows, keys=columns, dim=dim, block_m=1, block_n=1, count=count, sink=1, local=1, causal=0,
                   q_codes=q.data_ptr(), k_codes=k.data_ptr(), k_scales=s.data_ptr(), k_stride=(columns * dim, columns * dim, dim),
                   scale_stride=(columns, columns, 1), pos=pos.data_ptr(), crd=crd.data_ptr())
    gpu.init()
    lib, bytes_ = gpu.load(), ctypes.c_int64()
    gpu.check(lib.lapis_hip_block_select_work(ctypes.byref(a), ctypes.byref(bytes_)))
    assert bytes_.value <= 1 << 28
    work = torch.full((bytes_.value + (1 << 28),), 0xa5, dtype=torch.uint8, device="cuda")
    a.work = work.data_ptr()
    torch.cuda.synchronize()
    gpu.check(lib.lapis_hip_block_select(ctypes.byref(a), None))
    torch.cuda.synchronize()
    assert bool((work[bytes_.value:] == 0xa5).all())
    assert torch.equal(pos, torch.arange(0, rows * count + 1, count, dtype=torch.int32, device="cuda"))
    assert torch.equal(crd.view(rows, count).long(), best_on_the_device(q, k, s, count, 1, 1))


@pytest.mark.parametrize("block", [1, 16])
def test_pool_of_no_heads(gpu, block):
    """The mean over no heads is not finite: codes 0, scales NaN, not what the outputs held."""
    x = torch.empty((2, 32, 0, 64), dtype=torch.bfloat16, device="cuda")
    codes, scales = torch.full((2, 3, 32 // block, 64), 9, dtype=torch.int8, device="cuda"), torch.full((2, 3, 32 // block), 7.0, device="cuda")
    gpu.block_pool(x, block, codes, scales)
    torch.cuda.synchronize()
    assert not bool(codes.any()) and bool(torch.isnan(scales).all())


def test_pool_of_a_block_longer_than_any_number_of_tokens(gpu):
    x = torch.randn((1, 40, 4, 64), device="cuda").to(torch.bfloat16)
    results = []
    for block in (40, 2 ** 62, 2 ** 63 - 1):
        codes, scales = torch.full((1, 2, 1, 64), 9, dtype=torch.int8, device="cuda"), torch.full((1, 2, 1), 7.0, device="cuda")
        gpu.block_pool(x, block, codes, scales)
        results.append((codes, scales))
    torch.cuda.synchronize()
    assert all(torch.equal(c, results[0][0]) and torch.equal(s, results[0][1]) for c, s in results)
    assert int(results[0][0].abs().max()) == 127


@pytest.mark.parametrize("dim", [40, 128, 256])
@pytest.mark.parametrize("columns", [256, 257, 512, 513, 1024, 1025, 1500, 2048, 2049])
def test_selection_at_the_widths_where_kernels_change(gpu, columns, dim):
    """Rows that see all blocks and rows that see some, scores full of ties, scales that are NaN: one list each."""
    rng = np.random.default_rng(columns + dim)
    rows, count = 37, 50
    q = rng.integers(-127, 128, (1, 3, rows, dim)).astype(np.int8)
    k = rng.integers(-127, 128, (1, 3, columns, dim)).astype(np.int8)
    s = rng.uniform(0.001, 0.1, (1, 3, columns)).astype(np.float32)
    q[0, 1], k[0, 1], s[0, 1] = rng.integers(-1, 2, q[0, 1].shape), rng.integers(-1, 2, k[0, 1].shape), np.float32(0.01)
    s[0, 2, rng.random(columns) < 0.97] = np.nan
    t = [torch.from_numpy(x) for x in (q, k, s)]
    for causal in (False, True):  # causal: the rows see from columns - 36 * m / n blocks to all of them
        m = max(1, columns // 50)
        queries = rows * m
        pos, crd = run_select(gpu, *t, count, queries, columns, m, 1, causal, 2, 3)
        at = 0
        for h in range(3):
            for r in range(rows):
                seen = min(max((r + 1) * m + columns - queries, 0), columns) if causal else columns
                want = reference(q[0, h, r], k[0, h], s[0, h], count, seen, 2, 3)
                assert pos[h * rows + r] == at
                assert crd[at:at + len(want)].tolist() == want, (causal, h, r)
                at += len(want)
        assert pos[-1] == at and bool((crd[at:] == -9).all())


def test_selection_over_a_wide_table(gpu):
    """1500 pages to a sequence, some of which do not exist; lengths that reach every one of the kernels' widths."""
    rng = np.random.default_rng(9)
    pages, heads, dim, width, count = 4000, 2, 128, 1500, 40
    blocks = np.array([1500, 1025, 41, 40, 700, 2000], dtype=np.int32)
    table = rng.integers(0, pages, (6, width)).astype(np.int32)
    table[rng.random(table.shape) < 0.01] = -1
    table[rng.random(table.shape) < 0.01] = pages
    q = rng.integers(-127, 128, (6, heads, 1, dim)).astype(np.int8)
    k = rng.integers(-127, 128, (pages, heads, dim)).astype(np.int8)
    s = rng.uniform(0, 1, (pages, heads)).astype(np.float32)
    pos = torch.full((6 * heads + 1,), -9, dtype=torch.int32, device="cuda")
    crd = torch.full((6 * heads * count,), -9, dtype=torch.int32, device="cuda")
    gpu.block_select(*(torch.from_numpy(x).cuda() for x in (q, k, s)), count, pos, crd, queries=1, keys=width, block_m=1, block_n=1,
                     causal=False, sink=1, local=2, table=torch.from_numpy(table).cuda(), blocks=torch.from_numpy(blocks).cuda())
    pos, crd = pos.cpu().numpy(), crd.cpu().numpy()
    at = 0
    for b in range(6):
        for h in range(heads):
            seen = min(max(int(blocks[b]), 0), width)
            page = np.clip(table[b], 0, pages - 1)
            scale = np.where((table[b] >= 0) & (table[b] < pages), s[page, h], np.nan).astype(np.float32)
            want = reference(q[b, h, 0], k[page, h], scale, count, seen, 1, 2)
            assert pos[b * heads + h] == at
            assert crd[at:at + len(want)].tolist() == [int(table[b, j]) for j in want], (b, h)
            at += len(want)
    assert pos[-1] == at


def test_pool_of_more_parts_of_blocks_than_31_bits(gpu):
    """2^28 blocks and some, eight groups of lanes to each: one row of values, given 2^29 times over by a stride of 0."""
    blocks = (1 << 28) + 3
    x = torch.arange(1, 9, dtype=torch.bfloat16, device="cuda")
    codes = torch.full((1, 1, blocks, 8), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((1, 1, blocks), 7.0, device="cuda")
    gpu.block_pool(x.view(1, 1, 1, 8).expand(1, 2 * blocks, 1, 8), 2, codes, scales)
    torch.cuda.synchronize()
    want = torch.tensor([16, 32, 48, 64, 79, 95, 111, 127], dtype=torch.int8, device="cuda")  # 127 n / 8: 63.5 is a tie, to even
    assert bool((codes == want).all()) and bool((scales == torch.tensor(8.0) / 127.0).all())
