"""Sequences longer than their row of the table: the window is the last tokens of the sequence, and those beyond the table do not exist."""
import pytest
import torch

from test_gpu_window_cache import TYPES, check_row, rows_of_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["same", "f8", "f4"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,width,window,sink,dtype", [
    (4, 2, 64, 16, 4, 50, 0, "bf16"), (4, 2, 64, 16, 4, 50, 9, "f16"), (8, 1, 128, 64, 30, 700, 33, "bf16"), (2, 2, 32, 1, 5, 3, 2, "bf16"), (6, 3, 96, 32, 1, 1, 100, "f16")])
def test_window_of_a_sequence_longer_than_its_table(gpu, heads, kv_heads, dim, page, width, window, sink, dtype, kind):
    held = width * page  # tokens that a table's row has
    lengths = [held - 1, held, held + 1, held + window // 2, held + window - 1, held + window, held + window + 1, 2 ** 31 - 1]
    g = torch.Generator().manual_seed(dim + held)
    pages = len(lengths) * width
    (kc, vc), (ks, vs), values = rows_of_cache(kind, TYPES[dtype], pages, kv_heads, page, dim, g)
    table = torch.randperm(pages, generator=g).to(torch.int32).reshape(len(lengths), width)
    q = torch.randn((len(lengths), heads, dim), generator=g).to(TYPES[dtype])
    out, lse = torch.full_like(q, 9.0).cuda(), torch.full((len(lengths), heads), 9.0, device="cuda")
    gpu.paged_window_attention(q.cuda(), kc, vc, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), out, window, sink, lse=lse, k_scale=ks, v_scale=vs)
    for s, n in enumerate(lengths):
        t = torch.tensor([t for t in range(min(n, held)) if t >= n - window or t < sink], dtype=torch.long)
        k, v = (x[table[s, t // page].long(), :, t % page] for x in values)
        check_row(out[s], lse[s], q[s], k, v, dim ** -0.5, "%d tokens, %d in the table" % (n, held))


@pytest.mark.parametrize("kind", ["same", "f4"])
def test_a_table_far_wider_than_its_sequences(gpu, kind):
    """Scratch memory stays with what a sequence may spread over, not with what its table could name; and the longer units of such a table."""
    page, width, kv_heads, dim, lengths = 64, 2 ** 14, 8, 64, [3, 20000, 0, 700, 8192, 64, 9000, 1]
    g = torch.Generator().manual_seed(5)
    held = [-(-n // page) for n in lengths]
    (kc, vc), (ks, vs), values = rows_of_cache(kind, torch.bfloat16, sum(held), kv_heads, page, dim, g)
    table, order, at = torch.full((len(lengths), width), -1, dtype=torch.int32), torch.randperm(sum(held), generator=g).to(torch.int32), 0
    for s, n in enumerate(held):
        table[s, :n] = order[at:at + n]
        at += n
    q = torch.randn((len(lengths), 16, dim), generator=g).to(torch.bfloat16)
    out, lse = torch.full_like(q, 9.0).cuda(), torch.full((len(lengths), 16), 9.0, device="cuda")
    operands = q.cuda(), kc, vc, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), out, 2 ** 30
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    gpu.paged_window_attention(*operands, lse=lse, k_scale=ks, v_scale=vs)
    scratch = torch.cuda.max_memory_allocated() - before
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    # a unit more for each head where the tokens do not divide, units cut to multiples of 32 tokens, and the allocator's own rounding up
    assert scratch <= len(lengths) * (4 * cus * 1.04 + kv_heads) * 64 * (dim + 2) + 2 ** 21
    for s, n in enumerate(lengths):
        t = torch.arange(n)
        k, v = (x[table[s, t // page].long(), :, t % page] for x in values)
        check_row(out[s], lse[s], q[s], k, v, dim ** -0.5, "%d tokens" % n)
