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
