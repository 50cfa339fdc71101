"""Enough rows that a thread takes four of them, with heads that are a wavefront's together and heads that are not."""
import pytest
import torch

from test_gpu_rotate import frequencies, test_append as check_append, test_rotate as check_rotate

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,tokens,heads,dim,pairs,axes,neighbours,dtype", [
    (1, 16411, 8, 64, 32, 1, False, "bf16"), (2, 6001, 12, 64, 24, 2, True, "f16"), (3, 2801, 8, 128, 64, 3, False, "bf16"), (1, 22003, 3, 104, 52, 1, False, "f16"),
    (1, 4200, 16, 256, 128, 1, False, "bf16"), (2, 5600, 3, 200, 100, 1, True, "bf16"), (1, 66000, 1, 128, 64, 1, False, "bf16"), (1, 8300, 8, 96, 44, 2, False, "f16")])
@pytest.mark.parametrize("inverse", [False, True], ids=["forward", "inverse"])
def test_rotate_of_many_rows(gpu, batch, tokens, heads, dim, pairs, axes, neighbours, dtype, inverse):
    check_rotate(gpu, batch, tokens, heads, dim, pairs, axes, neighbours, dtype, inverse)


@pytest.mark.parametrize("kind", ["same", "f8", "f4"])
@pytest.mark.parametrize("tokens,q_heads,heads,dim,pairs,axes,neighbours,page,dtype,token_major", [
    (4111, 8, 4, 128, 64, 1, False, 64, "bf16", False), (4099, 14, 1, 128, 48, 2, True, 32, "f16", True), (8203, 8, 8, 64, 32, 3, False, 128, "bf16", False),
    (3001, 5, 3, 256, 128, 1, False, 16, "bf16", True), (2803, 8, 2, 160, 72, 1, False, 64, "f16", False)])
def test_append_of_many_rows(gpu, tokens, q_heads, heads, dim, pairs, axes, neighbours, page, dtype, token_major, kind):
    check_append(gpu, tokens, q_heads, heads, dim, pairs, axes, neighbours, page, dtype, token_major, kind)


@pytest.mark.parametrize("heads", [8, 3])
def test_one_head_for_all(gpu, heads):
    """A broadcast head and positions, out with gaps between its rows, which stay."""
    g = torch.Generator().manual_seed(heads)
    x = torch.randn((1, 24000, 1, 128), generator=g).bfloat16().cuda().expand(1, 24000, heads, 128)
    positions = torch.randint(0, 1000, (24000,), generator=g, dtype=torch.int32).cuda().expand(2, 1, 24000)
    freq = frequencies(2, 64, g).cuda()
    memory = torch.full((1, 24000, heads + 1, 136), 3.0, dtype=torch.bfloat16, device="cuda")
    gpu.rotate(x, positions, freq, memory[:, :, :heads, :128])
    by_itself = torch.empty((1, 24000, 1, 128), dtype=torch.bfloat16, device="cuda")
    gpu.rotate(x[:, :, :1].contiguous(), positions, freq, by_itself)
    assert torch.equal(memory[:, :, :heads, :128], by_itself.expand_as(x))
    assert bool((memory[:, :, heads] == 3).all() and (memory[..., 128:] == 3).all())
