"""Attention over a window at the edges of its gradient's layout: columns of their own workgroups, first keys of several columns, strides."""
import pytest
import torch

import attention_ref as ref
from test_gpu_window_attention import backward, forward, inputs, mask_of

pytestmark = pytest.mark.gpu


def check(gpu, q, k, v, dout, window, sink):
    w, scale = mask_of(q.shape[0], k.shape[2], q.shape[1], k.shape[1], window, sink), q.shape[3] ** -0.5
    out, lse = forward(gpu, q, k, v, window, sink)
    want, want_lse, bound, lse_bound = ref.forward(q, k, v, w, scale)
    ref.assert_within(out, want, bound, "out")
    ref.assert_within(lse, want_lse, lse_bound, "lse")
    grads = backward(gpu, dout, q, k, v, out, lse, window, sink)
    for name, got, x, b in zip(("dq", "dk", "dv"), grads, *ref.backward(dout, q, k, v, out, lse, w, scale)):
        ref.assert_within(got, x, b, name)


@pytest.mark.parametrize("batch,queries,keys,heads,kv_heads,dim,window,sink,dtype", [
    (1, 600, 700, 6, 6, 64, 90, 300, "bf16"), (2, 500, 500, 3, 3, 128, 200, 129, "f16"), (1, 900, 1000, 4, 4, 72, 256, 128, "bf16"),
    (2, 1100, 1100, 4, 2, 64, 50, 257, "bf16"), (1, 2300, 2300, 9, 9, 64, 128, 1, "f16"), (1, 1, 900, 8, 8, 64, 1, 700, "bf16"),
    (1, 700, 300, 5, 5, 96, 100, 150, "bf16")])
def test_columns_that_are_one_workgroups(gpu, batch, queries, keys, heads, kv_heads, dim, window, sink, dtype):
    q, k, v = inputs(batch, queries, keys, heads, kv_heads, dim, dtype)
    check(gpu, q, k, v, inputs(batch, queries, keys, heads, kv_heads, dim, dtype, seed=3)[0], window, sink)


@pytest.mark.parametrize("batch,queries,keys,heads,kv_heads,dim,window,sink", [
    (1, 1100, 1100, 16, 16, 64, 1100, 0), (1, 1000, 2050, 32, 8, 128, 700, 33), (2, 1100, 1100, 8, 8, 96, 65, 64), (1, 520, 4000, 32, 2, 64, 3000, 16)])
def test_two_sides_of_a_workgroup(gpu, batch, queries, keys, heads, kv_heads, dim, window, sink):
    """128 to 256 workgroups of 128 rows, whose two halves share the keys: odd and even numbers of tiles, one side with nothing to see."""
    q, k, v = inputs(batch, queries, keys, heads, kv_heads, dim, "bf16")
    v = v.clone()
    v[0, 5, 0, 3], v[0, keys - 3, -1, 5] = float("inf"), float("nan")
    w, scale = mask_of(batch, kv_heads, queries, keys, window, sink), dim ** -0.5
    out, lse = forward(gpu, q, k, v, window, sink)
    want, want_lse, bound, lse_bound = ref.forward(q, k, v, w, scale)
    # who sees the infinity or the NaN has it, nobody else
    seen = torch.zeros(want.shape, dtype=torch.bool)
    group = heads // kv_heads
    seen[0, :, :group, 3] = w[0, 0, :, 5][:, None] > 0
    seen[0, :, -group:, 5] |= w[0, 0, :, keys - 3][:, None] > 0
    assert torch.equal(~torch.isfinite(out.cpu()), seen)
    ref.assert_within(torch.where(seen.cuda(), 0.0, out), torch.where(seen, 0.0, want), torch.where(seen, 1.0, bound), "out")
    ref.assert_within(lse, want_lse, lse_bound, "lse")


def strided(x, token, head):
    """The same elements, tokens and heads these many elements apart."""
    _, tokens, heads, dim = x.shape
    memory = torch.empty((tokens - 1) * token + (heads - 1) * head + dim, dtype=x.dtype, device="cuda")
    return memory.as_strided(x.shape, (0, token, head, 1)).copy_(x)


def test_heads_that_lie_far_apart(gpu):
    """64 heads of a group 2^25 - 8 elements apart: the last row of a tile is almost 2^32 bytes from the first."""
    q, k, v = inputs(1, 40, 70, 64, 1, 64, "bf16")
    dout = strided(inputs(1, 40, 70, 64, 1, 64, "bf16", seed=3)[0], 64, 2 ** 25 - 8)
    check(gpu, strided(q, 64, 2 ** 25 - 8), k, v, dout, 30, 3)


@pytest.mark.parametrize("heads,token,head,match", [(66, 2 ** 25 - 8, 2 ** 25 - 8, "66 heads of a group"), (200, 64, 2 ** 25 - 8, "200 heads"), (2, 64, 2 ** 25, "a stride of 33554432"), (2, 2 ** 25, 64, "a stride of 33554432")])
def test_strides_that_are_refused(gpu, heads, token, head, match):
    """By the gradient; the forward call takes them.  (Memory that nobody writes.)"""
    q = torch.empty(3 * token + (heads - 1) * head + 64, dtype=torch.bfloat16, device="cuda").as_strided((1, 4, heads, 64), (0, token, head, 1))
    k = torch.zeros((1, 9, 1, 64), dtype=torch.bfloat16, device="cuda")
    rows, lse = torch.zeros((1, 4, heads, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, heads, 4), device="cuda")
    for args in ((rows, q), (q, rows)):
        with pytest.raises(gpu.LapisHipError, match=match):
            gpu.window_attention_backward(*args, k, k, rows, lse, torch.empty_like(rows), torch.empty_like(k), torch.empty_like(k), 3)


def test_too_many_rows_are_refused(gpu):
    """2^29 queries times heads of a group, all of them the same memory."""
    q = torch.zeros((1, 1, 1, 8), dtype=torch.bfloat16, device="cuda").expand(1, 2 ** 23, 64, 8)
    k = torch.zeros((1, 9, 1, 8), dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((1, 64, 2 ** 23), device="cuda")
    dq = torch.empty((1, 2 ** 23, 64, 8), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(gpu.LapisHipError, match="8388608 queries of 64 heads"):
        gpu.window_attention_backward(q, q, k, k, q, lse, dq, torch.empty_like(k), torch.empty_like(k), 3)
