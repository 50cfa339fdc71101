"""The attention layer's window with queries whose tokens or heads lie further apart than the gradient's kernel takes: they are copied for it."""
import pytest
import torch

from test_gpu_window_limits import strided

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,token,head", [(2, 64, 2 ** 25), (2, 2 ** 25, 64), (1, 2 ** 25, 64), (66, 2 ** 25 - 8, 2 ** 25 - 8), (200, 64, 2 ** 25 - 8), (64, 64, 2 ** 25 - 8), (3, 192, 64)])
def test_gradient_of_queries_far_apart(gpu, heads, token, head):
    from lapis_amd import attention

    g = torch.Generator().manual_seed(heads)
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    q, k, v, dout = r(1, 4, heads, 64), r(1, 9, 1, 64), r(1, 9, 1, 64), r(1, 4, heads, 64)
    far = strided(q, token, head)  # (where both strides are the same, a token's heads are the next one's too: what far holds is not what q does)
    assert (far.stride(1), far.stride(2)) == (token, head)
    results = []
    for x in (far.contiguous(), far):
        leaves = [t.detach().requires_grad_() for t in (x, k, v)]
        out = attention.attend_window(*leaves, 3, 1)
        results.append((out, *torch.autograd.grad(out, leaves, dout)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
