"""Attention's entries with operands on a device that is not the current one: its streams are not where their work would run."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")]


def test_operands_on_another_device_are_refused(gpu):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype, device="cuda:1")  # noqa: E731
    i = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    x, cache, lse, freq = z(1, 32, 2, 64), z(4, 2, 16, 64), z(1, 2, 32, dtype=torch.float32), z(1, 32, dtype=torch.float64)
    rows, codes, scales = z(3, 2, 64), z(1, 2, 2, 64, dtype=torch.int8), z(1, 2, 2, dtype=torch.float32)
    pos, crd = i(5), i(0)
    calls = [
        lambda: gpu.kv_store(rows, rows, i(3), cache, cache.clone()), lambda: gpu.kv_load(cache, cache, i(3), rows, rows.clone()),
        lambda: gpu.kv_append(rows, rows, i(1, 3), freq, i(3), cache, cache.clone()), lambda: gpu.rotate(x, i(1, 1, 32), freq, x),
        lambda: gpu.paged_attention(rows, cache, cache, i(4), crd, i(3), rows.clone()),
        lambda: gpu.paged_window_attention(rows, cache, cache, i(3, 1), i(3), rows.clone(), 4), lambda: gpu.block_pool(x, 16, codes, scales),
        lambda: gpu.block_select(codes, codes, scales, 1, pos, i(4), 32, 32, 16, 16, True, 0, 1),
        lambda: gpu.block_attention(x, x, x, pos, crd, x.clone(), lse, 16, 16), lambda: gpu.window_attention(x, x, x, x.clone(), 4, 0, lse),
        lambda: gpu.block_attention_backward(x, x, x, x, x, lse, pos, crd, x.clone(), x.clone(), x.clone(), 16, 16),
        lambda: gpu.window_attention_backward(x, x, x, x, x, lse, x.clone(), x.clone(), x.clone(), 4)]
    with torch.cuda.device(0):
        for call in calls:
            with pytest.raises(ValueError, match="on device 1, the current one is 0"):
                call()
