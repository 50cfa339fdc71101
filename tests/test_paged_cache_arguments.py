"""What a cache refuses, and how it lies in memory, without a GPU."""
import pytest
import torch

from lapis_amd import attention


def make(**more):
    return attention.PagedCache(2, 6, 96, 3, 64, page=16, device="cpu", **more)


def test_formats():
    for more, kept, scales in (({}, torch.bfloat16, None), ({"f8": True}, torch.float8_e4m3fn, ((6, 3, 16), torch.float32)), ({"f4": True}, torch.uint8, ((6, 3, 16, 2), torch.uint8)),
                               ({"dtype": torch.float16}, torch.float16, None)):
        cache = make(**more)
        for x, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            assert x.shape == (6, 3, 16, 32 if "f4" in more else 64) and x.dtype == kept
            assert (scale is None) == (scales is None)
            assert scales is None or (scale.shape, scale.dtype) == (torch.Size(scales[0]), scales[1])


def test_refusals():
    with pytest.raises(ValueError, match="codes of 8 bits and of 4 bits"):
        make(f8=True, f4=True)
    with pytest.raises(ValueError, match="rows of 72 elements"):
        attention.PagedCache(2, 6, 96, 3, 72, page=16, device="cpu", f4=True)
    cache = make()
    q, k, positions = torch.zeros((2, 3, 64), dtype=torch.bfloat16), torch.zeros((2, 3, 64), dtype=torch.bfloat16), torch.zeros((1, 2), dtype=torch.int32)
    for call in (lambda: cache.prefill(0, k, k, positions=positions), lambda: cache.step(q, k, k, 3, positions=positions),
                 lambda: cache.step_window(q, k, k, 3, positions=positions)):
        with pytest.raises(ValueError, match="positions, and no frequencies"):
            call()
    assert len(cache.free) == 6 and cache.lengths == [0, 0]
