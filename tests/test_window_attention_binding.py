"""What the Python entries of rotated positions, the 4-bit cache and windows refuse: no GPU needed."""
import ctypes

import pytest
import torch

from lapis_amd import hip

B, F, H, D, U8 = torch.bfloat16, torch.float32, torch.float16, torch.float64, torch.uint8


def z(*shape, dtype=B):
    return torch.zeros(shape, dtype=dtype)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def rotate(**change):
    a = dict(x=z(2, 5, 4, 64), positions=i32(1, 2, 5), frequencies=z(1, 32, dtype=D), out=z(2, 5, 4, 64))
    a.update(change)
    return hip.rotate(**a)


def append(**change):
    a = dict(k=z(3, 2, 64), v=z(3, 2, 64), positions=i32(1, 3), frequencies=z(1, 32, dtype=D), slots=i32(3), k_cache=z(4, 2, 16, 64), v_cache=z(4, 2, 16, 64))
    a.update(change)
    return hip.kv_append(**a)


def step(**change):
    a = dict(q=z(3, 4, 64), k_cache=z(4, 2, 16, 64), v_cache=z(4, 2, 16, 64), table=i32(3, 2), lengths=i32(3), out=z(3, 4, 64), window=8)
    a.update(change)
    return hip.paged_window_attention(**a)


def window(**change):
    a = dict(q=z(1, 32, 4, 64), k=z(1, 32, 2, 64), v=z(1, 32, 2, 64), out=z(1, 32, 4, 64), window=8, sink=2, lse=z(1, 4, 32, dtype=F))
    a.update(change)
    return hip.window_attention(**a)


def gradient(**change):
    a = dict(dout=z(1, 32, 4, 64), q=z(1, 32, 4, 64), k=z(1, 32, 2, 64), v=z(1, 32, 2, 64), out=z(1, 32, 4, 64), lse=z(1, 4, 32, dtype=F), dq=z(1, 32, 4, 64),
             dk=z(1, 32, 2, 64), dv=z(1, 32, 2, 64), window=8)
    a.update(change)
    return hip.window_attention_backward(**a)


F4 = dict(k_cache=z(4, 2, 16, 32, dtype=U8), v_cache=z(4, 2, 16, 32, dtype=U8), k_scale=z(4, 2, 16, 2, dtype=U8), v_scale=z(4, 2, 16, 2, dtype=U8))


def f4(**change):
    return dict(F4, **change)


@pytest.mark.parametrize("call,change", [
    (rotate, dict(x=z(2, 5, 4, 64, dtype=F))), (rotate, dict(out=z(2, 5, 4, 64, dtype=H))), (rotate, dict(positions=torch.zeros((1, 2, 5), dtype=torch.int64))),
    (rotate, dict(frequencies=z(1, 32, dtype=F))), (append, dict(k=z(3, 2, 64, dtype=H))), (append, dict(q=z(3, 4, 64))), (append, dict(q_out=z(3, 4, 64))),
    (append, dict(q=z(3, 4, 64, dtype=H), q_out=z(3, 4, 64, dtype=H))), (append, dict(k_cache=z(4, 2, 16, 64, dtype=H), v_cache=z(4, 2, 16, 64, dtype=H))),
    (append, f4(k_scale=None)), (append, f4(k_scale=z(4, 2, 16, 2, dtype=F))), (step, dict(q=z(3, 4, 64, dtype=H))), (step, dict(table=z(3, 2))),
    (step, dict(lengths=torch.zeros(3, dtype=torch.int64))), (step, dict(lse=z(3, 4))), (step, dict(window="8")), (step, dict(window=8.5)),
    (window, dict(k=z(1, 32, 2, 64, dtype=H))), (window, dict(q=z(1, 32, 4, 64, dtype=F))), (window, dict(lse=z(1, 4, 32))), (window, dict(sink=None)),
    (gradient, dict(lse=None)), (gradient, dict(dq=z(1, 32, 4, 64, dtype=H)))])
def test_types(call, change):
    with pytest.raises(TypeError):
        call(**change)


@pytest.mark.parametrize("call,change", [
    (rotate, dict(out=z(2, 5, 4, 32))), (rotate, dict(x=z(2, 5, 64))), (rotate, dict(positions=i32(1, 2, 4))), (rotate, dict(positions=i32(2, 2, 5))),
    (rotate, dict(frequencies=z(32, 1, dtype=D).T.expand(1, 32)[:, ::2])), (rotate, dict(out=z(2, 5, 1, 64).expand(2, 5, 4, 64))),
    (rotate, dict(x=z(2, 5, 4, 128)[..., ::2])), (append, dict(v=z(2, 2, 64))), (append, dict(positions=i32(1, 2))), (append, dict(slots=i32(2))),
    (append, dict(q=z(3, 4, 64), q_out=z(3, 5, 64))), (append, dict(k_scale=z(4, 2, 16, dtype=F), v_scale=z(4, 2, 16, dtype=F))),
    (append, f4(k_cache=z(4, 2, 16, 16, dtype=U8), v_cache=z(4, 2, 16, 16, dtype=U8))), (append, f4(k_scale=z(4, 2, 16, 1, dtype=U8))),
    (append, f4(v_scale=z(4, 16, 2, 2, dtype=U8).transpose(1, 2))), (append, f4(k_scale=z(4, 2, 16, 4, dtype=U8)[..., ::2])),
    (append, f4(k_cache=z(4, 2, 16, 24, dtype=U8), v_cache=z(4, 2, 16, 24, dtype=U8))), (append, f4(k_cache=z(4, 2, 1, 32, dtype=U8).expand(4, 2, 16, 32))),
    (step, dict(table=i32(2, 2))), (step, dict(lengths=i32(4))), (step, dict(out=z(3, 4, 32))), (step, dict(window=0)), (step, dict(window=-1)), (step, dict(sink=-1)),
    (step, dict(table=i32(3, 4)[:, ::2])), (step, dict(lse=z(4, 3, dtype=F))), (step, dict(out=z(1, 4, 64).expand(3, 4, 64))),
    (window, dict(window=0)), (window, dict(sink=-1)), (window, dict(k=z(1, 31, 2, 64))), (window, dict(k=z(1, 32, 3, 64), v=z(1, 32, 3, 64))),
    (window, dict(out=z(1, 32, 4, 32))), (window, dict(lse=z(1, 32, 4, dtype=F))), (window, dict(k=z(1, 32, 0, 64), v=z(1, 32, 0, 64))),
    (gradient, dict(dk=z(1, 32, 4, 64))), (gradient, dict(dout=z(1, 31, 4, 64))), (gradient, dict(dv=z(1, 1, 2, 64).expand(1, 32, 2, 64))), (gradient, dict(window=0))])
def test_shapes(call, change):
    with pytest.raises(ValueError):
        call(**change)


def test_output_over_its_input_in_another_order():
    x = z(4, 4, 4, 64)
    with pytest.raises(ValueError, match="another order"):
        hip.rotate(x, i32(1, 4, 4), z(1, 32, dtype=D), x.transpose(1, 2))


@pytest.mark.parametrize("call", [rotate, append, step, window, gradient])
def test_operands_in_host_memory(call):
    with pytest.raises(ValueError, match="not in device memory"):
        call()


@pytest.mark.parametrize("call", [append, step])
def test_a_4_bit_cache_in_host_memory(call):
    with pytest.raises(ValueError, match="not in device memory"):
        call(**F4)


def test_calls_before_init():
    lib = hip.load()
    for name, n in (("lapis_hip_kv_append", 3), ("lapis_hip_paged_window_attention", 3), ("lapis_hip_window_attention", 2), ("lapis_hip_window_attention_backward", 2)):
        assert lib.lapis_hip_status_name(getattr(lib, name)(*[None] * n)) == b"LAPIS_HIP_ERR_NOT_INITIALIZED", name
    rc = lib.lapis_hip_rotate(0, 0, 0, 64, None, 0, None, None, 0, None)
    assert lib.lapis_hip_status_name(rc) == b"LAPIS_HIP_ERR_NOT_INITIALIZED"
    for name, n in (("lapis_hip_paged_window_attention_work", 2), ("lapis_hip_window_attention_backward_work", 1)):
        assert lib.lapis_hip_status_name(getattr(lib, name)(*[None] * n, ctypes.byref(ctypes.c_int64()))) == b"LAPIS_HIP_ERR_NOT_INITIALIZED", name
