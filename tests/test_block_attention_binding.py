"""What the Python entries of block-sparse attention refuse, and the entries' answer before lapis_hip_init: no GPU needed."""
import ctypes

import pytest
import torch

from lapis_amd import hip

B, F, H, I8 = torch.bfloat16, torch.float32, torch.float16, torch.int8
F8 = torch.float8_e4m3fn


def z(*shape, dtype=B):
    return torch.zeros(shape, dtype=dtype)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def attention(**change):
    a = dict(q=z(1, 32, 4, 64), k=z(1, 32, 2, 64), v=z(1, 32, 2, 64), pos=i32(0, 0, 0), crd=i32(), out=z(1, 32, 4, 64), lse=z(1, 4, 32, dtype=F),
             block_m=32, block_n=32)
    a.update(change)
    return hip.block_attention(**a)


def gradient(**change):
    a = dict(dout=z(1, 32, 4, 64), q=z(1, 32, 4, 64), k=z(1, 32, 2, 64), v=z(1, 32, 2, 64), out=z(1, 32, 4, 64), lse=z(1, 4, 32, dtype=F),
             pos=i32(0, 0, 0), crd=i32(), dq=z(1, 32, 4, 64), dk=z(1, 32, 2, 64), dv=z(1, 32, 2, 64), block_m=32, block_n=32)
    a.update(change)
    return hip.block_attention_backward(**a)


def store(**change):
    a = dict(k=z(3, 2, 64), v=z(3, 2, 64), slots=i32(0, 1, 2), k_cache=z(4, 2, 16, 64), v_cache=z(4, 2, 16, 64))
    a.update(change)
    return hip.kv_store(**a)


def load(**change):
    a = dict(k_cache=z(4, 2, 16, 64), v_cache=z(4, 2, 16, 64), slots=i32(0, 1, 2), k=z(3, 2, 64), v=z(3, 2, 64))
    a.update(change)
    return hip.kv_load(**a)


def paged(**change):
    a = dict(q=z(3, 4, 64), k_cache=z(4, 2, 16, 64), v_cache=z(4, 2, 16, 64), pos=i32(0, 0, 0, 0), crd=i32(), tokens=i32(0, 0, 0), out=z(3, 4, 64))
    a.update(change)
    return hip.paged_attention(**a)


def pool(**change):
    a = dict(x=z(1, 32, 4, 64), block=16, codes=z(1, 2, 2, 64, dtype=I8), scales=z(1, 2, 2, dtype=F))
    a.update(change)
    return hip.block_pool(**a)


def select(**change):
    a = dict(q_codes=z(1, 2, 2, 64, dtype=I8), k_codes=z(1, 2, 4, 64, dtype=I8), k_scales=z(1, 2, 4, dtype=F), count=2, pos=i32(0, 0, 0, 0, 0),
             crd=i32(*[0] * 8), queries=32, keys=64, block_m=16, block_n=16)
    a.update(change)
    return hip.block_select(**a)


SCALES = z(4, 2, 16, dtype=F)

WRONG_SHAPE = [
    (attention, dict(k=z(1, 32, 3, 64), v=z(1, 32, 3, 64))), (attention, dict(v=z(1, 31, 2, 64))), (attention, dict(q=z(32, 4, 64))),
    (attention, dict(out=z(1, 32, 4, 32))), (attention, dict(lse=z(1, 32, 4, dtype=F))), (attention, dict(pos=i32(0, 0))),
    (attention, dict(block_m=0)), (attention, dict(block_n=0)), (attention, dict(k=z(2, 32, 2, 64), v=z(2, 32, 2, 64))),
    (attention, dict(out=z(1, 32, 1, 64).expand(1, 32, 4, 64))), (attention, dict(q=z(1, 32, 4, 128)[..., ::2])), (attention, dict(crd=i32(0, 1, 2, 3)[::2])),
    (attention, dict(k=z(1, 32, 0, 64), v=z(1, 32, 0, 64))),
    (gradient, dict(dout=z(1, 32, 2, 64))), (gradient, dict(dk=z(1, 32, 4, 64))), (gradient, dict(dq=z(1, 1, 4, 64).expand(1, 32, 4, 64))),
    (gradient, dict(lse=z(1, 4, 31, dtype=F))),
    (store, dict(k=z(3, 1, 64))), (store, dict(v=z(3, 2, 32))), (store, dict(slots=i32(0, 1))), (store, dict(v_cache=z(4, 2, 32, 64))),
    (store, dict(k_cache=z(4, 2, 16, 64, dtype=F8), v_cache=z(4, 2, 16, 64, dtype=F8), k_scale=SCALES, v_scale=z(4, 2, 15, dtype=F))),
    (store, dict(k_scale=SCALES, v_scale=SCALES)), (store, dict(k_cache=z(4, 2, 1, 64).expand(4, 2, 16, 64))),
    (store, dict(v_cache=z(4, 16, 2, 64).transpose(1, 2))), (load, dict(k=z(2, 2, 64))), (load, dict(k=z(1, 2, 64).expand(3, 2, 64))),
    (paged, dict(tokens=i32(0, 0), pos=i32(0, 0, 0))), (paged, dict(pos=i32(0, 0, 0))), (paged, dict(out=z(3, 2, 64))), (paged, dict(q=z(3, 4, 32))),
    (paged, dict(lse=z(4, 3, dtype=F))),
    (pool, dict(codes=z(1, 3, 2, 64, dtype=I8), scales=z(1, 3, 2, dtype=F))), (pool, dict(codes=z(1, 2, 3, 64, dtype=I8))), (pool, dict(block=0)),
    (pool, dict(scales=z(1, 2, 1, dtype=F))),
    (select, dict(k_codes=z(1, 2, 5, 64, dtype=I8))), (select, dict(q_codes=z(1, 2, 3, 64, dtype=I8))), (select, dict(block_m=0)),
    (select, dict(table=z(1, 4, dtype=torch.int32))), (select, dict(blocks=i32(1, 1))), (select, dict(queries=-1)),
]
WRONG_TYPE = [
    (attention, dict(q=z(1, 32, 4, 64, dtype=F))), (attention, dict(k=z(1, 32, 2, 64, dtype=H))), (attention, dict(pos=torch.zeros(3, dtype=torch.int64))),
    (attention, dict(lse=z(1, 4, 32))), (attention, dict(out=z(1, 32, 4, 64, dtype=F))), (attention, dict(q=5)), (attention, dict(crd=None)),
    (gradient, dict(dv=z(1, 32, 2, 64, dtype=H))), (gradient, dict(lse=None)),
    (store, dict(k_cache=z(4, 2, 16, 64, dtype=H), v_cache=z(4, 2, 16, 64, dtype=H))), (store, dict(slots=torch.zeros(3, dtype=torch.int64))),
    (store, dict(k_cache=z(4, 2, 16, 64, dtype=F8), v_cache=z(4, 2, 16, 64, dtype=F8))),
    (store, dict(k_cache=z(4, 2, 16, 64, dtype=F8))), (load, dict(k=z(3, 2, 64, dtype=F))),
    (paged, dict(q=z(3, 4, 64, dtype=H))), (paged, dict(crd=torch.zeros(0, dtype=torch.int64))), (paged, dict(lse=z(3, 4))),
    (pool, dict(x=z(1, 32, 4, 64, dtype=F))), (pool, dict(codes=z(1, 2, 2, 64, dtype=torch.uint8))), (pool, dict(scales=z(1, 2, 2))),
    (select, dict(k_scales=z(1, 2, 4))), (select, dict(pos=torch.zeros(5, dtype=torch.int64))),
]


@pytest.mark.parametrize("call,change", WRONG_SHAPE)
def test_shapes_strides_and_sizes(call, change):
    with pytest.raises(ValueError):
        call(**change)


@pytest.mark.parametrize("call,change", WRONG_TYPE)
def test_types(call, change):
    with pytest.raises(TypeError):
        call(**change)


@pytest.mark.parametrize("call", [attention, gradient, store, load, paged, pool, select])
def test_tensors_in_host_memory(call):
    with pytest.raises(ValueError, match="not in device memory"):
        call()


def test_calls_before_init_report_not_initialized():
    lib = hip.load()
    if hip._initialized:
        pytest.skip("another test has initialised the library")
    buffer = ctypes.create_string_buffer(1024)
    for rc in (lib.lapis_hip_kv_store(buffer, 0, buffer, buffer, 0, None, None), lib.lapis_hip_paged_attention(buffer, buffer, None),
               lib.lapis_hip_block_pool(1, 1, 1, 1, 8, 1, buffer, 0, None, None, None), lib.lapis_hip_block_select(buffer, None),
               lib.lapis_hip_block_attention(buffer, None), lib.lapis_hip_block_attention_backward(buffer, None)):
        assert lib.lapis_hip_status_name(rc) == b"LAPIS_HIP_ERR_NOT_INITIALIZED"


class SelectArgs(ctypes.Structure):
    """lapis_hip_select_args"""
    _fields_ = ([(n, ctypes.c_int64) for n in ("batch", "heads", "queries", "keys", "dim", "block_m", "block_n", "count", "sink", "local")] +
                [("causal", ctypes.c_int)] + [(n, ctypes.c_void_p) for n in ("q_codes", "k_codes", "k_scales")] +
                [("k_stride", ctypes.c_int64 * 3), ("scale_stride", ctypes.c_int64 * 3), ("table", ctypes.c_void_p), ("blocks", ctypes.c_void_p),
                 ("table_width", ctypes.c_int64), ("pages", ctypes.c_int64)] + [(n, ctypes.c_void_p) for n in ("pos", "crd", "work")])


def test_entries_of_a_selection_are_counted_without_a_gpu():
    """The closed form against a count row by row."""
    class Args(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_int64) for n in ("batch", "heads", "queries", "keys", "dim", "block_m", "block_n", "count", "sink", "local")] +
                    [("causal", ctypes.c_int)] + [(n, ctypes.c_void_p) for n in ("q_codes", "k_codes", "k_scales")] +
                    [("k_stride", ctypes.c_int64 * 3), ("scale_stride", ctypes.c_int64 * 3), ("table", ctypes.c_void_p), ("blocks", ctypes.c_void_p),
                     ("table_width", ctypes.c_int64), ("pages", ctypes.c_int64)] + [(n, ctypes.c_void_p) for n in ("pos", "crd", "work")])
    lib = hip.load()
    for queries in (0, 1, 5, 37, 100):
        for keys in (0, 1, 9, 64, 101):
            for m in (1, 2, 7, 64):
                for n in (1, 3, 16, 50):
                    for count in (1, 4, 1000):
                        for causal in (0, 1):
                            a = Args(batch=1, heads=1, queries=queries, keys=keys, dim=8, block_m=m, block_n=n, count=count, causal=causal)
                            got = ctypes.c_int64(-1)
                            assert lib.lapis_hip_block_select_entries(ctypes.byref(a), ctypes.byref(got)) == 0
                            columns, want = -(-keys // n), 0
                            for r in range(-(-queries // m)):
                                last = min((r + 1) * m, queries) - 1
                                seen = min(max((last + keys - queries) // n + 1, 0), columns) if causal else columns
                                want += min(seen, count)
                            assert got.value == want, (queries, keys, m, n, count, causal)


def test_scratch_sizes_are_asked_for_after_init():
    """They go by the number of compute units."""
    lib = hip.load()
    if hip._initialized:
        pytest.skip("another test has initialised the library")
    buffer, bytes_ = ctypes.create_string_buffer(1024), ctypes.c_int64(-1)
    for rc in (lib.lapis_hip_block_attention_backward_work(buffer, ctypes.byref(bytes_)), lib.lapis_hip_paged_attention_work(buffer, buffer, ctypes.byref(bytes_))):
        assert lib.lapis_hip_status_name(rc) == b"LAPIS_HIP_ERR_NOT_INITIALIZED" and bytes_.value == -1


@pytest.mark.parametrize("call", [attention, gradient, select])
def test_a_flag_that_has_no_truth_value(call):
    class Flag:
        def __bool__(self):
            raise KeyError("neither")
    with pytest.raises(KeyError, match="neither"):
        call(causal=Flag())
