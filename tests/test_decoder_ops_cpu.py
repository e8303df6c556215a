"""Host-side checks of the decoder-block entry points, on CPU: descriptions
that the C interface refuses before any launch (the pointers are never
followed), and what the Python side refuses without a device."""

import copy
import ctypes
import pickle

import pytest
import torch

from cim22_b200 import abi, cim_ops, kv_cache, native
from cim22_b200.kv_cache import Int8KVCache

HERE = 4096  # an address that is never read


def cache(**kw):
    d = dict(codes=HERE, scales=HERE, pages=4, kv_heads=2, block=16, head_dim=32)
    return abi.KvCache(**{**d, **kw})


def sequences(**kw):
    d = dict(batch=2, table=HERE, table_stride=3, table_width=3, lengths=HERE, starts=HERE, rows=9,
             most=9)
    return abi.KvSequences(**{**d, **kw})


def attention(**kw):
    d = dict(type=abi.FLOAT32, q_heads=4, q=HERE, q_row_stride=128, q_head_stride=32, out=HERE,
             lse=None, scale=1.0, causal=1, window=0, longest=48)
    return abi.KvAttention(**{**d, **kw})


CACHES = [dict(block=8), dict(block=24), dict(head_dim=8), dict(head_dim=40), dict(head_dim=144),
          dict(kv_heads=0), dict(kv_heads=40000), dict(pages=-1), dict(pages=2 ** 31),
          dict(codes=None), dict(scales=None), dict(codes=HERE + 8), dict(scales=HERE + 4)]
SEQUENCES = [dict(batch=-1), dict(batch=65536), dict(lengths=None), dict(table=None),
             dict(table_width=-1), dict(table_stride=2), dict(rows=-1), dict(most=-1),
             dict(starts=None, rows=1)]
ATTENTIONS = [dict(type=7), dict(q_heads=0), dict(q_heads=3), dict(window=-1), dict(longest=-1),
              dict(q_row_stride=-1), dict(q_head_stride=-1), dict(scale=float("nan")),
              dict(scale=float("inf")), dict(q=None), dict(out=None)]


@pytest.mark.parametrize("c,s,a", [(c, {}, {}) for c in CACHES] + [({}, s, {}) for s in SEQUENCES]
                         + [({}, {}, a) for a in ATTENTIONS])
def test_attend_refuses(c, s, a):
    lib = native.lib()
    args = (ctypes.byref(cache(**c)), ctypes.byref(sequences(**s)), ctypes.byref(attention(**a)))
    assert lib.cim22_cuda_kv_attend(*args, HERE, 1 << 40, HERE, None) != 0
    assert native.last_error().startswith("cim22_cuda_kv_attend: ")


@pytest.mark.parametrize("c,s", [(c, {}) for c in CACHES] + [({}, s) for s in SEQUENCES])
def test_write_and_read_refuse(c, s):
    lib = native.lib()
    args = (ctypes.byref(cache(**c)), ctypes.byref(sequences(**s)))
    assert lib.cim22_cuda_kv_write(*args, abi.FLOAT32, HERE, 64, 32, HERE, 64, 32, HERE, None) != 0
    assert native.last_error().startswith("cim22_cuda_kv_write: ")
    assert lib.cim22_cuda_kv_read(*args, abi.FLOAT32, HERE, HERE, HERE, None) != 0
    assert native.last_error().startswith("cim22_cuda_kv_read: ")


def test_launches_past_the_grid_are_refused():
    lib = native.lib()
    wide = ctypes.byref(cache(kv_heads=32767))
    long = ctypes.byref(sequences(rows=2 ** 30, most=2 ** 30, table_width=2 ** 20,
                                  table_stride=2 ** 20))
    assert lib.cim22_cuda_kv_write(wide, long, abi.FLOAT16, HERE, 64, 32, HERE, 64, 32, HERE,
                                   None) != 0
    assert "too many rows" in native.last_error()
    assert lib.cim22_cuda_kv_read(wide, long, abi.FLOAT16, HERE, HERE, HERE, None) != 0
    assert "too many rows" in native.last_error()
    call = ctypes.byref(attention(type=abi.FLOAT16, q_heads=32767))
    assert lib.cim22_cuda_kv_attend(wide, long, call, HERE, 1 << 40, HERE, None) != 0
    assert "too many query rows" in native.last_error()


def test_null_and_unknown_arguments_are_refused():
    lib = native.lib()
    c, s, a = cache(), sequences(), attention()
    assert lib.cim22_cuda_kv_attend(None, ctypes.byref(s), ctypes.byref(a), HERE, 64, HERE, None)
    assert lib.cim22_cuda_kv_attend(ctypes.byref(c), None, ctypes.byref(a), HERE, 64, HERE, None)
    assert lib.cim22_cuda_kv_attend(ctypes.byref(c), ctypes.byref(s), None, HERE, 64, HERE, None)
    assert lib.cim22_cuda_kv_attend(ctypes.byref(c), ctypes.byref(s), ctypes.byref(a), HERE,
                                    1 << 40, None, None)
    for kind, k, row, status in ((7, HERE, 64, HERE), (0, None, 64, HERE), (0, HERE, -1, HERE),
                                 (0, HERE, 64, None)):
        assert lib.cim22_cuda_kv_write(ctypes.byref(c), ctypes.byref(s), kind, k, row, 32, HERE,
                                       64, 32, status, None) != 0
    assert lib.cim22_cuda_kv_read(ctypes.byref(c), ctypes.byref(s), 7, HERE, HERE, HERE, None)
    assert lib.cim22_cuda_kv_read(ctypes.byref(c), ctypes.byref(s), 0, HERE, HERE, None, None)


def test_workspace_too_small_is_refused():
    lib = native.lib()
    c = cache(pages=4096, block=64, head_dim=128)
    s = sequences(batch=1, table_width=4096, starts=None, rows=1)
    a = attention(longest=200000)
    need = lib.cim22_cuda_kv_attend_workspace(ctypes.byref(c), ctypes.byref(s), ctypes.byref(a))
    assert need > 0
    for ws, size in ((HERE, need - 1), (None, need), (HERE + 4, need)):
        assert lib.cim22_cuda_kv_attend(ctypes.byref(c), ctypes.byref(s), ctypes.byref(a), ws,
                                        size, HERE, None) != 0
        assert "workspace" in native.last_error()


def block_norm(post=None, pre=None, **kw):
    d = dict(type=abi.FLOAT32, rows=4, dim=32, x=HERE, x_stride=32, residual=HERE,
             residual_stride=32, residual_scale=1.0, gate=HERE, gate_stride=32, gate_rows=0,
             gate_columns=32, gate_type=abi.FLOAT32, gate_activation=0, h=HERE, h_stride=32,
             y=HERE, y_stride=32)
    call = abi.BlockNorm(**{**d, **kw})
    if post:
        call.post = ctypes.pointer(post)
    if pre:
        call.pre = ctypes.pointer(pre)
    return call


@pytest.mark.parametrize("call", [
    dict(type=5), dict(rows=-1), dict(rows=2 ** 31), dict(dim=0), dict(dim=16385), dict(x=None),
    dict(h=None, y=None), dict(x_stride=31), dict(residual_stride=31), dict(h_stride=31),
    dict(y_stride=31), dict(gate_type=abi.BFLOAT16), dict(gate_columns=2), dict(gate_rows=-1),
    dict(gate_activation=3), dict(post=abi.Norm(kind=3)), dict(pre=abi.Norm(kind=0)),
    dict(pre=abi.Norm(kind=1, eps=-1.0)), dict(pre=abi.Norm(kind=1, eps=float("nan"))),
    dict(post=abi.Norm(kind=1, type=abi.FLOAT16))])
def test_block_norm_refuses(call):
    assert native.lib().cim22_cuda_block_norm(ctypes.byref(block_norm(**call)), None) != 0
    assert native.last_error().startswith("cim22_cuda_block_norm: ")
    assert native.lib().cim22_cuda_block_norm(None, None) != 0


def test_empty_calls_do_nothing():
    lib = native.lib()
    assert lib.cim22_cuda_block_norm(ctypes.byref(block_norm(rows=0)), None) == 0
    c, a = ctypes.byref(cache()), ctypes.byref(attention())
    for kw in (dict(rows=0), dict(batch=0, rows=0)):
        s = ctypes.byref(sequences(**kw))
        assert lib.cim22_cuda_kv_attend(c, s, a, None, 0, HERE, None) == 0
        assert lib.cim22_cuda_kv_write(c, s, 0, HERE, 64, 32, HERE, 64, 32, HERE, None) == 0
        assert lib.cim22_cuda_kv_read(c, s, 0, HERE, HERE, HERE, None) == 0


def test_cpu_tensors_and_shapes_are_refused():
    x = torch.zeros(4, 8)
    with pytest.raises(TypeError, match="CUDA"):
        cim_ops.block_norm(x, pre=cim_ops.Norm("rms"))
    with pytest.raises(TypeError, match="CUDA"):
        Int8KVCache.over(torch.zeros(2, 1, 2, 16, 16, dtype=torch.int8), torch.zeros(2, 1, 2))
    for shape in ((2, 1, 24, 16), (2, 1, 144, 16), (2, 0, 16, 16), (2, 1, 16, 48), (-1, 1, 16, 16)):
        with pytest.raises(ValueError):
            Int8KVCache(*shape)


def test_status_messages():
    assert native.status_message(0x400) == "key/value cache page, length or start out of range"
    assert native.status_message(0x800) == "key/value cache does not support NaN or infinity"


def host_cache():
    """A cache whose tensors lie on the host, for what happens before a launch."""
    c = Int8KVCache.__new__(Int8KVCache)
    c._init(torch.zeros(2, 1, 2, 16, 16, dtype=torch.int8), torch.zeros(2, 1, 2))
    return c


def test_the_cache_keeps_the_memory_that_its_calls_use():
    c = host_cache()
    at = abi.KvCache.from_buffer_copy(c._view).codes, abi.KvCache.from_buffer_copy(c._view).scales
    storages = c.codes.untyped_storage(), c.scales.untyped_storage()
    for name in ("codes", "scales"):
        # A rebound name would let the memory go that the calls still address.
        with pytest.raises(AttributeError):
            setattr(c, name, getattr(c, name).clone())
        getattr(c, name).data = getattr(c, name).clone()
    held = {t.data_ptr() for x in vars(c).values() for t in (x if isinstance(x, tuple) else (x,))
            if isinstance(t, torch.Tensor)}
    assert at == tuple(s.data_ptr() for s in storages) and held >= set(at)


def test_copies_do_not_take_addresses_along():
    """They are made anew over the copied tensors, which have to be on a device."""
    c = host_cache()
    for copied in (copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
        with pytest.raises(TypeError, match="CUDA"):
            copied(c)


@pytest.mark.parametrize("device", ["cpu", "meta", torch.device("cpu")])
def test_a_cache_off_the_gpu_is_refused(device):
    """Its calls would hand a kernel addresses of the host."""
    with pytest.raises(TypeError, match="CUDA"):
        Int8KVCache(2, 1, 16, 16, device=device)


class Elsewhere:
    """A tensor of another device, as far as the checks look."""

    shape = (1,)
    dtype = torch.int32

    def get_device(self):
        return 5

    def data_ptr(self):
        return HERE


def test_a_status_word_of_another_device_is_refused(monkeypatch):
    """The kernels write to it."""
    launched = []
    monkeypatch.setattr(kv_cache, "launch", lambda *a: launched.append(a))
    c = host_cache()
    status = cim_ops.StatusWord(torch.device("cpu"))
    k, q = torch.zeros(2, 1, 16), torch.zeros(2, 2, 16)
    table, lengths = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    calls = [lambda: c.write(k, k, table, lengths, status=status),
             lambda: c.read(table, lengths, out=(k, k.clone()), status=status),
             lambda: c.attend(q, table, lengths, status=status)]
    for call in calls:
        call()
    assert len(launched) == 3
    status.tensor = Elsewhere()
    for call in calls:
        with pytest.raises(ValueError, match="status"):
            call()
    assert len(launched) == 3


@pytest.mark.parametrize("x,gate,rows", [
    ((12, 8), (8,), (0, 8)), ((12, 8), (1, 8), (0, 8)), ((12, 8), (3, 8), (4, 8)),
    ((12, 8), (12, 1), (1, 1)), ((3, 4, 8), (3, 8), (4, 8)), ((3, 4, 8), (12, 8), (1, 8)),
    ((3, 4, 8), (3, 4, 8), (1, 8)), ((3, 4, 8), (3, 4, 1), (1, 1)), ((3, 4, 8), (3, 1, 8), (4, 8)),
    ((3, 4, 8), (1, 1, 8), (0, 8)), ((1, 4, 8), (1, 4, 8), (1, 8)),
    ((2, 3, 4, 8), (2, 3, 8), (4, 8)), ((2, 3, 4, 8), (2, 1, 1, 1), (12, 1)),
    ((0, 4, 8), (0, 4, 8), None)])
def test_gate_shapes(x, gate, rows):
    got = cim_ops._gate_rows(torch.zeros(gate), torch.zeros(x), torch.zeros(x).numel() // 8, 8)
    assert rows is None or got == rows


@pytest.mark.parametrize("x,gate", [
    ((3, 4, 8), (1, 4, 8)), ((4, 4, 8), (1, 4, 8)), ((3, 4, 8), (1, 4, 1)), ((2, 3, 4, 8), (1, 3, 8)),
    ((2, 3, 4, 8), (2, 1, 4, 8)), ((2, 3, 4, 8), (1, 3, 1, 8)), ((6, 2, 8), (2, 3, 8)),
    ((12, 8), (3, 1, 8)), ((12, 8), (3, 4, 8)), ((3, 4, 8), (3, 4, 1, 8)), ((3, 4, 8), (4, 3, 8))])
def test_gates_of_more_axes_that_are_no_prefix_of_the_rows_are_refused(x, gate):
    """[1, T, dim] would broadcast over the batch anywhere else; its values must
    not go to consecutive rows instead."""
    with pytest.raises(ValueError, match="gate must be"):
        cim_ops._gate_rows(torch.zeros(gate), torch.zeros(x), torch.zeros(x).numel() // 8, 8)
