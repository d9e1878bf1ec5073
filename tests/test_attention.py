"""Refusals of the operators on sequences, without a GPU: argument checks answer before any kernel is launched."""
import ctypes

import pytest
import torch

import sapa_b200


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def _packed(q=(6, 4, 16), k=(6, 2, 16), v=None, dtype=torch.float32, offsets=None, **kw):
    return sapa_b200.packed_attention(torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=dtype), torch.zeros(v or k, dtype=dtype),
                                      _ints(0, 6) if offsets is None else offsets, **kw)


def _paged(q=(2, 4, 16), pages=(5, 8, 2, 16), table=(2, 3), lengths=2, offsets=3, dtype=torch.float32, **kw):
    return sapa_b200.paged_attention(torch.zeros(q, dtype=dtype), torch.zeros(pages, dtype=dtype), torch.zeros(pages, dtype=dtype),
                                     torch.zeros(table, dtype=torch.int32), torch.zeros(lengths, dtype=torch.int32),
                                     torch.zeros(offsets, dtype=torch.int32), **kw)


def _write(k=(2, 2, 16), v=None, pages=(5, 8, 2, 16), table=(2, 3), lengths=2, offsets=3, dtype=torch.float32):
    sapa_b200.paged_write(torch.zeros(k, dtype=dtype), torch.zeros(v or k, dtype=dtype), torch.zeros(pages, dtype=dtype), torch.zeros(pages, dtype=dtype),
                          torch.zeros(table, dtype=torch.int32), torch.zeros(lengths, dtype=torch.int32), torch.zeros(offsets, dtype=torch.int32))


@pytest.mark.parametrize("call", [_packed, _paged, _write])
def test_cpu_tensors_are_not_implemented(call):
    with pytest.raises(NotImplementedError):
        call()


@pytest.mark.parametrize("kw", [dict(q=(6, 4)), dict(q=(6, 3, 16)), dict(q=(6, 4, 24)), dict(k=(5, 2, 16)), dict(v=(6, 1, 16)), dict(v=(6, 2, 8)),
                                dict(offsets=_ints()), dict(offsets=_ints(0, 6).view(1, 2)), dict(key_offsets=_ints(0, 3, 6)), dict(k=(6, 0, 16))])
def test_packed_shapes(kw):
    with pytest.raises(AssertionError):
        _packed(**kw)


@pytest.mark.parametrize("kw", [dict(q=(2, 4)), dict(q=(2, 3, 16)), dict(q=(2, 4, 8)), dict(pages=(0, 8, 2, 16)), dict(table=(1, 3)), dict(table=(2, 0)),
                                dict(lengths=3), dict(offsets=2)])
def test_paged_shapes(kw):
    with pytest.raises(AssertionError):
        _paged(**kw)


@pytest.mark.parametrize("kw", [dict(k=(2, 2)), dict(v=(1, 2, 16)), dict(k=(2, 1, 16)), dict(pages=(5, 8, 2, 8)), dict(table=(3, 3)), dict(lengths=1)])
def test_write_shapes(kw):
    with pytest.raises(AssertionError):
        _write(**kw)


@pytest.mark.parametrize("call", [lambda **kw: _packed(q=(6, 4, kw.pop("dim", 16)), k=(6, 2, kw.pop("kd", 16)), **kw),
                                  lambda **kw: _paged(q=(2, 4, kw.pop("dim", 16)), pages=(5, 8, 2, kw.pop("kd", 16)), **kw)])
def test_sizes_and_types_without_a_kernel(call):
    for dim in (4, 12, 136, 256):
        with pytest.raises(RuntimeError, match="multiple of 8 up to 128"):
            call(dim=dim, kd=dim)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        call(dtype=torch.float64)
    for scale in (float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="scale"):
            call(scale=scale)
    with pytest.raises(RuntimeError, match="128 query heads"):
        _packed(q=(6, 129, 16), k=(6, 1, 16))


# ---------------------------------------------------------------------------------- the C ABI
class _Attention(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("query", "key", "value", "out", "lse", "low", "offsets", "key_offsets", "page_table", "key_lengths")] +
                [("query_strides", ctypes.c_longlong * 2), ("key_strides", ctypes.c_longlong * 3), ("value_strides", ctypes.c_longlong * 3)] +
                [(n, ctypes.c_int) for n in ("B", "tokens", "keys", "pages", "page", "max_pages", "heads", "groups", "dim", "causal")] +
                [("scale", ctypes.c_float)])


def _arguments(**kw):
    a = _Attention(query=4096, key=4096, value=4096, out=4096, lse=4096, low=4096, offsets=4096, key_offsets=4096, B=1, tokens=4, keys=4, heads=4, groups=2, dim=16, causal=1,
                   scale=1.0)
    a.query_strides[:] = (64, 16)
    a.key_strides[:] = a.value_strides[:] = (32, 16, 0)
    for name, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, name)[:] = v
        else:
            setattr(a, name, v)
    return a


@pytest.mark.parametrize("kw, dtype, status, text", [
    (dict(), 3, -2, b"dtype"), (dict(query=0), 0, -1, b"NULL"), (dict(out=0), 0, -1, b"NULL"), (dict(key=0), 0, -1, b"NULL"), (dict(offsets=0), 0, -1, b"NULL"),
    (dict(key_offsets=0), 0, -1, b"NULL"), (dict(heads=3), 0, -1, b"share"), (dict(groups=0), 0, -1, b"share"), (dict(dim=12), 0, -5, b"dim"),
    (dict(dim=136), 0, -5, b"dim"), (dict(heads=258), 0, -5, b"128"), (dict(tokens=-1), 0, -1, b"size"), (dict(query=4100), 0, -3, b"aligned"),
    (dict(query_strides=(66, 16)), 0, -3, b"strides"), (dict(key_strides=(32, -16, 0)), 0, -3, b"strides"), (dict(query_strides=(68, 16)), 1, -3, b"strides"),
    (dict(page_table=4096), 0, -1, b"key_lengths"), (dict(page_table=4096, key_lengths=4096), 0, -1, b"positive"),
    (dict(page_table=4096, key_lengths=4096, pages=1, page=1 << 16, max_pages=1 << 16), 0, -5, b"positions"), (dict(scale=float("inf")), 0, -1, b"scale")])
def test_c_entry_points_refuse(kw, dtype, status, text):
    from sapa_b200 import _lib
    h = _lib.lib()
    a = _arguments(**kw)
    ref = ctypes.byref(a)
    assert h.sapa_attention_forward(ref, None, 0, dtype, None) == status
    assert text in h.sapa_last_error()
    assert h.sapa_attention_workspace(ref, dtype) == 0
    assert h.sapa_attention_backward(ref, 4096, 64, 16, 4096, 4096, 4096, 4096, 1 << 20, dtype, None) < 0


def test_c_backward_refuses():
    from sapa_b200 import _lib
    h = _lib.lib()

    def call(a, go=4096, stride=64, gq=4096, gk=4096, ws=4096, size=1 << 20):
        return h.sapa_attention_backward(ctypes.byref(a), go, stride, 16, gq, gk, 4096, ws, size, 0, None)
    assert call(_arguments(page_table=4096, key_lengths=4096, pages=1, page=1, max_pages=1)) == -5
    assert call(_arguments(lse=0)) == -1 and call(_arguments(low=0)) == -1 and call(_arguments(), go=0) == -1 and call(_arguments(), gq=0) == -1 and call(_arguments(), gk=0) == -1
    assert call(_arguments(), stride=66) == -3 and call(_arguments(), go=4100) == -3
    assert call(_arguments(), size=8) == -6 and call(_arguments(), ws=0) == -6
    assert h.sapa_attention_forward(None, None, 0, 0, None) == -1
