"""Embedding table, CPU side: sizes, refusals (every argument check comes before the GPU is touched), the 64-bit reference."""
import ctypes as C

import numpy as np
import pytest
import torch

from vectordb_amd import _ffi
import vectordb_amd
from vectordb_amd import rows as R

import rows_reference as ref

L = _ffi.lib()


def _desc(n=32, dim=128, group=64, codes=0x10000, scales=0x10000, sq=0x10000):
    return _ffi.Int4RowsDesc(codes, scales, sq, n, dim, group)


def _sizes(n, dim, group):
    b, s = C.c_uint64(0), C.c_uint32(0)
    st = L.cuddle_int4_sizes(n, dim, group, C.byref(b), C.byref(s))
    return st, int(b.value), int(s.value)


def test_struct_layout():
    assert C.sizeof(_ffi.Int4RowsDesc) == 40


@pytest.mark.parametrize("n,dim,group,want", [(1, 1, 32, (512 + 16, 4)), (16, 64, 64, (512 + 16, 2)), (17, 65, 64, (2048, 2)), (1000, 960, 64, (63 * 15 * 512 + 16, 16)),
                                              (1000, 960, 32, (63 * 15 * 512 + 16, 32)), (10, 1536, 128, (24 * 512, 16)), (0, 8, 32, (0, 4)),
                                              (3, 300, 128, (5 * 512 + 16, 4))])
def test_sizes(n, dim, group, want):
    assert _sizes(n, dim, group) == (_ffi.OK,) + want


def test_sizes_refusals():
    assert _sizes(1, 0, 64)[0] == _ffi.ERR_BAD_ARG
    assert _sizes(1, 40000, 64)[0] == _ffi.ERR_UNSUPPORTED
    assert _sizes(1, 64, 48)[0] == _ffi.ERR_BAD_ARG
    assert _sizes(2 ** 32, 64, 64)[0] == _ffi.ERR_UNSUPPORTED
    assert L.cuddle_int4_sizes(1, 64, 64, None, None) == _ffi.ERR_BAD_ARG


def test_encode_refusals():
    f = L.cuddle_int4_encode_device
    P = 0x20000
    ok = _desc()
    assert f(None, 0, 1, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG
    assert f(C.byref(ok), 0, 1, None, 0, 128, 0, None) == _ffi.ERR_BAD_ARG
    assert f(C.byref(ok), 0, 1, P, 3, 128, 0, None) == _ffi.ERR_BAD_ARG            # element type
    assert f(C.byref(ok), 0, 2, P, 0, 127, 0, None) == _ffi.ERR_BAD_ARG            # rows overlap
    assert f(C.byref(ok), 31, 2, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG           # past the end
    assert f(C.byref(ok), 2 ** 63, 2 ** 63, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG
    assert f(C.byref(ok), 0, 1, P + 2, 0, 128, 0, None) == _ffi.ERR_BAD_ARG        # f32 rows at an odd address
    assert f(C.byref(_desc(group=16)), 0, 1, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG
    assert f(C.byref(_desc(dim=0)), 0, 1, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG
    assert f(C.byref(_desc(dim=32769)), 0, 1, P, 0, 40000, 0, None) == _ffi.ERR_UNSUPPORTED
    assert f(C.byref(_desc(sq=None)), 0, 1, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG
    assert f(C.byref(_desc(codes=0x10008)), 0, 1, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG
    assert f(C.byref(_desc(scales=0x10002)), 0, 1, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG
    assert f(C.byref(_desc(sq=0x10004)), 0, 1, P, 0, 128, 0, None) == _ffi.ERR_BAD_ARG


def test_query_refusals():
    P, ws = 0x20000, 0x40000
    need = C.c_uint64(0)
    assert L.cuddle_int4_workspace(32, 128, 2, 5, C.byref(need)) == _ffi.OK and need.value > 0
    assert L.cuddle_int4_workspace(32, 128, 2, 1025, C.byref(need)) == _ffi.ERR_UNSUPPORTED
    assert L.cuddle_int4_workspace(32, 128, 2, 5, None) == _ffi.ERR_BAD_ARG
    assert L.cuddle_int4_workspace(10_000_000, 128, 0, 5, C.byref(need)) == _ffi.OK  # no queries: no work
    d = lambda r=_desc(), q=P, t=0, nq=5, m=0, out=P, w=ws, b=1 << 30: L.cuddle_int4_distances_device(  # noqa: E731
        None if r is None else C.byref(r), q, t, nq, m, out, w, b, 0, None)
    s = lambda r=_desc(), q=P, t=0, nq=2, k=5, m=0, i=P, o=P, w=ws, b=1 << 30: L.cuddle_int4_search_device(  # noqa: E731
        None if r is None else C.byref(r), q, t, nq, k, m, i, o, None, w, b, 0, None)
    for call in (d, s):
        assert call(r=None) == _ffi.ERR_BAD_ARG
        assert call(q=None) == _ffi.ERR_BAD_ARG
        assert call(t=7) == _ffi.ERR_BAD_ARG
        assert call(m=3) == _ffi.ERR_BAD_ARG
        assert call(w=None) == _ffi.ERR_BAD_ARG
        assert call(b=16) == _ffi.ERR_BAD_ARG
        assert call(w=ws + 16) == _ffi.ERR_BAD_ARG
        assert call(r=_desc(sq=None)) == _ffi.ERR_BAD_ARG  # L2 needs the norms
        assert call(r=_desc(n=2 ** 32)) == _ffi.ERR_UNSUPPORTED
    assert d(out=None) == _ffi.ERR_BAD_ARG
    assert L.cuddle_int4_workspace(32, 128, 4, 0, C.byref(need)) == _ffi.OK and need.value == 0  # up to four queries need none
    assert s(k=0) == _ffi.ERR_BAD_ARG
    assert s(k=1025) == _ffi.ERR_UNSUPPORTED
    assert s(i=None) == _ffi.ERR_BAD_ARG
    assert s(o=None) == _ffi.ERR_BAD_ARG


def test_lookup_and_grad_refusals():
    P, ws = 0x20000, 0x40000
    lk = lambda table=P, t=0, stride=64, n=10, dim=64, ids=P, bits=64, m=4, out=P: L.cuddle_rows_lookup_device(  # noqa: E731
        table, t, stride, n, dim, ids, bits, m, 1.0, out, 0, None)
    assert lk(table=None) == lk(ids=None) == lk(out=None) == _ffi.ERR_BAD_ARG
    assert lk(t=9) == lk(bits=16) == lk(stride=63) == lk(dim=0) == lk(ids=P + 4) == lk(table=P + 1) == _ffi.ERR_BAD_ARG
    assert lk(dim=32769, stride=32769) == _ffi.ERR_UNSUPPORTED
    i4 = lambda r=_desc(), ids=P, bits=64, m=4, t=0, out=P: L.cuddle_int4_lookup_device(C.byref(r), ids, bits, m, 1.0, t, out, 0, None)  # noqa: E731
    assert i4(bits=8) == i4(t=4) == i4(out=None) == i4(out=P + 2) == _ffi.ERR_BAD_ARG
    assert i4(ids=None, m=33) == _ffi.ERR_BAD_ARG  # all rows: no more than there are
    need = C.c_uint64(0)
    assert L.cuddle_rows_grad_workspace(4, 10, 64, C.byref(need)) == _ffi.OK
    assert L.cuddle_rows_grad_workspace(2 ** 31, 10, 64, C.byref(need)) == _ffi.ERR_UNSUPPORTED
    assert L.cuddle_rows_grad_workspace(4, 2 ** 32, 64, C.byref(need)) == _ffi.ERR_UNSUPPORTED
    assert L.cuddle_rows_grad_workspace(4, 10, 64, None) == _ffi.ERR_BAD_ARG
    gr = lambda g=P, t=0, stride=64, ids=P, bits=64, m=4, n=10, dim=64, fl=0, gt=0, out=P, w=ws, b=1 << 30: L.cuddle_rows_grad_device(  # noqa: E731
        g, t, stride, ids, bits, m, 1.0, n, dim, fl, gt, out, w, b, 0, None)
    assert gr(g=None) == gr(ids=None) == gr(out=None) == gr(w=None) == gr(b=8) == gr(w=ws + 8) == _ffi.ERR_BAD_ARG
    assert gr(t=5) == gr(gt=5) == gr(fl=2) == gr(bits=1) == gr(stride=63) == gr(dim=0) == gr(out=P + 2) == _ffi.ERR_BAD_ARG
    assert gr(m=2 ** 31) == gr(n=2 ** 32) == _ffi.ERR_UNSUPPORTED


def test_valid_calls_without_a_gpu_fail_loudly():
    if L.cuddle_device_count() > 0:
        pytest.skip("a GPU is visible here")
    P, ws = 0x20000, 0x40000
    r = _desc()
    assert L.cuddle_int4_encode_device(C.byref(r), 0, 1, P, 0, 128, 0, None) == _ffi.ERR_NO_DEVICE
    assert L.cuddle_int4_distances_device(C.byref(r), P, 0, 1, 0, P, ws, 1 << 30, 0, None) == _ffi.ERR_NO_DEVICE
    assert L.cuddle_int4_search_device(C.byref(r), P, 0, 1, 3, 0, P, P, None, ws, 1 << 30, 0, None) == _ffi.ERR_NO_DEVICE
    assert L.cuddle_rows_lookup_device(P, 0, 64, 10, 64, P, 64, 4, 1.0, P, 0, None) == _ffi.ERR_NO_DEVICE
    assert L.cuddle_rows_grad_device(P, 0, 64, P, 64, 4, 1.0, 10, 64, 0, 0, P, ws, 1 << 30, 0, None) == _ffi.ERR_NO_DEVICE


def test_python_refusals():
    x = torch.zeros((4, 64))
    with pytest.raises(ValueError, match="GPU"):
        R.int4_encode_device(x)
    with pytest.raises(ValueError, match="GPU"):
        R.rows_lookup_device(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU"):
        R.rows_grad_device(x, torch.zeros(4, dtype=torch.int64), 9)
    with pytest.raises(ValueError, match="fit"):
        R.rows_grad_device(x, torch.zeros(5, dtype=torch.int64), 9)
    with pytest.raises(ValueError):
        R.rows_lookup_device(torch.zeros(4), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(AttributeError):
        vectordb_amd.no_such_name
    assert vectordb_amd.Int4Rows is R.Int4Rows


def test_reference_encode_is_the_definition():
    """The 64-bit reference against itself stated element by element, ties and tiny groups included."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 70)).astype(np.float32)
    x[1] = 0.0
    x[2, :64] = 0.0
    x[2, 0], x[2, 1], x[2, 2], x[2, 3] = 7.0, 0.5, 1.5, -2.5  # scale 1: halves go to the even code
    x[3, 5] = np.inf
    x[4] = np.float32(1e-45)
    codes, scales, values, sq = ref.encode(x, 64)
    assert codes[2, :4].tolist() == [7, 0, 2, -2] and scales[2, 0] == 1.0
    assert not codes[1].any() and not scales[1].any() and sq[1] == 0.0
    assert np.isnan(scales[3, 0]) and np.isfinite(scales[3, 1]) and np.isnan(values[3, :64]).all() and np.isfinite(values[3, 64:]).all()
    assert scales[4, 0] == 0.0 and not codes[4].any()
    for r in (0, 2):
        for i in range(70):
            s = float(scales[r, i // 64])
            assert abs(x[r, i] / s - codes[r, i]) <= 0.5 or abs(codes[r, i]) == 7
    assert np.allclose(sq[0], (values[0] ** 2).sum(), rtol=1e-14)
