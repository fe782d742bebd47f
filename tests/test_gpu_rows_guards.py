"""GPU: the embedding table's C entry points on arrays that lie tightly between guard bytes, at the sizes where a list or an
array ends inside what a kernel handles at a time."""
import ctypes as C

import numpy as np
import pytest
import torch

from vectordb_amd import _ffi
from vectordb_amd import rows as R

import rows_reference as ref

pytestmark = pytest.mark.gpu

GUARD, MARK = 16384, 0xA5


class Carver:
    """Arrays out of one allocation, 256-byte aligned, GUARD marked bytes behind each one's last byte."""

    def __init__(self, gpu, room):
        self.buf = torch.full((room,), MARK, dtype=torch.uint8, device=torch.device("cuda", gpu))
        self.at, self.spans = 0, []

    def take(self, shape, dtype):
        size = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
        a = self.at
        self.spans.append((a, a + size))
        self.at = (a + size + GUARD + 255) // 256 * 256
        assert self.at <= self.buf.numel()
        return self.buf[a:a + size].view(dtype).view(shape)

    def check(self):
        torch.cuda.synchronize()
        for _, end in self.spans:
            assert bool((self.buf[end:end + GUARD] == MARK).all()), f"written behind byte {end}"


def _search(gpu, x, q, k, group=32):
    """cuddle_int4_search_device on tight arrays: (ids, dist, the table)."""
    n, dim = x.shape
    nq = q.shape[0]
    code_bytes, stride = R.Int4Rows._sizes(n, dim, group)
    need = C.c_uint64(0)
    _ffi.check(_ffi.lib().cuddle_int4_workspace(n, dim, nq, k, C.byref(need)))
    sizes = [code_bytes, 2 * n * stride, 8 * n, 4 * nq * dim, 8 * nq * k, 4 * nq * k, 4 * nq, need.value]
    c = Carver(gpu, sum(s + GUARD + 256 for s in sizes))
    table = R.Int4Rows(c.take((code_bytes,), torch.uint8), c.take((n, stride), torch.bfloat16), c.take((n,), torch.float64), n, dim, group)
    table.encode_device(x)
    qt = c.take((nq, dim), torch.float32)
    qt.copy_(q)
    ids, dist, count = c.take((nq, k), torch.int64), c.take((nq, k), torch.float32), c.take((nq,), torch.int32)
    ws = c.take((need.value,), torch.uint8)
    _ffi.check(_ffi.lib().cuddle_int4_search_device(C.byref(table._desc), qt.data_ptr(), _ffi.TYPE_F32, nq, k, _ffi.METRIC_L2, ids.data_ptr(), dist.data_ptr(),
                                                    count.data_ptr(), ws.data_ptr(), need.value, gpu, torch.cuda.current_stream().cuda_stream))
    c.check()
    assert count.tolist() == [min(k, n)] * nq
    return ids, dist, table


# second-level chunks that are longer than k and hold fewer than k rows (the rest is fill): 908 of 1808, 64 of 108,
# 47 of 124, 36 of 208
@pytest.mark.parametrize("n,nq,k", [(73_828, 1, 1000), (73_828, 3, 1000), (671_800, 1, 100), (671_800, 2, 100), (876_545, 2, 77), (335_900, 4, 200)])
def test_search_with_short_last_lists(gpu, n, nq, k):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n + nq)
    x = torch.randn((n, 16), generator=gen, device="cuda")
    q = torch.randn((nq, 16), generator=gen, device="cuda")
    ids, dist, table = _search(gpu, x, q, k)
    d = table.distances_device(q)
    order = torch.argsort(d, dim=1, stable=True)[:, :k]
    assert torch.equal(ids, order)
    assert torch.equal(dist, torch.gather(d, 1, order))


def test_search_with_short_last_lists_after_an_overflow(gpu):
    """A sampled search whose collections all overflow (every row the same): the levels answer, with such a last list."""
    n, nq, k = 335_900, 100, 200
    x = torch.ones((n, 16), device="cuda")
    ids, dist, table = _search(gpu, x, torch.zeros((nq, 16), device="cuda"), k)
    assert torch.equal(ids, torch.arange(k, device="cuda").expand(nq, k))
    assert bool((dist == dist[0, 0]).all()) and abs(float(dist[0, 0]) - 16) < 0.1


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,dim,nq", [(256, 64, 24), (4096, 128, 32), (513, 16, 61), (1024, 100, 128), (16, 65, 88), (1, 128, 101), (2048, 33, 200)])
def test_distances_of_short_rows(gpu, n, dim, nq, group):
    """Eight quartets of queries against rows of one or two units, the scales' last row at the array's end."""
    rng = np.random.default_rng(n + dim + nq)
    x = torch.from_numpy(rng.standard_normal((n, dim)).astype(np.float32)).cuda(gpu)
    q = torch.from_numpy(rng.standard_normal((nq, dim)).astype(np.float32)).cuda(gpu)
    code_bytes, stride = R.Int4Rows._sizes(n, dim, group)
    need = C.c_uint64(0)
    _ffi.check(_ffi.lib().cuddle_int4_workspace(n, dim, nq, 0, C.byref(need)))
    c = Carver(gpu, code_bytes + 2 * n * stride + 8 * n + 4 * n * nq + need.value + 5 * (GUARD + 256))
    table = R.Int4Rows(c.take((code_bytes,), torch.uint8), c.take((n, stride), torch.bfloat16), c.take((n,), torch.float64), n, dim, group)
    table.encode_device(x)
    out, ws = c.take((nq, n), torch.float32), c.take((need.value,), torch.uint8)
    _ffi.check(_ffi.lib().cuddle_int4_distances_device(C.byref(table._desc), q.data_ptr(), _ffi.TYPE_F32, nq, _ffi.METRIC_L2, out.data_ptr(), ws.data_ptr(),
                                                       need.value, gpu, torch.cuda.current_stream().cuda_stream))
    c.check()
    values = ref.encode(x.cpu().numpy(), group)[2]
    want = ref.distances(values, q.cpu().numpy(), "l2")
    assert np.all(np.abs(out.cpu().double().numpy() - want) <= ref.distance_tolerance(values, q.cpu().numpy(), want, "l2"))


@pytest.mark.parametrize("dtype,out", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float16)])
@pytest.mark.parametrize("n,dim,t,accumulate", [(1, 1, 1, 0), (7, 33, 5, 0), (50, 128, 2048, 1), (300, 130, 2049, 0), (40, 24, 8192, 0), (40, 24, 8193, 1),
                                                (1000, 8, 70_000, 0), (3, 520, 140_001, 0), (1_200_001, 3, 300_000, 0)])
def test_gradient_between_guards(gpu, n, dim, t, accumulate, dtype, out):
    rng = np.random.default_rng(n + dim + t)
    need = C.c_uint64(0)
    _ffi.check(_ffi.lib().cuddle_rows_grad_workspace(t, n, dim, C.byref(need)))
    c = Carver(gpu, 4 * (t + n) * dim + 8 * t + need.value + 5 * (GUARD + 256))
    g, ids = c.take((t, dim), dtype), c.take((t,), torch.int64)
    grad, ws = c.take((n, dim), out), c.take((need.value,), torch.uint8)
    g.copy_(torch.from_numpy(rng.integers(-8, 9, (t, dim)).astype(np.float32)))  # whole numbers: f32 sums are exact
    at = rng.integers(-2, n, t)
    at[rng.random(t) < 0.3] = n - 1  # a run over many chunks, at the end of the table
    ids.copy_(torch.from_numpy(at))
    grad.fill_(3.0 if accumulate else float("nan"))
    _ffi.check(_ffi.lib().cuddle_rows_grad_device(g.data_ptr(), R._TYPES[dtype], dim, ids.data_ptr(), 64, t, 0.5, n, dim, accumulate, R._TYPES[out],
                                                  grad.data_ptr(), ws.data_ptr(), need.value, gpu, torch.cuda.current_stream().cuda_stream))
    c.check()
    want = torch.from_numpy(ref.grad(g.double().cpu().numpy(), at, n, 0.5)[0] + 3.0 * accumulate)
    assert torch.equal(grad.cpu(), want.to(torch.float32).to(out))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,dim,group,nq", [(1, 1, 32, 1), (17, 65, 64, 4), (16, 130, 128, 5), (31, 200, 32, 9), (100, 960, 64, 17), (33, 2050, 32, 33), (5, 4500, 128, 3)])
def test_rows_between_guards(gpu, n, dim, group, nq, dtype):
    """Encoding, distances, decoding and lookups, of tables and rows that end inside a tile, a unit and a store."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n + dim)
    lib, kind, st = _ffi.lib(), R._TYPES[dtype], torch.cuda.current_stream().cuda_stream
    code_bytes, stride = R.Int4Rows._sizes(n, dim, group)
    need = C.c_uint64(0)
    _ffi.check(lib.cuddle_int4_workspace(n, dim, nq, 0, C.byref(need)))
    c = Carver(gpu, code_bytes + 2 * n * stride + 8 * n + 4 * nq * (n + dim) + need.value + 4 * 8 * n * dim + 8 * 3 * n + 12 * (GUARD + 256))
    table = R.Int4Rows(c.take((code_bytes,), torch.uint8), c.take((n, stride), torch.bfloat16), c.take((n,), torch.float64), n, dim, group)
    x = c.take((n, dim), dtype)
    x.copy_(torch.randn((n, dim), generator=gen, device="cuda"))
    q = c.take((nq, dim), dtype)
    q.copy_(torch.randn((nq, dim), generator=gen, device="cuda"))
    dist, ws = c.take((nq, n), torch.float32), c.take((need.value,), torch.uint8)
    decoded, fetched, looked = c.take((n, dim), dtype), c.take((3 * n, dim), dtype), c.take((3 * n, dim), dtype)
    ids = c.take((3 * n,), torch.int64)
    ids.copy_(torch.randint(-1, n + 1, (3 * n,), generator=gen, device="cuda"))
    _ffi.check(lib.cuddle_int4_encode_device(C.byref(table._desc), 0, n, x.data_ptr(), kind, dim, gpu, st))
    _ffi.check(lib.cuddle_int4_distances_device(C.byref(table._desc), q.data_ptr(), kind, nq, _ffi.METRIC_DOT, dist.data_ptr(), ws.data_ptr(), need.value, gpu, st))
    _ffi.check(lib.cuddle_int4_lookup_device(C.byref(table._desc), None, 32, n, 1.0, kind, decoded.data_ptr(), gpu, st))
    _ffi.check(lib.cuddle_int4_lookup_device(C.byref(table._desc), ids.data_ptr(), 64, 3 * n, 2.0, kind, fetched.data_ptr(), gpu, st))
    _ffi.check(lib.cuddle_rows_lookup_device(x.data_ptr(), kind, dim, n, dim, ids.data_ptr(), 64, 3 * n, 2.0, looked.data_ptr(), gpu, st))
    c.check()
    xs, qs, at = x.double().cpu().numpy(), q.double().cpu().numpy(), ids.cpu().numpy()
    values = ref.encode(xs, group)[2]
    want = ref.distances(values, qs, "dot")
    assert np.all(np.abs(dist.double().cpu().numpy() - want) <= ref.distance_tolerance(values, qs, want, "dot"))
    # 12 significant bits times a power of two, and a value times a power of two: one rounding, to the type
    assert torch.equal(decoded.cpu(), torch.from_numpy(values).to(dtype))
    assert torch.equal(fetched.cpu(), torch.from_numpy(ref.lookup(values, at, 2.0)).to(dtype))
    assert torch.equal(looked.cpu(), torch.from_numpy(ref.lookup(xs, at, 2.0)).to(dtype))
