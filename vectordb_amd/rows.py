"""An embedding table on the GPU: rows held in 4 bits (`Int4Rows`), rows fetched by id, and that fetch's gradient.

Where `ClusteredIndex` answers from 1-bit codes and reranks with f32 rows, `Int4Rows` holds every row in 4 bits a
component with one bf16 scale per group of 32, 64 or 128, answers exhaustively (`search_batch`), and gives rows back by
id (`lookup_device`). `rows_lookup_device` / `rows_grad_device` are the lookup in a float table and its gradient, for
tables that are trained. All of it runs in libcuddle_hip.so on the GPU; there is no CPU path behind it. The reference has
no counterpart (its codes are 1-bit, its rows are fetched one at a time: src/storage/mmap.rs:106-115).

The `*_device` calls take CUDA tensors, run on their device, enqueue on `stream` (default: torch's current stream of that
device) and return tensors that are valid once that stream has been waited for. Work space comes from torch's
allocator, on the same stream; a call may be recorded into a graph. Autograd records none of them, so a call whose result
is a smooth function of an input (a lookup's table, the queries of distances, a gradient) refuses one that requires a
gradient outside `torch.no_grad()`: detach it and call `rows_grad_device`.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools
from typing import List, Optional, Tuple

import numpy as np
import torch

from . import _ffi
from .builder import metric_id

_TYPES = {torch.float32: _ffi.TYPE_F32, torch.float16: _ffi.TYPE_F16, torch.bfloat16: _ffi.TYPE_BF16}


def _type_id(t: torch.dtype) -> int:
    if t not in _TYPES:
        raise ValueError(f"float32, float16 or bfloat16, not {t}")
    return _TYPES[t]


def _cuda(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("this runs on the GPU: pass CUDA tensors")
        if t.device != dev:
            raise ValueError(f"tensors on {dev} and {t.device}")
    return dev


def _no_grad(what: str, t: torch.Tensor) -> None:
    """Refuses an input whose gradient would be lost without a word: no call here is recorded by autograd."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, which autograd does not record here: pass {what}.detach()")


def _rows2d(x: torch.Tensor) -> torch.Tensor:
    """x with unit stride along its rows (itself, where it has that already)."""
    if x.dim() != 2:
        raise ValueError(f"rows must be [n, dim], not {tuple(x.shape)}")
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _id_bits(ids: torch.Tensor) -> int:
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be int32 or int64, not {ids.dtype}")
    return 32 if ids.dtype == torch.int32 else 64


_NO_CTX = contextlib.nullcontext()
# the current stream's handle without a Stream object around it, where torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _enter(dev: torch.device, stream, *inputs: torch.Tensor):
    """(context, device index, hipStream_t) for work on `dev` and `stream`: inside the context torch's copies and
    allocations belong to the stream. Inputs used on a stream that is not the current one are kept for it."""
    index = dev.index if dev.index is not None else torch.cuda.current_device()
    if stream is not None and stream.device.index != index:
        raise ValueError(f"a stream of {stream.device} for tensors on {dev}")
    if stream is None or stream.cuda_stream == _raw_stream(index):
        return _NO_CTX, index, _raw_stream(index)
    for t in inputs:
        t.record_stream(stream)
    return torch.cuda.stream(stream), index, stream.cuda_stream


def _workspace(nbytes: int, dev: torch.device) -> Optional[torch.Tensor]:
    return torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes else None


class Int4Rows:
    """Rows in 4 bits (struct cuddle_int4_rows): `codes` uint8 [bytes], `scales` bfloat16 [n, scale_stride], `sqnorm`
    float64 [n], all on one GPU. Made by `int4_encode_device`, or by `empty` and `encode_device` in pieces."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, sqnorm: torch.Tensor, n: int, dim: int, group: int):
        nbytes, stride = self._sizes(n, dim, group)
        dev = _cuda(codes, scales, sqnorm)
        if codes.dtype != torch.uint8 or codes.numel() < nbytes or not codes.is_contiguous():
            raise ValueError(f"codes must be {nbytes} contiguous bytes")
        if scales.dtype != torch.bfloat16 or tuple(scales.shape) != (n, stride) or not scales.is_contiguous():
            raise ValueError(f"scales must be contiguous bfloat16 [{n}, {stride}]")
        if sqnorm.dtype != torch.float64 or tuple(sqnorm.shape) != (n,) or not sqnorm.is_contiguous():
            raise ValueError(f"sqnorm must be contiguous float64 [{n}]")
        self.codes, self.scales, self.sqnorm = codes, scales, sqnorm
        self.n, self.dim, self.group, self.device = n, dim, group, dev
        self._desc = _ffi.Int4RowsDesc(codes.data_ptr(), scales.data_ptr(), sqnorm.data_ptr(), n, dim, group)

    @staticmethod
    @functools.lru_cache(maxsize=256)
    def _sizes(n: int, dim: int, group: int) -> Tuple[int, int]:
        nbytes, stride = C.c_uint64(0), C.c_uint32(0)
        _ffi.check(_ffi.lib().cuddle_int4_sizes(n, dim, group, C.byref(nbytes), C.byref(stride)))
        return int(nbytes.value), int(stride.value)

    @classmethod
    def empty(cls, n: int, dim: int, group: int = 64, device="cuda") -> "Int4Rows":
        """Room for n rows, to be filled by `encode_device`."""
        nbytes, stride = cls._sizes(n, dim, group)
        dev = torch.device(device)
        return cls(torch.empty((nbytes,), dtype=torch.uint8, device=dev), torch.empty((n, stride), dtype=torch.bfloat16, device=dev),
                   torch.empty((n,), dtype=torch.float64, device=dev), n, dim, group)

    def __len__(self) -> int:
        return self.n

    @property
    def device_bytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel() + 8 * self.sqnorm.numel()

    @property
    def group_scales(self) -> torch.Tensor:
        """The scales without the padding of their rows: a view, bfloat16 [n, ceil(dim / group)]."""
        return self.scales[:, :-(-self.dim // self.group)]

    def encode_device(self, x: torch.Tensor, first_row: int = 0, stream=None) -> "Int4Rows":
        """Encodes x [m, dim] (float32, float16, bfloat16; rows may be strided) into rows first_row .. first_row + m - 1."""
        if x.dim() != 2 or x.shape[1] != self.dim:
            raise ValueError("dimension mismatch")
        dev, kind = _cuda(self.codes, x), _type_id(x.dtype)
        if first_row < 0 or first_row + x.shape[0] > self.n:
            raise ValueError(f"rows {first_row} .. {first_row + x.shape[0]} of {self.n}")
        ctx, index, st = _enter(dev, stream, x, *self._arrays)
        with ctx:
            x = _rows2d(x)
            _ffi.check(_ffi.lib().cuddle_int4_encode_device(C.byref(self._desc), first_row, x.shape[0], x.data_ptr(), kind,
                                                            x.stride(0) if x.shape[0] > 1 else self.dim, index, st))
        return self

    def lookup_device(self, ids: Optional[torch.Tensor], scale: float = 1.0, dtype: torch.dtype = torch.float32, stream=None) -> torch.Tensor:
        """scale * row ids[...] as `dtype` [..., dim]; an id outside [0, n) gives zeros. ids None: all rows in order."""
        kind = _type_id(dtype)
        if ids is None:
            dev, bits, shape, given = self.device, 32, (self.n,), ()
        else:
            dev, bits, shape, given = _cuda(self.codes, ids), _id_bits(ids), tuple(ids.shape), (ids,)
        ctx, index, st = _enter(dev, stream, *given, *self._arrays)
        with ctx:
            out = torch.empty(shape + (self.dim,), dtype=dtype, device=dev)
            ids = None if ids is None else ids.contiguous()
            _ffi.check(_ffi.lib().cuddle_int4_lookup_device(C.byref(self._desc), None if ids is None else ids.data_ptr(), bits,
                                                            self.n if ids is None else ids.numel(), float(scale), kind, out.data_ptr(), index, st))
        return out

    def decode_device(self, dtype: torch.dtype = torch.float32, stream=None) -> torch.Tensor:
        """What all rows stand for, [n, dim]."""
        return self.lookup_device(None, 1.0, dtype, stream)

    @property
    def _arrays(self):
        return self.codes, self.scales, self.sqnorm

    def _queries(self, q: torch.Tensor) -> Tuple[torch.device, int]:
        if q.dim() != 2 or q.shape[1] != self.dim:
            raise ValueError("Query dimension mismatch")
        return _cuda(self.codes, q), _type_id(q.dtype)

    def _ws(self, nq: int, k: int, dev: torch.device):
        """(tensor that keeps the work space, its address or None, bytes)"""
        need = C.c_uint64(0)
        _ffi.check(_ffi.lib().cuddle_int4_workspace(self.n, self.dim, nq, k, C.byref(need)))
        ws = _workspace(need.value, dev)
        return ws, None if ws is None else ws.data_ptr(), need.value

    def distances_device(self, queries: torch.Tensor, metric="l2", stream=None) -> torch.Tensor:
        """distance(query, row) of queries [nq, dim] (float32, float16, bfloat16) to every row: float32 [nq, n]."""
        (dev, kind), m = self._queries(queries), metric_id(metric)
        _no_grad("queries", queries)
        ctx, index, st = _enter(dev, stream, queries, *self._arrays)
        with ctx:
            q = queries.contiguous()
            out = torch.empty((q.shape[0], self.n), dtype=torch.float32, device=dev)
            ws, at, need = self._ws(q.shape[0], 0, dev)
            _ffi.check(_ffi.lib().cuddle_int4_distances_device(C.byref(self._desc), q.data_ptr(), kind, q.shape[0], m, out.data_ptr(), at, need,
                                                               index, st))
        return out

    def search_batch_device(self, queries: torch.Tensor, k: int, metric="l2", stream=None):
        """The k nearest rows of every query, over all rows: (ids int64 [nq, k], dist float32 [nq, k], count int32 [nq]),
        ordered by (distance, row); unused slots hold -1 (UINT64_MAX) and +inf."""
        (dev, kind), m = self._queries(queries), metric_id(metric)
        nq = queries.shape[0]
        ctx, index, st = _enter(dev, stream, queries, *self._arrays)
        with ctx:
            q = queries.contiguous()
            k = min(max(int(k), 0), 0xFFFFFFFF)  # refused by the library
            ws, at, need = self._ws(nq, k, dev)
            ids = torch.empty((nq, k), dtype=torch.int64, device=dev)
            dist = torch.empty((nq, k), dtype=torch.float32, device=dev)
            count = torch.empty((nq,), dtype=torch.int32, device=dev)
            _ffi.check(_ffi.lib().cuddle_int4_search_device(C.byref(self._desc), q.data_ptr(), kind, nq, k, m, ids.data_ptr(), dist.data_ptr(),
                                                            count.data_ptr(), at, need, index, st))
        return ids, dist, count

    # ---- host forms, as ClusteredIndex has them ---------------------------------------------------
    def search_batch(self, queries: np.ndarray, k: int, metric="l2"):
        """search_batch_device for host queries: (ids uint64 [nq, k], dist [nq, k], count [nq])."""
        q = torch.from_numpy(np.ascontiguousarray(queries, dtype=np.float32)).to(self.device)
        ids, dist, count = self.search_batch_device(q, k, metric)
        return ids.cpu().numpy().view(np.uint64), dist.cpu().numpy(), count.cpu().numpy().view(np.uint32)

    def search(self, query, k: int, metric="l2") -> List[Tuple[int, float]]:
        """The k nearest rows of one query: [(id, distance)], ascending."""
        ids, dist, count = self.search_batch(np.asarray(query, dtype=np.float32)[None, :], k, metric)
        return [(int(i), float(d)) for i, d in zip(ids[0, :count[0]], dist[0, :count[0]])]


def int4_encode_device(x: torch.Tensor, group: int = 64, stream=None) -> Int4Rows:
    """x [n, dim] (float32, float16, bfloat16) as 4-bit rows (cuddle_int4_encode_device)."""
    if x.dim() != 2:
        raise ValueError(f"rows must be [n, dim], not {tuple(x.shape)}")
    ctx, _, _ = _enter(_cuda(x), stream, x)
    with ctx:
        return Int4Rows.empty(x.shape[0], x.shape[1], group, x.device).encode_device(x)


def rows_lookup_device(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, stream=None) -> torch.Tensor:
    """scale * table[ids] for a float32, float16 or bfloat16 table [n, dim] (rows may be strided) and int32 or int64 ids of
    any shape: [*ids.shape, dim] of the table's type. An id outside [0, n) gives zeros."""
    if table.dim() != 2:
        raise ValueError(f"rows must be [n, dim], not {tuple(table.shape)}")
    _no_grad("table", table)
    dev, bits, kind = _cuda(table, ids), _id_bits(ids), _type_id(table.dtype)
    n, dim = table.shape
    ctx, index, st = _enter(dev, stream, table, ids)
    with ctx:
        out = torch.empty(tuple(ids.shape) + (dim,), dtype=table.dtype, device=dev)
        table, ids = _rows2d(table), ids.contiguous()
        _ffi.check(_ffi.lib().cuddle_rows_lookup_device(table.data_ptr(), kind, table.stride(0) if n > 1 else dim, n, dim, ids.data_ptr(), bits,
                                                        ids.numel(), float(scale), out.data_ptr(), index, st))
    return out


def rows_grad_device(grad_out: torch.Tensor, ids: torch.Tensor, n_rows: int, scale: float = 1.0, dtype: Optional[torch.dtype] = None,
                     out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Gradient of rows_lookup_device with respect to the table: row v = scale * the sum of grad_out [*ids.shape, dim] over
    the ids equal to v, summed in float32 in a fixed order: [n_rows, dim] of `dtype` (default: grad_out's).
    out: a contiguous gradient [n_rows, dim], apart from grad_out, that the sums are added to (rows without ids are not
    touched); returned."""
    dim = grad_out.shape[-1]
    if tuple(grad_out.shape[:-1]) != tuple(ids.shape):
        raise ValueError(f"grad_out {tuple(grad_out.shape)} does not fit ids {tuple(ids.shape)}")
    _no_grad("grad_out", grad_out)
    given = (grad_out, ids) if out is None else (grad_out, ids, out)
    dev, bits, kind = _cuda(*given), _id_bits(ids), _type_id(grad_out.dtype)
    out_dtype = out.dtype if out is not None else dtype or grad_out.dtype
    out_kind = _type_id(out_dtype)
    if out is not None and (tuple(out.shape) != (n_rows, dim) or not out.is_contiguous() or (dtype is not None and dtype != out.dtype)):
        raise ValueError(f"out must be a contiguous [{n_rows}, {dim}]")
    flags = _ffi.GRAD_ACCUMULATE if out is not None else 0
    ctx, index, st = _enter(dev, stream, *given)
    with ctx:
        grad = out if out is not None else torch.empty((n_rows, dim), dtype=out_dtype, device=dev)
        g, ids = _rows2d(grad_out.reshape(ids.numel(), dim)), ids.contiguous()
        need = C.c_uint64(0)
        _ffi.check(_ffi.lib().cuddle_rows_grad_workspace(ids.numel(), n_rows, dim, C.byref(need)))
        ws = _workspace(need.value, dev)
        _ffi.check(_ffi.lib().cuddle_rows_grad_device(g.data_ptr(), kind, g.stride(0) if g.shape[0] > 1 else dim, ids.data_ptr(), bits, ids.numel(),
                                                      float(scale), n_rows, dim, flags, out_kind, grad.data_ptr(), None if ws is None else ws.data_ptr(), need.value,
                                                      index, st))
    return grad
