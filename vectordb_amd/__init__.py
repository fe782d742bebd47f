"""vectordb_amd — MI355X-native batched two-phase ANN query path of CuddleDB (LLay/vectordb).

Only what the path needs: the HIP library (csrc/ -> libcuddle_hip.so, C ABI in
include/cuddle_hip.h), its ctypes binding, the flat index form + builder, and the host-side
mirror of the reference's `ClusteredIndex` search API; beside it an embedding table in 4 bits with
exhaustive search, row lookup and the lookup's gradient (rows.py).
"""
from importlib.util import find_spec

from ._ffi import CuddleError, METRIC_L2, METRIC_COSINE, METRIC_DOT, CODE_BINARY, CODE_RABITQ  # noqa: F401
from .flat_index import FlatIndex, pack_binary_codes  # noqa: F401
from .index import ClusteredIndex, ClusteredIndexWithRaBitQ, DeviceIndex, SearchStats  # noqa: F401

from .pyvectordb import PyVectorDB  # noqa: E402

__all__ = ["ClusteredIndex", "ClusteredIndexWithRaBitQ", "DeviceIndex", "FlatIndex", "SearchStats", "CuddleError", "PyVectorDB"]

# the embedding table works on torch tensors: torch is imported with its first use, not before, and a host without it has
# the rest of the names
_ROWS = ("Int4Rows", "int4_encode_device", "rows_lookup_device", "rows_grad_device")
if find_spec("torch") is not None:
    __all__ += _ROWS


def __getattr__(name):
    if name in _ROWS:
        from . import rows

        return getattr(rows, name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
