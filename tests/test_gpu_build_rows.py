"""GPU: the index builder takes its rows through the library's lookup; inputs of other layouts than whole rows."""
import numpy as np
import pytest
import torch

from vectordb_amd import rows as R
from vectordb_amd.builder import build_index

from helpers import clustered

pytestmark = pytest.mark.gpu


def _same(a, b):
    for name in ("centroids", "child_offsets", "children", "roots", "vec_offsets", "ids", "vectors", "codes"):
        assert np.array_equal(getattr(a, name), getattr(b, name)), name
    assert a.threshold == b.threshold


@pytest.mark.parametrize("layout", ["transposed", "fortran", "every other column", "part of wider rows"])
def test_strided_rows_are_copied_once(gpu, monkeypatch, layout):
    x = clustered(3000, 24, 20, 5)
    want = build_index(torch.from_numpy(x).cuda(gpu), 8, 30, "l2", 10, seed=2, threshold=0.0)
    if layout == "transposed":
        given = torch.from_numpy(np.ascontiguousarray(x.T)).cuda(gpu).t()
    elif layout == "fortran":
        given = torch.from_numpy(np.asfortranarray(x)).cuda(gpu)
    elif layout == "part of wider rows":
        wide = torch.zeros((3000, 40), device=torch.device("cuda", gpu))
        wide[:, 7:31] = torch.from_numpy(x).cuda(gpu)
        given = wide[:, 7:31]
    else:
        wide = torch.zeros((3000, 48), device=torch.device("cuda", gpu))
        wide[:, ::2] = torch.from_numpy(x).cuda(gpu)
        given = wide[:, ::2]
    tables, lookup = [], R.rows_lookup_device

    def seen(table, ids, *args, **kw):
        tables.append((table.data_ptr(), table.stride()))
        return lookup(table, ids, *args, **kw)

    monkeypatch.setattr(R, "rows_lookup_device", seen)
    _same(build_index(given, 8, 30, "l2", 10, seed=2, threshold=0.0, device="cuda"), want)
    assert len(tables) > 10 and len(set(tables)) == 1 and tables[0][1][1] == 1  # one table, whole rows
    assert (tables[0][0] == given.data_ptr()) if layout == "part of wider rows" else (tables[0][1][0] == 24)  # a copy only where needed


def test_rows_longer_than_a_lookup_takes(gpu):
    """A single leaf needs no assignment, whose dimensions are limited too."""
    x = clustered(12, 33_000, 3, 6)
    want = build_index(x, 8, 30, "l2", 10, seed=2, threshold=0.0)
    got = build_index(torch.from_numpy(x).cuda(gpu), 8, 30, "l2", 10, seed=2, threshold=0.0)
    assert np.array_equal(got.vectors, want.vectors) and np.array_equal(got.codes, want.codes) and np.array_equal(got.ids, want.ids)
    # a mean of 12 floats in two orders: 11 roundings of sums each, and one of the quotient
    assert np.all(np.abs(got.centroids - want.centroids) <= (2 * 11 + 2) * 2.0 ** -24 * np.abs(x).sum(0) / 12)
