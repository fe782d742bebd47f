"""The package's public names, with and without torch."""
import subprocess
import sys

import pytest


def _python(code):
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)


def test_star_import_without_torch():
    """A host without torch gets everything that works without it."""
    r = _python("import sys; sys.modules['torch'] = None\n"
                "from vectordb_amd import *\n"
                "print(ClusteredIndex.__name__, PyVectorDB.__name__, FlatIndex.__name__, CuddleError.__name__)")
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == ["ClusteredIndex", "PyVectorDB", "FlatIndex", "CuddleError"]


def test_star_import_with_torch():
    pytest.importorskip("torch")
    r = _python("from vectordb_amd import *\nprint(Int4Rows.__name__, int4_encode_device.__name__, rows_lookup_device.__name__, rows_grad_device.__name__)")
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == ["Int4Rows", "int4_encode_device", "rows_lookup_device", "rows_grad_device"]


def test_import_alone_leaves_torch_alone():
    r = _python("import sys, vectordb_amd; print('torch' in sys.modules)")
    assert r.returncode == 0 and r.stdout.split() == ["False"], r.stdout + r.stderr
