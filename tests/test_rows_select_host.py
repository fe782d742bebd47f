"""The selection kernels of the exhaustive search (csrc/cuddle_rows_select.hpp) run on the CPU, thread by thread, by a host
program that gives each list exactly the room a launch asks for and looks behind it afterwards."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("select") / "select_on_host")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wno-unknown-pragmas", "-I", os.path.join(ROOT, "vectordb_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "select_on_host.cpp"), "-o", exe], check=True)
    return exe


# 73 828 rows, k = 1000: the second level's last chunk has 1808 places, of which 908 hold rows and the rest is fill, for
# lists of 1000; 671 800 rows, k = 100: the same a hundred times smaller. The others are the ordinary run of sizes.
@pytest.mark.parametrize("n,k,nq,kind", [(73_828, 1000, 1, "random"), (73_828, 1000, 3, "random"), (73_828, 1000, 2, "nan"), (73_828, 1000, 2, "ties"),
                                         (671_800, 100, 1, "random"), (671_800, 100, 2, "nan"), (1, 3, 2, "nan"), (100, 10, 2, "random"),
                                         (8192, 100, 1, "random"), (8193, 1024, 2, "random"), (50_000, 100, 1, "random"), (30_000, 16, 3, "nan"),
                                         (30_000, 16, 3, "ties"), (600_000, 1024, 1, "random"), (5, 100, 2, "collection"), (8000, 100, 3, "collection")])
def test_selection_on_the_host(program, n, k, nq, kind):
    r = subprocess.run([program, str(n), str(k), str(nq), kind], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_no_launch_reads_behind_the_scales(tmp_path):
    exe = str(tmp_path / "plan_on_host")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", os.path.join(ROOT, "vectordb_amd", "csrc"), os.path.join(ROOT, "tests", "cpp", "plan_on_host.cpp"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
