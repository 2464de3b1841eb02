"""What importing the package brings in."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)


def test_formats_and_coarsener_do_not_import_torch():
    """Host-side use (formats, coarsening) needs numpy alone; torch comes with the first plan or serving operator."""
    r = run("import sys, sparse_computation_b200 as sc; sc.CSR; assert 'torch' not in sys.modules, 'torch was imported'")
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("code", [
    "import sparse_computation_b200 as sc; sc.PagedKVCache; sc.RotaryTable; sc.DecodeAttention; sc.LowRankAdapters",
    "from sparse_computation_b200 import PagedKVCache, RotaryTable, DecodeAttention, LowRankAdapters",
    "import sparse_computation_b200 as sc; assert 'LowRankAdapters' in dir(sc) and not hasattr(sc, 'nothing')",
    "import sparse_computation_b200 as sc; from sparse_computation_b200 import serving; assert sc.PagedKVCache is serving.PagedKVCache",
])
def test_serving_operators_are_names_of_the_package(code):
    r = run(code)
    assert r.returncode == 0, r.stderr
