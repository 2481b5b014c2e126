"""examples/tree_verify.py runs: the draft-tree operators together, checked against decode over the compacted cache."""
import importlib.util
import os

import pytest

from _util import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v_fmt", ["q8_0", "fp16"])
def test_example(v_fmt):
    spec = importlib.util.spec_from_file_location("tree_verify", os.path.join(ROOT, "examples", "tree_verify.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    # both rows are rounded to bf16 (2^-8 of |o| < 1 here) and differ by the kernels' own 2e-3 + 1e-2 |o|
    assert m.main(v_fmt, seed=3) < 1e-2
