"""The example that runs the E4M3 operators and the router's gradient together does what it says."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_router_evens_out():
    spec = importlib.util.spec_from_file_location("balance_router_fp8", os.path.join(ROOT, "examples", "balance_router_fp8.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    loads = example.main(steps=15, tokens=1024, quiet=True)
    assert loads[0] > 3 and min(loads[-5:]) < loads[0] / 2
