"""pytest configuration: the `gpu` marker, import paths for the product package (microscaling-quant_b200/mxq)
and the test-only oracle (oracle/oracle.py)."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "microscaling-quant_b200")
for p in (PKG, os.path.join(ROOT, "oracle"), os.path.join(ROOT, "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (B200); run with -m gpu")


#: Tests that hold a value that was found wrong and is no longer returned; they stand as they were written and are expected to fail.
#: test_groups: without a bias its helper sums the two largest *logits* of a group, which ranks [10, -5] (scores 1.0000 and 0.0067)
#: before [2, 2] (0.8808 each); groups are ranked by the sum of scores (test_gpu_route_groups.py has the same shapes and more).
WRONG_VALUES = {f"test_gpu_route.py::test_groups[{case}]" for case in (
    "8-4-2-softmax", "64-8-3-softmax", "64-8-3-sigmoid", "256-8-4-softmax", "96-4-1-softmax", "40-5-2-softmax", "40-5-2-sigmoid",
    "128-32-7-softmax", "128-32-7-sigmoid", "1024-16-4-softmax", "1024-16-4-sigmoid")}


def pytest_collection_modifyitems(items):
    for item in items:
        if item.nodeid.split("/")[-1] in WRONG_VALUES:
            item.add_marker(pytest.mark.xfail(strict=True, raises=AssertionError, reason="sums logits where scores are meant"))


@pytest.fixture(scope="session")
def oracle():
    import oracle as o
    o.lib()
    return o


@pytest.fixture(autouse=True)
def _no_lost_tiles(request):
    """After every GPU test: no bounded TMA wait gave up (a lost tile is written as NaN and would otherwise only show
    as wrong values). The timeout test clears what it provokes."""
    yield
    if request.node.get_closest_marker("gpu") is None:
        return
    import torch
    if not torch.cuda.is_available() or not torch.cuda.is_initialized():
        return
    torch.cuda.synchronize()
    from mxq import _lib
    w = _lib._wait_word
    assert w is None or w.value == 0, f"{w.value} bounded TMA wait(s) gave up during this test"
