import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


@pytest.fixture(autouse=True)
def no_wait_runs_out(request):
    """The paged cache's GPU tests leave no copy wait that ran out unnoticed."""
    watched = request.module.__name__.startswith('test_paged') and request.node.get_closest_marker('gpu')
    if watched:
        from motif_b200 import _lib
        _lib.wait_timeouts()
    yield
    if watched:
        assert _lib.wait_timeouts() == 0


def pytest_configure(config):
    config.addinivalue_line('markers', 'gpu: needs a CUDA B200 and the built libmotif_b200.so')
