import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_collection_modifyitems(config, items):
    import torch

    if torch.cuda.is_available():
        return
    skip = pytest.mark.skip(reason="no GPU in this environment")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(autouse=True)
def product_table_as_it_was():
    """The table of measured products is the process's: what a test tunes or loads does not choose the kernels of the tests behind it."""
    ops = sys.modules.get("arle_amd.kernels.ops")
    before = dict(ops._PRODUCT_TABLE) if ops is not None else None
    yield
    if before is not None and ops._PRODUCT_TABLE != before:
        ops.clear_product_table()
        ops._PRODUCT_TABLE.update(before)


def pytest_sessionfinish(session, exitstatus):
    """With ARLE_TEST_STATS=<file>: the worst maximum and rms errors that the comparisons with the plain
    implementation saw, one line a comparison (what the tolerances are set against)."""
    path = os.environ.get("ARLE_TEST_STATS")
    if not path:
        return
    try:
        import replay
    except ImportError:
        return
    with open(path, "w") as fh:
        for what, (worst, rms, spread) in sorted(replay.last_stats.items()):
            fh.write(f"{worst:.3e} {rms:.3e} {spread:5.2f} {what}\n")
