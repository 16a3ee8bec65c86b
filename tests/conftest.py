"""Shared pytest setup: the `gpu` marker, repo import path, fixture loading."""

import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent
if str(REPO) not in sys.path:
    sys.path.insert(0, str(REPO))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA (B200) device")
    config.addinivalue_line("markers", "bench: large shapes whose timing is reported")


def pytest_collection_modifyitems(config, items):
    try:
        import torch

        have_gpu = torch.cuda.is_available()
    except Exception:  # pragma: no cover
        have_gpu = False
    if have_gpu:
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(autouse=True)
def no_wait_runs_out(request):
    """After every GPU test of the paged operators: no bounded wait of the tree attention ran out."""
    yield
    if "gpu" in request.keywords and request.module.__name__.startswith(("test_tree", "test_page")):
        import torch

        if torch.cuda.is_available():
            from iron_b200 import _lib

            assert _lib.load().iron_tree_attn_status(1) == 0, "a wait of the tree attention timed out"
