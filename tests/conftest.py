"""Test configuration: import paths and the ``gpu`` marker.

Tests marked ``gpu`` need a B200 and call the kernels through the public API and
the C-ABI library; everything else runs on a CPU-only host.
"""

import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for path in (os.path.join(ROOT, "atrex-kernels_b200", "python"), ROOT, os.path.join(ROOT, "tests")):
    if path not in sys.path:
        sys.path.insert(0, path)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an sm_100a GPU (B200)")


def pytest_collection_modifyitems(config, items):
    # Profiler sessions come back without device events once the process is a minute or two old, and a test that needs
    # them then skips: those tests run first, close to each other.
    items.sort(key=lambda item: "only_atrex_kernels_run" not in item.name)
    try:
        import torch

        has_gpu = torch.cuda.is_available()
    except Exception:  # pragma: no cover
        has_gpu = False
    if has_gpu:
        return
    skip = pytest.mark.skip(reason="no CUDA device")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)
