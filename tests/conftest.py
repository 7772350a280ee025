import importlib
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA GPU (B200, sm_100a)")


@pytest.fixture(autouse=True)
def _no_device_errors(request):
    """After each GPU test: no kernel's bounded wait gave up in it."""
    yield
    if request.node.get_closest_marker("gpu"):
        import torch
        if torch.cuda.is_available() and torch.cuda.is_initialized():
            importlib.import_module("0xbitnet_b200").check_device_errors()
