"""CPU checks of the 8-bit cache's and the logit rules' host side: what it needs of torch, the
device a call runs on, and arguments that must not reach a kernel."""
import importlib
import subprocess
import sys

import pytest

from _util import ROOT

WITHOUT = """
import importlib, torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
att = importlib.import_module("0xbitnet_b200.attention")
importlib.import_module("0xbitnet_b200.logits")
class Stream:
    cuda_stream = 77
torch.cuda.current_stream = lambda index: Stream if index == 1 else None
assert att._raw_stream(1) == 77
assert att._current_device is torch.cuda.current_device
"""


def test_import_without_torchs_private_calls():
    r = subprocess.run([sys.executable, "-c", WITHOUT], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("value", [2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 31 - 1, 10 ** 30])
def test_positions_beyond_32_bits_are_refused(value):
    """2^32 + 5 is not position 5."""
    att = importlib.import_module("0xbitnet_b200.attention")
    with pytest.raises(ValueError):
        att._host_or_dev(value, None, "pos")
    assert att._host_or_dev(2 ** 31 - 1, None, "pos") == (2 ** 31 - 1, None)
    assert att._host_or_dev(-2 ** 31, None, "pos") == (-2 ** 31, None)
