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


def cpu_rules(**kw):
    """LogitRules of tensors on the CPU: its own checks but for the device's; nothing is launched."""
    import torch
    lg = importlib.import_module("0xbitnet_b200.logits")

    class Rules(lg.LogitRules):
        def _take(self, t, name, dtype):
            assert t.dtype is dtype
            self._kept.append(t)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    return Rules(**{k: i32(*v) if k != "bias_values" else torch.zeros(v) for k, v in kw.items()})


@pytest.mark.parametrize("shapes", [
    dict(mask=(4, 0)), dict(mask=(0,)), dict(mask=(1, 0)),            # an empty mask allowed all ids
    dict(history=(1, 3, 5)), dict(mask=(1, 2, 4)), dict(history=()),  # only [rows, cap] or [cap]
    dict(bias_ids=(1, 2, 2), bias_values=(1, 2, 2)), dict(history=(2, 3, 5))])
def test_rule_lists_of_other_shapes_are_refused(shapes):
    with pytest.raises(ValueError):
        cpu_rules(**shapes)


def test_rule_lists_that_stay_allowed():
    assert cpu_rules(mask=(3, 4)).mask_words == 4
    r = cpu_rules(history=(1, 7), mask=(5,))
    assert (r._struct.history_ld, r._struct.history_cap, r.rows) == (0, 7, None)
    r = cpu_rules(history=(2, 0), bias_ids=(2, 3), bias_values=(2, 3))
    assert (r._struct.history_cap, r._struct.bias_cap, r.rows) == (0, 3, 2)


@pytest.mark.parametrize("shift", [4, -4, 4 * 100, 4 * 199, -4 * 199])
def test_overlapping_logits_and_out_are_refused(shift):
    """Rows written over others that are still to be read; refused before anything is launched."""
    import ctypes
    obn = importlib.import_module("0xbitnet_b200")
    rules = obn._lib.LogitRulesStruct()
    at = 1 << 20  # never read
    assert obn.lib().obn_logits_process(at, 2, 100, ctypes.addressof(rules), at + shift, None, None) == -1
    assert b"overlap" in obn.lib().obn_error_message()


def test_a_call_runs_on_its_tensors_device(monkeypatch):
    """From another current device: the device is switched for the call, and the stream is that
    device's. From the same one: no switch."""
    import contextlib
    import types
    att = importlib.import_module("0xbitnet_b200.attention")
    current, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        was, current[0] = current[0], index
        yield
        current[0] = was
    entry = lambda *args: seen.append((current[0], args)) or 0
    monkeypatch.setattr(att, "lib", lambda: types.SimpleNamespace(obn_entry=entry))
    monkeypatch.setattr(att, "_current_device", lambda: current[0])
    monkeypatch.setattr(att, "_raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(att.torch.cuda, "device", device)
    att._call("obn_entry", 1, "a", 2)
    att._call("obn_entry", 0, "b")
    assert seen == [(1, ("a", 2, 101)), (0, ("b", 100))] and current == [0]
