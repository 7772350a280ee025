"""GPU checks of how the 8-bit cache's and the logit rules' calls are made: defaults, other
alignments, what a call leaves alone."""
import importlib

import numpy as np
import pytest

from _util import need_cuda

pytestmark = pytest.mark.gpu

D = 128


def att():
    return importlib.import_module("0xbitnet_b200.attention")


def test_appends_without_a_position_follow_one_another():
    """Two calls without pos write the rows that one call for both writes."""
    torch = need_cuda()
    B, H, Hkv, n = 2, 4, 2, 5
    rng = np.random.default_rng(0)
    qkv = torch.from_numpy(rng.standard_normal((B, 2 * n, (H + 2 * Hkv) * D)).astype(np.float32))
    one, two = att().KVCacheQ8(B, 16, Hkv), att().KVCacheQ8(B, 16, Hkv)
    rows = lambda t: t.reshape(-1, t.shape[-1]).contiguous().cuda()
    want = att().rope_kv_append_q8(rows(qkv), one, H, 2 * n).view(B, 2 * n, -1)
    for i in range(2):
        got = att().rope_kv_append_q8(rows(qkv[:, i * n:(i + 1) * n]), two, H, n).view(B, n, -1)
        assert torch.equal(got, want[:, i * n:(i + 1) * n])
        assert two.seq_len == (i + 1) * n
    for a, b in zip(one.read(0, 2 * n), two.read(0, 2 * n)):  # a step apart where the scale grew
        step = torch.maximum(one.k_scale, one.v_scale).max()
        assert torch.all((a - b).abs() <= step)
    assert torch.equal(one.k_scale, two.k_scale) and torch.equal(one.v_scale, two.v_scale)
    # an earlier position given by the caller moves nothing back, one on the device nothing at all
    att().rope_kv_append_q8(rows(qkv[:, :n]), two, H, n, pos=3)
    att().rope_kv_append_q8(rows(qkv[:, :n]), two, H, n,
                            pos=torch.tensor([1, 11], dtype=torch.int32, device="cuda"))
    assert two.seq_len == 2 * n
    with pytest.raises(importlib.import_module("0xbitnet_b200").ObnError):
        att().rope_kv_append_q8(rows(qkv[:, :2 * n - 1]), two, H, 2 * n - 1)  # no room for all
    assert two.seq_len == 2 * n
