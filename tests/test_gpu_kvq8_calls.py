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


@pytest.mark.parametrize("B,n,H,Hkv,S,ragged", [
    (1, 4, 300, 75, 6000, False), (2, 4, 320, 80, 2000, False), (4, 4, 160, 40, 1000, False),
    (8, 1, 40, 40, 3000, False), (1, 1, 32, 32, 60000, False), (3, 4, 128, 32, 2000, True),
    (1, 2, 150, 150, 5000, True), (1, 1, 300, 300, 3000, False)])
def test_many_kv_heads(B, n, H, Hkv, S, ragged):
    """KV heads that do not divide the CTAs, few of them and more than there are CTAs: every head
    and sequence against the same call for that head alone (another split of the keys)."""
    torch = need_cuda()
    g = torch.Generator(device="cuda")
    g.manual_seed(B + Hkv)
    c = att().KVCacheQ8(B, S, Hkv)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda").to(torch.int8))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp2(torch.randint(-8, -4, t.shape, generator=g, device="cuda").float()))
    q = torch.randn((B, n, H, D), generator=g, device="cuda")
    L = [S - 700 * b for b in range(B)] if ragged else [S] * B
    arg = torch.tensor(L, dtype=torch.int32, device="cuda") if ragged else S
    got = att().attention_q8(q.view(B * n, -1), c, H, n, arg).view(B, n, H, D)
    G = H // Hkv
    for h in sorted({0, 1, Hkv // 2, Hkv - 2, Hkv - 1}):
        for b in range(B):
            one = att().KVCacheQ8.wrap(*[t[b:b + 1, :, h:h + 1].contiguous()
                                         for t in (c.k, c.k_scale, c.v, c.v_scale)])
            rows = q[b, :, h * G:(h + 1) * G].reshape(n, -1).contiguous()
            want = att().attention_q8(rows, one, G, n, L[b]).view(n, G, D)
            # both are f32 results of the same values: apart by two roundings of the scores' range
            # (|s| < 64 in log2, 48 u of it and of the sums' 24 steps), relative to the mean of |v|
            err = (got[b, :, h * G:(h + 1) * G] - want).abs().max().item()
            top = (one.v.float().abs().amax() * one.v_scale.max()).item()
            assert err <= 2 * 2.0 ** -24 * (2 * 48 * 64 + 64) * top, (h, b, err)


@pytest.mark.parametrize("R,V", [(1, 40000), (3, 9999), (5, 31), (2, 1), (64, 1003)])
@pytest.mark.parametrize("x_off,y_off", [(0, 1), (1, 0), (2, 1), (3, 3), (1, 2)])
def test_logits_and_out_of_different_alignment(R, V, x_off, y_off):
    """Buffers that begin 0 to 3 elements behind a 16-byte boundary: the same bits, and nothing
    around the output is written."""
    torch = need_cuda()
    lg = importlib.import_module("0xbitnet_b200.logits")
    g = torch.Generator(device="cuda")
    g.manual_seed(R + V)
    x = torch.randn((R, V), generator=g, device="cuda")
    hist = torch.randint(0, V, (R, 200), generator=g, device="cuda").int()
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (R, -(-V // 32)), generator=g, device="cuda").int()
    ids = torch.randint(0, V, (R, 9), generator=g, device="cuda").int()
    rules = lg.LogitRules(repetition=torch.full((R,), 1.3, device="cuda"), history=hist, mask=mask,
                          bias_ids=ids, bias_values=torch.randn((R, 9), generator=g, device="cuda"))
    want, token = lg.logits_process(x, rules)
    a, b = torch.full((2, R * V + 8), 5.0, device="cuda")
    a[x_off:x_off + R * V] = x.view(-1)
    out = b[y_off:y_off + R * V].view(R, V)
    _, got = lg.logits_process(a[x_off:x_off + R * V].view(R, V), rules, out=out)
    assert torch.equal(out, want) and torch.equal(got, token)
    assert bool((b[:y_off] == 5.0).all()) and bool((b[y_off + R * V:] == 5.0).all())
