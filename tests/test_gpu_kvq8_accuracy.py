"""GPU checks of attention over the 8-bit cache against a bound near the error of f32 arithmetic,
row by row (oracle/q8_ref.py: attention_rms). A lost or additional key, at a border of units, CTAs or
of the sequence, and any operand held in fewer bits than the comments say are far outside it."""
import importlib

import numpy as np
import pytest

from _util import need_cuda
from oracle import q8_ref as ref

pytestmark = pytest.mark.gpu

D = 128
SCALE = float(np.float32(1.0) / np.sqrt(np.float32(D)))


def cache(torch, rng, B, S, Hkv):
    """Random codes with scales a factor of 4 apart, and the values in 64 bits."""
    att = importlib.import_module("0xbitnet_b200.attention")
    c = att.KVCacheQ8(B, S, Hkv, D)
    vals = []
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        cn = rng.integers(-127, 128, (B, S, Hkv, D), dtype=np.int8)
        sn = np.exp2(rng.integers(-7, -4, (B, -(-S // ref.BLOCK), Hkv))).astype(np.float32)
        codes.copy_(torch.from_numpy(cn))
        scale.copy_(torch.from_numpy(sn))
        vals.append(np.stack([ref.values(cn[b], sn[b]) for b in range(B)]))
    return c, vals[0], vals[1]


def ratio(got, want, tol):
    """The error's root mean square over each row, against its bound."""
    return (np.sqrt(((got - want) ** 2).mean(-1)) / tol).max()


@pytest.mark.parametrize("B,n,H,Hkv,S", [
    (1, 1, 20, 5, 2048), (1, 1, 4, 4, 40000), (1, 1, 4, 2, 131072), (6, 1, 10, 5, 900),
    (2, 4, 32, 4, 3000), (1, 8, 2, 2, 20000), (1, 24, 5, 5, 3000), (1, 60, 4, 4, 1500),
    (1, 128, 16, 8, 1025), (1, 512, 20, 5, 2100), (3, 260, 8, 2, 3000), (1, 100, 2, 2, 40000)])
def test_error_is_near_that_of_f32(B, n, H, Hkv, S):
    torch = need_cuda()
    att = importlib.import_module("0xbitnet_b200.attention")
    rng = np.random.default_rng(S + n)
    c, k, v = cache(torch, rng, B, S, Hkv)
    q = rng.standard_normal((B, n, H, D)).astype(np.float32)
    got = att.attention_q8(torch.from_numpy(q.reshape(B * n, -1)).cuda(), c, H, n, S)
    got = got.cpu().numpy().reshape(B, n, H, D)
    for b in range(B):
        want, tol = ref.attention_rms(q[b], k[b], v[b], S, SCALE)
        assert ratio(got[b], want, tol) <= 1, b


@pytest.mark.parametrize("n,H,Hkv,lens", [(1, 20, 5, [1, 129, 700, 2500, 16]), (4, 8, 2, [4, 128, 1000, 131]),
                                          (130, 2, 1, [130, 257, 2000]), (20, 4, 2, [20, 640, 33])])
def test_ragged_error_is_near_that_of_f32(n, H, Hkv, lens):
    torch = need_cuda()
    att = importlib.import_module("0xbitnet_b200.attention")
    rng = np.random.default_rng(n)
    B, S = len(lens), max(lens)
    c, k, v = cache(torch, rng, B, S, Hkv)
    q = rng.standard_normal((B, n, H, D)).astype(np.float32)
    got = att.attention_q8(torch.from_numpy(q.reshape(B * n, -1)).cuda(), c, H, n,
                           torch.tensor(lens, dtype=torch.int32, device="cuda"))
    got = got.cpu().numpy().reshape(B, n, H, D)
    for b, L in enumerate(lens):
        want, tol = ref.attention_rms(q[b], k[b], v[b], L, SCALE)
        assert ratio(got[b], want, tol) <= 1, b
