"""GPU checks of attention over 8-bit caches whose value scales lie far apart, against the 64-bit
restatement and a bound by what adds up to each element (oracle/q8_ref.py). Query rows are one
number in dimension 0, so that key j's code there is the base-2 logarithm of its weight."""
import importlib

import numpy as np
import pytest

from _util import need_cuda
from oracle import q8_ref as ref

pytestmark = pytest.mark.gpu

D = 128
SCALE = float(np.float32(1.0) / np.sqrt(np.float32(D)))


def run_planted(torch, rng, n, H, Hkv, log2w, v_scale, B=1):
    """log2w [S] whole numbers up to 127, v_scale [blocks] -> asserts every output element, of B
    sequences alike, which are split among the CTAs at other places each."""
    att = importlib.import_module("0xbitnet_b200.attention")
    S, nb = len(log2w), len(v_scale)
    c = att.KVCacheQ8(B, S, Hkv, D)
    kc = rng.integers(-127, 128, (S, Hkv, D)).astype(np.int8)
    kc[:, :, 0] = np.asarray(log2w)[:, None]
    vc = rng.integers(-127, 128, (S, Hkv, D)).astype(np.int8)
    ks = np.ones((nb, Hkv), np.float32)
    vs = np.repeat(np.asarray(v_scale, np.float32)[:, None], Hkv, axis=1)
    for t, a in ((c.k, kc), (c.v, vc), (c.k_scale, ks), (c.v_scale, vs)):
        t.copy_(torch.from_numpy(a).unsqueeze(0))
    q = np.zeros((n, H, D), np.float32)
    q[:, :, 0] = np.log(2.0) / SCALE
    qd = torch.from_numpy(np.tile(q.reshape(n, H * D), (B, 1))).cuda()
    got = att.attention_q8(qd, c, H, n, S).cpu().numpy().reshape(B, n, H, D)
    wide = np.repeat(vs.astype(np.float64), ref.BLOCK, axis=0)[:S]
    want, bound = ref.attention_by_products(q, ref.values(kc, ks), ref.values(vc, vs), wide, S, SCALE)
    bad = ~(np.abs(got - want) <= bound)
    if bad.any():
        b, *at = np.argwhere(bad)[0]
        at = tuple(at)
        assert False, (b, at, got[(b, *at)], want[at], bound[at])


# few query rows (4, 8 and 16 to a tile), and many
ROWS = [(1, 2, 2), (4, 4, 2), (9, 2, 1), (40, 4, 2), (130, 2, 1)]


@pytest.mark.parametrize("n,H,Hkv", ROWS)
@pytest.mark.parametrize("S,B", [(150, 1), (700, 1), (700, 80), (3000, 1)])
@pytest.mark.parametrize("what", ["tiny_first", "tiny_last", "small_behind_large", "one_tiny_block"])
def test_two_scales(n, H, Hkv, S, B, what):
    """Equal weights on values of two magnitudes: every key counts in the total."""
    torch = need_cuda()
    rng = np.random.default_rng(S + n)
    nb = -(-S // ref.BLOCK)
    vs = np.full(nb, 2.0 ** 3)
    if what == "tiny_first":            # nothing above 1.5e-36 in the first unit of 128 keys
        vs[:8] = 2.0 ** -126
    elif what == "tiny_last":
        vs[nb // 2:] = 2.0 ** -126
    elif what == "small_behind_large":
        vs[:nb // 2] = 2.0 ** 100
        vs[nb // 2:] = 2.0 ** -40
    else:
        vs[nb // 3] = 2.0 ** -120
    run_planted(torch, rng, n, H, Hkv, np.zeros(S, np.int64), vs, B)


@pytest.mark.parametrize("n,H,Hkv", ROWS)
def test_large_scale_with_a_far_weight(n, H, Hkv):
    """Small values of nearly all the weight beside ordinary ones of a weight near 2^-110."""
    torch = need_cuda()
    rng = np.random.default_rng(n)
    for blk, exp, w in ((5, -6, -110), (0, -6, -110), (6, 100, -120), (11, 90, -105)):
        log2w = np.zeros(200, np.int64)
        log2w[16 * blk:16 * blk + 16] = w
        vs = np.full(13, 2.0 ** -106)
        vs[blk] = 2.0 ** exp
        run_planted(torch, rng, n, H, Hkv, log2w, vs)


@pytest.mark.parametrize("n,H,Hkv", ROWS)
@pytest.mark.parametrize("S,B", [(200, 1), (900, 1), (900, 60), (3000, 1)])
def test_scales_over_the_whole_range(n, H, Hkv, S, B):
    """Random value scales from 2^-126 to 2^100, some blocks of zeros; with random weights,
    and with weights that make the products alike."""
    torch = need_cuda()
    rng = np.random.default_rng(7 * S + n)
    nb = -(-S // ref.BLOCK)
    for kind in ("any", "alike", "flat"):
        e = rng.integers(-126, 101, nb)
        per_key = np.repeat(e, ref.BLOCK)[:S]
        log2w = {"any": rng.integers(-127, 128, S),
                 "alike": np.clip(-per_key - 13 + rng.integers(-8, 9, S), -127, 127),
                 "flat": np.zeros(S, np.int64)}[kind]
        vs = np.where(rng.random(nb) < 0.1, 0.0, np.exp2(e.astype(np.float64)))
        run_planted(torch, rng, n, H, Hkv, log2w, vs, B)


@pytest.mark.parametrize("n,H,Hkv", ROWS)
def test_zero_blocks_beside_small_values(n, H, Hkv):
    """Blocks of zeros with the largest weights take no bits from what is held beside them."""
    torch = need_cuda()
    rng = np.random.default_rng(n)
    for first, exp, w in ((0, -32, 0), (0, -126, -20), (-50, -120, 0), (3, 3, -30)):
        log2w = np.zeros(400, np.int64)
        vs = np.zeros(25)
        vs[1], vs[7], vs[20] = 2.0 ** first, 2.0 ** exp, 2.0 ** exp
        log2w[16:32] = -60
        log2w[7 * 16:8 * 16] = log2w[320:336] = w
        run_planted(torch, rng, n, H, Hkv, log2w, vs)
        run_planted(torch, rng, n, H, Hkv, log2w, vs, 70)


@pytest.mark.parametrize("n,H,Hkv", ROWS)
@pytest.mark.parametrize("exp", [105, -126])
def test_one_far_scale(n, H, Hkv, exp):
    """All values huge, or all tiny, over keys enough to be split among CTAs."""
    torch = need_cuda()
    rng = np.random.default_rng(n)
    for S, B in ((3000, 1), (1500, 30)):
        run_planted(torch, rng, n, H, Hkv, rng.integers(-20, 1, S),
                    np.full(-(-S // ref.BLOCK), 2.0 ** exp), B)


@pytest.mark.parametrize("n,H,Hkv", ROWS)
@pytest.mark.parametrize("S,B", [(150, 1), (700, 1), (700, 80), (3000, 1)])
@pytest.mark.parametrize("exp,rise", [(12, 20), (30, 40), (100, 120), (0, 100), (-20, 60)])
def test_large_values_before_larger_scores(n, H, Hkv, S, B, exp, rise):
    """The first block's values are 2^exp times the others', and the scores grow by `rise` binary
    digits along the keys: what was large against the first scores takes no bits from the rest."""
    torch = need_cuda()
    rng = np.random.default_rng(S + n + rise)
    nb = -(-S // ref.BLOCK)
    vs = np.exp2(rng.integers(-3, 4, nb).astype(np.float64))
    vs[0] *= 2.0 ** exp
    vs[nb // 2] = 0.0
    log2w = np.linspace(0, rise, S).astype(np.int64) + rng.integers(-2, 3, S)
    log2w[nb // 2 * ref.BLOCK:nb // 2 * ref.BLOCK + ref.BLOCK] += 7  # the weightiest have no values
    run_planted(torch, rng, n, H, Hkv, log2w, vs, B)


def any_scales(torch, rng, B, S, Hkv, k_exp, v_exp):
    """A cache whose scales are any numbers, no powers of two; its f64 values and value scales."""
    att = importlib.import_module("0xbitnet_b200.attention")
    nb = -(-S // ref.BLOCK)
    c = att.KVCacheQ8(B, S, Hkv, D)
    vals = []
    for codes, scale, (lo, hi) in ((c.k, c.k_scale, k_exp), (c.v, c.v_scale, v_exp)):
        cn = rng.integers(-127, 128, (B, S, Hkv, D)).astype(np.int8)
        sn = np.exp2(rng.uniform(lo, hi, (B, nb, Hkv))).astype(np.float32)
        codes.copy_(torch.from_numpy(cn))
        scale.copy_(torch.from_numpy(sn))
        vals.append(np.stack([ref.values(cn[b], sn[b]) for b in range(B)]))
    wide = np.repeat(sn.astype(np.float64), ref.BLOCK, axis=1)[:, :S]
    return c, vals[0], vals[1], wide


@pytest.mark.parametrize("B,n,H,Hkv,S", [(1, 1, 5, 1, 500), (2, 4, 8, 2, 300), (1, 9, 4, 2, 900),
                                         (1, 40, 4, 2, 300), (2, 130, 2, 1, 700), (30, 130, 2, 1, 900)])
@pytest.mark.parametrize("v_exp", [(-8, -4), (-100, -90), (-60, 60), (-126, -118)])
def test_scales_that_are_no_powers_of_two(B, n, H, Hkv, S, v_exp):
    """Wrapped buffers may hold any scales: each pass takes them as they are."""
    torch = need_cuda()
    att = importlib.import_module("0xbitnet_b200.attention")
    rng = np.random.default_rng(B + n + S)
    c, k, v, wide = any_scales(torch, rng, B, S, Hkv, (-8, -4), v_exp)
    q = rng.standard_normal((B * n, H * D)).astype(np.float32)
    got = att.attention_q8(torch.from_numpy(q).cuda(), c, H, n, S).cpu().numpy()
    for b in range(min(B, 3)):
        want, bound = ref.attention_by_products(q.reshape(B, n, H, D)[b], k[b], v[b], wide[b], S, SCALE)
        err = np.abs(got.reshape(B, n, H, D)[b] - want)
        assert np.all(err <= bound), (b, (err / bound).max())
