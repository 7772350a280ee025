"""GPU checks of the 8-bit KV cache: append, read-back and attention against 64-bit restatements.

Codes and scales are compared exactly (the kernels rotate and divide in f64; a code may go
either way only where its unrounded value is within 1e-9 of a half). q is off by at most three
f32 roundings of its pair. Attention is held to the bound that oracle/q8_ref.py derives.
"""
import numpy as np
import pytest

from _util import need_cuda
from oracle import q8_ref as ref

pytestmark = pytest.mark.gpu

D = 128
U = 2.0 ** -24
BASE = 500000.0


def att():
    import importlib
    return importlib.import_module("0xbitnet_b200.attention")


def host(cache):
    return [t.cpu().numpy() for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]


def random_cache(torch, rng, B, S_max, Hkv, sigma=1.0):
    """Device cache and its f64 values k, v [B, S_max, Hkv, D]."""
    nb = -(-S_max // ref.BLOCK)
    c = att().KVCacheQ8(B, S_max, Hkv, D)
    vals = []
    for codes, scale, sg in ((c.k, c.k_scale, sigma), (c.v, c.v_scale, 0.5)):
        cn = rng.integers(-127, 128, (B, S_max, Hkv, D)).astype(np.int8)
        sn = np.exp2(rng.integers(-8, -4, (B, nb, Hkv))).astype(np.float32) * np.float32(sg)
        codes.copy_(torch.from_numpy(cn))
        scale.copy_(torch.from_numpy(sn))
        vals.append(np.stack([ref.values(cn[b], sn[b]) for b in range(B)]))
    return c, vals[0], vals[1]


def check_append(torch, qkv, cache, H, n, pos, dev_pos):
    """One append against the oracle, started from the cache's current contents."""
    B, Hkv, S_max = cache.B, cache.Hkv, cache.S_max
    k0, ks0, v0, vs0 = [a.copy() for a in host(cache)]
    posv = [pos] * B if np.isscalar(pos) else list(pos)
    parg = torch.tensor(posv, dtype=torch.int32, device="cuda") if dev_pos else pos
    q = att().rope_kv_append_q8(torch.from_numpy(qkv).cuda(), cache, H, n, BASE, pos=parg)
    q = q.cpu().numpy().reshape(B, n, H, D)
    k1, ks1, v1, vs1 = host(cache)
    x = qkv.reshape(B, n, H + 2 * Hkv, D)
    for b in range(B):
        krows = np.zeros((n, Hkv, D))
        for t in range(n):
            p = posv[b] + t
            if not 0 <= p < S_max:
                assert not q[b, t].any()
                continue
            want = ref.rope(x[b, t, :H], p, BASE)
            pair = np.abs(x[b, t, :H]).reshape(H, D // 2, 2).sum(-1, keepdims=True)
            tol = np.broadcast_to(3 * U * pair, (H, D // 2, 2)).reshape(H, D) + 1e-44
            if np.isfinite(want).all():
                assert np.all(np.abs(q[b, t] - want) <= tol), (b, t)
            krows[t] = ref.rope(x[b, t, H:H + Hkv], p, BASE)
        vrows = x[b, :, H + Hkv:].astype(np.float64)
        for got, gs, c0, s0, rows in ((k1[b], ks1[b], k0[b], ks0[b], krows),
                                      (v1[b], vs1[b], v0[b], vs0[b], vrows)):
            want, ws = c0.astype(np.int64), s0.astype(np.float64)
            raw = ref.append(want, ws, rows, posv[b])
            assert np.array_equal(gs.astype(np.float64), ws, equal_nan=True), b
            with np.errstate(invalid="ignore"):
                half = np.abs(np.abs(raw - np.trunc(raw)) - 0.5) < 1e-9
            diff = np.abs(got.astype(np.int64) - want)
            assert not diff[~half].any(), (b, np.argwhere(diff * ~half)[:4])
            assert diff.max(initial=0) <= 1


@pytest.mark.parametrize("B,n,H,Hkv,pos,S_max,dev_pos", [
    (1, 1, 20, 5, 0, 1, False),              # the smallest cache
    (1, 1, 20, 5, 2047, 2048, False),        # the last row
    (2, 1, 8, 8, 16, 40, False),             # a block's first row
    (3, 1, 16, 2, [31, 0, 47], 50, True),    # lengths of their own, a cut last block
    (2, 5, 32, 4, 14, 33, False),            # across a block's end
    (1, 33, 14, 2, 0, 33, False),            # odd group, whole and cut blocks
    (2, 100, 12, 4, [3, 170], 300, True),
    (1, 300, 5, 1, 1001, 1301, False),
    (2, 7, 4, 1, [-3, -7], 20, True),        # left padding; nothing at all
    (4, 6, 4, 2, [18, 24, -40, 2147483640], 24, True),  # past the end, idle, far out
    (1, 2, 3, 1, 100001, 100005, False),     # far angles
    (2, 19, 40, 2, 3, 40, False),            # a large group
])
def test_append(B, n, H, Hkv, pos, S_max, dev_pos):
    torch = need_cuda()
    rng = np.random.default_rng(B * 1000 + n + H)
    cache, _, _ = random_cache(torch, rng, B, S_max, Hkv)
    qkv = (rng.standard_normal((B * n, (H + 2 * Hkv) * D)) *
           np.exp(rng.standard_normal((B * n, 1)))).astype(np.float32)
    check_append(torch, qkv, cache, H, n, pos, dev_pos)


def test_append_token_by_token_and_reread():
    """40 tokens one at a time, each larger than the one before: every scale change and
    requantization in turn; the values stay within one step of what was appended."""
    torch = need_cuda()
    rng = np.random.default_rng(1)
    H, Hkv, S_max = 4, 2, 45
    cache = att().KVCacheQ8(1, S_max, Hkv, D)
    kept = []
    for t in range(40):
        qkv = (rng.standard_normal((1, (H + 2 * Hkv) * D)) * 1.13 ** t).astype(np.float32)
        kept.append(qkv.reshape(H + 2 * Hkv, D)[H + Hkv:])
        check_append(torch, qkv, cache, H, 1, t, t % 2 == 1)
    k, v = cache.read(0, 40)
    scale = np.repeat(cache.v_scale.cpu().numpy()[0], ref.BLOCK, axis=0)[:40, :, None]
    assert np.all(np.abs(v.cpu().numpy()[0] - np.stack(kept)) <= scale)
    kn, ks, vn, vs = host(cache)
    assert np.array_equal(k.cpu().numpy()[0].astype(np.float64), ref.values(kn[0], ks[0])[:40])
    assert np.array_equal(v.cpu().numpy()[0].astype(np.float64), ref.values(vn[0], vs[0])[:40])


@pytest.mark.parametrize("what", ["zeros", "huge", "tiny", "nan", "inf", "border"])
def test_append_extreme_values(what):
    torch = need_cuda()
    rng = np.random.default_rng(5)
    H, Hkv, n = 2, 1, 5
    qkv = rng.standard_normal((n, (H + 2 * Hkv) * D)).astype(np.float32)
    if what == "zeros":
        qkv[:] = 0
    elif what == "huge":
        qkv *= np.float32(3e37)
    elif what == "tiny":
        qkv *= np.float32(1e-41)
    elif what in ("nan", "inf"):
        qkv[3, H * D + 7] = qkv[3, (H + Hkv) * D + 100] = np.nan if what == "nan" else -np.inf
    else:  # |x| at 127 * 2^e exactly and just above it, halves of a step
        qkv[:, (H + Hkv) * D:] = 0
        qkv[0, (H + Hkv) * D] = 127.0
        qkv[0, (H + Hkv) * D + 1:(H + Hkv) * D + 9] = np.arange(8) + 0.5
        qkv[2, (H + Hkv) * D] = np.nextafter(np.float32(127.0), np.float32(200.0))
    cache = att().KVCacheQ8(1, 40, Hkv, D)
    check_append(torch, qkv[:2], cache, H, 2, 12, False)   # 12, 13
    check_append(torch, qkv[2:], cache, H, 3, 14, False)   # 14, 15 and the next block's 16
    if what in ("nan", "inf"):  # row 3 is position 15: its block is poisoned, the next is not
        assert np.isnan(cache.k_scale.cpu().numpy()[0, 0, 0])
        assert np.isfinite(cache.v_scale.cpu().numpy()[0, 1, 0])
        check_append(torch, np.abs(qkv[:2]), cache, H, 2, 0, False)  # a block's start heals it
        assert np.isfinite(cache.k_scale.cpu().numpy()[0, 0, 0])


def test_read_windows():
    torch = need_cuda()
    rng = np.random.default_rng(2)
    cache, k, v = random_cache(torch, rng, 3, 37, 2)
    first = torch.tensor([-5, 20, 36], dtype=torch.int32, device="cuda")
    gk, gv = cache.read(first, 21)
    for b, f in enumerate([-5, 20, 36]):
        for i in range(21):
            p = f + i
            for got, want in ((gk, k), (gv, v)):
                row = got[b, i].cpu().numpy().astype(np.float64)
                assert np.array_equal(row, want[b, p] if 0 <= p < 37 else np.zeros_like(row))


def check_attention(torch, rng, B, n, H, Hkv, S, lens=None, sigma=1.0, qs=1.0, pad=5):
    S_max = max(S, 1) + pad
    cache, k, v = random_cache(torch, rng, B, S_max, Hkv, sigma)
    # what is behind each sequence's last block is never read
    Ls = [S] * B if lens is None else [min(max(x, 0), S_max) for x in lens]
    for b, L in enumerate(Ls):
        nb = -(-L // ref.BLOCK)
        cache.k_scale[b, nb:] = float("nan")
        cache.v_scale[b, nb:] = float("nan")
    q = (qs * rng.standard_normal((B * n, H * D))).astype(np.float32)
    arg = S if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = att().attention_q8(torch.from_numpy(q).cuda(), cache, H, n, arg)
    got = out.cpu().numpy().reshape(B, n, H, D)
    scale = float(np.float32(1.0) / np.sqrt(np.float32(D)))
    for b in range(B):
        want, bound = ref.attention(q.reshape(B, n, H, D)[b], k[b], v[b], Ls[b], scale)
        err = np.abs(got[b] - want).max(-1)
        assert np.all(err <= bound), (b, (err / np.maximum(bound, 1e-30)).max())


@pytest.mark.parametrize("B,n,H,Hkv,S", [
    (1, 1, 20, 5, 1), (1, 1, 20, 5, 2048), (2, 1, 8, 8, 15), (3, 1, 16, 2, 129),
    (1, 1, 3, 1, 33), (1, 1, 14, 2, 500), (5, 1, 5, 1, 64), (1, 1, 4, 4, 40000),
    (64, 1, 20, 5, 700), (2, 2, 20, 5, 300), (1, 3, 12, 4, 257), (2, 4, 32, 4, 1000),
    (1, 7, 8, 8, 7), (1, 5, 16, 2, 3), (2, 17, 4, 2, 140), (1, 24, 5, 5, 3000),
    (1, 33, 20, 5, 33), (2, 40, 8, 1, 200), (1, 130, 4, 1, 260), (1, 128, 16, 8, 1025),
    (1, 300, 6, 2, 400), (2, 257, 4, 4, 511), (1, 512, 20, 5, 512),
    # several pairs and many units to a CTA: parts, drained sums, staging reused
    (40, 300, 4, 1, 700), (150, 64, 2, 2, 640), (1, 512, 20, 5, 2100), (3, 260, 8, 2, 3000),
    (90, 2, 12, 4, 2000), (300, 1, 8, 8, 400), (60, 4, 16, 4, 1500),
    # one KV head for many query heads; rows on both sides of the passes' border
    (2, 1, 20, 1, 300), (1, 1, 71, 1, 500), (1, 3, 24, 2, 700), (3, 16, 4, 1, 90), (1, 13, 5, 1, 333),
    (2, 4, 48, 3, 150),
])
def test_attention(B, n, H, Hkv, S):
    torch = need_cuda()
    check_attention(torch, np.random.default_rng(B + n + H + S), B, n, H, Hkv, S)


@pytest.mark.parametrize("n,H,Hkv,lens", [
    (1, 20, 5, [0, 1, 16, 17, 700, 128, 0]),
    (1, 8, 1, [3000, 5, 0]),
    (4, 20, 5, [2, 0, 4, 333]),              # left padding: rows before the first token
    (20, 4, 2, [7, 0, 500, 20]),
    (130, 4, 1, [129, 0, 400]),
    (1, 4, 4, [-3, 1 << 30, 9]),             # brought into [0, S_max]
])
def test_attention_ragged(n, H, Hkv, lens):
    torch = need_cuda()
    S = max(min(x, 4000) for x in lens)
    check_attention(torch, np.random.default_rng(n + H), len(lens), n, H, Hkv, S, lens)


@pytest.mark.parametrize("n,H,S", [(1, 4, 0), (8, 4, 3), (40, 4, 0), (300, 4, 7), (520, 2, 100)])
def test_attention_host_length_shorter_than_the_pass(n, H, S):
    """Rows before the first position, whole tiles of them too, are zeros."""
    torch = need_cuda()
    rng = np.random.default_rng(n + S)
    cache, k, v = random_cache(torch, rng, 2, 128, 1)
    q = rng.standard_normal((2 * n, H * D)).astype(np.float32)
    out = torch.full((2 * n, H * D), float("nan"), device="cuda")
    att().attention_q8(torch.from_numpy(q).cuda(), cache, H, n, S, out=out)
    got = out.cpu().numpy().reshape(2, n, H, D)
    for b in range(2):
        want, bound = ref.attention(q.reshape(2, n, H, D)[b], k[b], v[b], S, D ** -0.5)
        assert np.all(got[b][:n - S] == 0)
        assert np.all(np.abs(got[b] - want).max(-1) <= bound)


@pytest.mark.parametrize("n,S", [(1, 900), (3, 900), (64, 300)])
@pytest.mark.parametrize("qs,sigma", [(0.0, 1.0), (30.0, 4.0), (1e-6, 1.0), (1e5, 2.0 ** -10),
                                      (1.0, 2.0 ** -100)])
def test_attention_score_ranges(n, S, qs, sigma):
    """Flat and one-hot rows, tiny and large queries, far scales."""
    torch = need_cuda()
    check_attention(torch, np.random.default_rng(n), 1, n, 8, 2, S, qs=qs, sigma=sigma)


@pytest.mark.parametrize("n", [1, 4, 64])
def test_attention_large_values_of_small_weight(n):
    """A block of values 2^24 times the others', with weights below 2^-60, takes no bits from
    them: the bound counts only the others and the block's own share."""
    torch = need_cuda()
    rng = np.random.default_rng(n)
    S, H, Hkv = 200, 4, 2
    cache, k, v = random_cache(torch, rng, 1, S, Hkv)
    q = np.abs(rng.standard_normal((n, H * D))).astype(np.float32) + np.float32(0.5)
    codes = cache.k.view(1, -1, Hkv, D)
    codes[:, 64:80] = -127
    cache.k_scale[:, 4] = 2.0 ** -3
    k[:, 64:80] = -127 * 2.0 ** -3
    cache.v_scale[:, 4] = cache.v_scale[:, 4] * 2.0 ** 24
    v[:, 64:80] *= 2.0 ** 24
    out = att().attention_q8(torch.from_numpy(q).cuda(), cache, H, n, S)
    got = out.cpu().numpy().reshape(n, H, D)
    scale = float(np.float32(1.0) / np.sqrt(np.float32(D)))
    want, _ = ref.attention(q.reshape(n, H, D), k[0], v[0], S, scale)
    rest = v[0].copy()
    rest[64:80] = 0
    _, bound = ref.attention(q.reshape(n, H, D), k[0], rest, S, scale)
    assert np.all(np.abs(got - want).max(-1) <= bound)


@pytest.mark.parametrize("n", [1, 4, 64])
def test_attention_zero_and_poisoned_blocks(n):
    """A block of zeros counts with its weight; a NaN scale reaches only the rows that see it."""
    torch = need_cuda()
    rng = np.random.default_rng(n)
    S, H, Hkv = 200, 4, 2
    cache, k, v = random_cache(torch, rng, 1, S, Hkv)
    cache.k_scale[:, 2] = 0
    cache.v_scale[:, 4] = 0
    k[:, 32:48] = 0
    v[:, 64:80] = 0
    q = rng.standard_normal((n, H * D)).astype(np.float32)
    qd = torch.from_numpy(q).cuda()
    got = att().attention_q8(qd, cache, H, n, S).cpu().numpy().reshape(n, H, D)
    want, bound = ref.attention(q.reshape(n, H, D), k[0], v[0], S, D ** -0.5)
    assert np.all(np.abs(got - want).max(-1) <= bound)
    for t in (cache.v_scale, cache.k_scale):
        keep = t.clone()
        t[0, 12, 0] = float("nan")  # positions 192 .. 199, KV head 0
        got2 = att().attention_q8(qd, cache, H, n, S).cpu().numpy().reshape(n, H, D)
        lim = S - n + np.arange(n) + 1
        hit = (lim > 192)[:, None] & (np.arange(H) < H // Hkv)
        assert np.isnan(got2[hit]).all() and np.array_equal(got2[~hit], got[~hit])
        t.copy_(keep)
    bad = qd.clone()
    bad[n - 1, 5] = float("inf")
    got3 = att().attention_q8(bad, cache, H, n, S).cpu().numpy().reshape(n, H, D)
    assert np.isnan(got3[n - 1, 0]).all()
    assert np.array_equal(got3[n - 1, 1:], got[n - 1, 1:])
    assert np.array_equal(got3[:n - 1], got[:n - 1])


@pytest.mark.parametrize("n,B", [(1, 1), (1, 9), (4, 2), (64, 1)])
def test_decode_run_captured_and_on_streams(n, B):
    """Append, then attention, as a decode loop uses them: on a side stream, captured once with
    device positions and lengths and replayed at later positions, against eager calls; results
    repeat bit for bit, and nothing behind the outputs is written."""
    torch = need_cuda()
    rng = np.random.default_rng(n + B)
    H, Hkv, S_max, steps = 8, 2, 900, 3
    start = [int(x) for x in rng.integers(0, S_max - steps * n, B)]
    c1, _, _ = random_cache(torch, rng, B, S_max, Hkv)
    c2 = att().KVCacheQ8.wrap(c1.k.clone(), c1.k_scale.clone(), c1.v.clone(), c1.v_scale.clone())
    qkvs = [torch.from_numpy(rng.standard_normal((B * n, (H + 2 * Hkv) * D)).astype(np.float32))
            .cuda() for _ in range(steps)]
    want = []
    pos = torch.tensor(start, dtype=torch.int32, device="cuda")
    for i in range(steps):
        q = att().rope_kv_append_q8(qkvs[i], c1, H, n, pos=pos + i * n)
        want.append(att().attention_q8(q, c1, H, n, pos + (i + 1) * n).clone())
        again = att().attention_q8(q, c1, H, n, pos + (i + 1) * n)
        assert torch.equal(want[-1], again)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    qkv, p, L = qkvs[0].clone(), pos.clone(), pos + n
    buf = torch.full((B * n * H * D + 64,), 7.0, device="cuda")
    out = buf[:B * n * H * D].view(B * n, H * D)
    ws = att().attention_q8_workspace(c2, H, n)
    qb = torch.empty((B * n, H * D), device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        att().rope_kv_append_q8(qkv, c2, H, n, pos=p, q_out=qb)   # warm-up of step 0
        att().attention_q8(qb, c2, H, n, L, out=out, workspace=ws)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            att().rope_kv_append_q8(qkv, c2, H, n, pos=p, q_out=qb)
            att().attention_q8(qb, c2, H, n, L, out=out, workspace=ws)
        for i in range(steps):
            qkv.copy_(qkvs[i])
            p.copy_(pos + i * n)
            L.copy_(pos + (i + 1) * n)
            out.fill_(float("nan"))
            g.replay()
            side.synchronize()
            assert torch.equal(out, want[i]), i
    del g
    assert torch.equal(c1.k, c2.k) and torch.equal(c1.v_scale, c2.v_scale)
    assert bool((buf[B * n * H * D:] == 7.0).all())


def test_long_cache_offsets():
    """Offsets past 2^31 elements: 3 sequences of 800,000 positions of 8 KV heads."""
    torch = need_cuda()
    B, S_max, Hkv, H = 3, 800_000, 8, 8
    cache = att().KVCacheQ8(B, S_max, Hkv, D)
    rng = np.random.default_rng(4)
    n = 50
    qkv = rng.standard_normal((B * n, (H + 2 * Hkv) * D)).astype(np.float32)
    pos = S_max - n
    q = att().rope_kv_append_q8(torch.from_numpy(qkv).cuda(), cache, H, n, BASE, pos=pos)
    k, v = cache.read(pos, n)
    vr = qkv.reshape(B, n, H + 2 * Hkv, D)[:, :, H + Hkv:]
    scale = np.repeat(cache.v_scale[:, pos // 16:].cpu().numpy(), 16, axis=1)
    scale = scale[:, pos % 16:][:, :n, :, None]
    assert np.all(np.abs(v.cpu().numpy() - vr) <= scale / 2)
    # every earlier row is zero: a score of 0 and a value of 0
    for m in (1, n):
        qd = q.view(B, n, H, D)[:, n - m:].reshape(B * m, H * D).contiguous()
        got = att().attention_q8(qd, cache, H, m, S_max).cpu().numpy().reshape(B, m, H, D)
        kv, vv, qn = k.double().cpu().numpy(), v.double().cpu().numpy(), qd.cpu().numpy()
        qn = qn.reshape(B, m, H, D).astype(np.float64)
        for b in range(B):
            for t in range(m):
                seen = n - m + t + 1
                s = np.einsum("shd,hd->hs", kv[b, :seen], qn[b, t]) * D ** -0.5
                top = np.maximum(s.max(-1), 0)[:, None]
                e = np.exp(s - top)
                total = e.sum(-1, keepdims=True) + pos * np.exp(-top)
                want = np.einsum("hs,shd->hd", e, vv[b, :seen]) / total
                # 2^-24 for each of up to 800,000 / 128 sums of a lane, worst case
                tol = np.abs(want) * (U * S_max / 32 + 1e-5) + 1e-9
                assert np.all(np.abs(got[b, t] - want) <= tol), (m, b, t)
