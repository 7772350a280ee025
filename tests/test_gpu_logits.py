"""GPU checks of the logit rules against a 64-bit restatement: changed values are computed in
f64 and rounded once (half a step, 2^-24, plus what the order of f64 sums leaves), the others
pass bit for bit, and the greedy token is the lowest index of the largest result."""
import importlib

import numpy as np
import pytest

from _util import need_cuda
from oracle import q8_ref as ref

pytestmark = pytest.mark.gpu


def mod():
    return importlib.import_module("0xbitnet_b200.logits")


def pack(mask):
    """[rows, V] bool -> int32 words [rows, ceil(V / 32)]."""
    rows, V = mask.shape
    bits = np.zeros((rows, -(-V // 32) * 32), np.uint8)
    bits[:, :V] = mask
    return np.packbits(bits, axis=1, bitorder="little").view("<i4")


def greedy(row):
    ok = np.where(np.isnan(row), -np.inf, row)
    return int(np.argmax(ok)) if ok.max() > -np.inf else -1


def check(got, token, x, want):
    for r in range(x.shape[0]):
        same = want[r] == x[r].astype(np.float64)
        assert np.array_equal(got[r][same], x[r][same]), r
        fin = np.isfinite(want[r])
        assert np.array_equal(got[r][~fin].astype(np.float64), want[r][~fin], equal_nan=True), r
        err = np.abs(got[r][fin] - want[r][fin])
        assert np.all(err <= 2.0 ** -24 * (1 + 1e-6) * np.abs(want[r][fin]) + 1e-12), r
        assert token[r] == greedy(got[r]), r


@pytest.mark.parametrize("R,V,hist,nb,masked,shared", [
    (1, 1, 1, 1, True, False), (1, 128256, 64, 16, True, False), (3, 31, 5, 2, True, True),
    (5, 1003, 700, 40, True, False), (2, 32003, 4096, 300, True, True),
    (70, 4097, 9, 0, False, False), (4, 50000, 0, 0, True, False), (2, 129, 0, 1024, False, True),
    (3, 8192, 65535, 1024, True, False), (2, 200001, 100, 3, True, False),
    (300, 257, 3, 3, True, True), (2, 7, 0, 0, False, False),
])
def test_rules(R, V, hist, nb, masked, shared):
    torch = need_cuda()
    rng = np.random.default_rng(R + V + hist)
    x = (3 * rng.standard_normal((R, V))).astype(np.float32)
    cu = lambda a: torch.from_numpy(a).cuda()
    kw, args = {}, [dict() for _ in range(R)]
    if hist:
        h = (V * 1.05 * rng.random((R, hist)) ** 3).astype(np.int32) - rng.integers(0, 2, (R, hist))
        h = h.astype(np.int32)   # some ids outside the vocabulary on both sides
        hl = rng.integers(0, hist + 1, R).astype(np.int32)
        hl[0] = hist
        rep = (1 + rng.random(R) * (0.5 if hist < 5000 else 1e-3)).astype(np.float32)
        fr, pr = rng.random((2, R)).astype(np.float32)
        kw.update(history=cu(h), history_lens=cu(hl), repetition=cu(rep), frequency=cu(fr),
                  presence=cu(pr))
        for r in range(R):
            args[r].update(history=h[r, :hl[r]].tolist(), repetition=rep[r], frequency=fr[r],
                           presence=pr[r])
    if nb:
        rows = 1 if shared else R
        ids = rng.integers(-1, V + 1, (rows, nb)).astype(np.int32)
        ids[:, nb // 2:] = ids[:, :nb - nb // 2]       # ids that occur twice
        val = rng.standard_normal((rows, nb)).astype(np.float32)
        val[0, 0] = -np.inf
        bl = rng.integers(0, nb + 1, R).astype(np.int32)
        kw.update(bias_ids=cu(ids), bias_values=cu(val), bias_lens=cu(bl))
        for r in range(R):
            m = r % rows
            args[r]["bias"] = list(zip(ids[m, :bl[r]].tolist(), val[m, :bl[r]].tolist()))
    if masked:
        rows = 1 if shared else R
        mask = rng.random((rows, V)) < rng.random((rows, 1))
        kw["mask"] = cu(pack(mask))
        for r in range(R):
            args[r]["mask"] = mask[r % rows]
    out, token = mod().logits_process(cu(x), mod().LogitRules(**kw))
    want = [ref.logits(x[r], **args[r]) for r in range(R)]
    check(out.cpu().numpy(), token.cpu().numpy(), x, want)


def test_single_occurrence_equals_the_sampler():
    """One occurrence gives the sampler's f32 quotient or product (sampling.rs:14-27)."""
    torch = need_cuda()
    rng = np.random.default_rng(3)
    V = 5000
    x = (8 * rng.standard_normal((1, V))).astype(np.float32)
    ids = rng.permutation(V)[:900].astype(np.int32)
    pen = np.float32(1.1)
    r = mod().LogitRules(repetition=torch.full((1,), 1.1, device="cuda"),
                         history=torch.from_numpy(ids).cuda())
    out, _ = mod().logits_process(torch.from_numpy(x).cuda(), r)
    want = x.copy()
    want[0, ids] = np.where(x[0, ids] > 0, x[0, ids] / pen, x[0, ids] * pen)
    assert np.array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("rep", [2.0, 0.5])
def test_powers_beyond_the_range(rep):
    """Thousands of occurrences: as dividing or multiplying once for each gives it."""
    torch = need_cuda()
    V, n = 40, 3000
    x = np.array([0.0, -0.0, 3.0, -3.0, np.inf, -np.inf, 1e-40, -1e-40], np.float32)
    row = np.zeros((1, V), np.float32)
    row[0, :8] = x
    r = mod().LogitRules(repetition=torch.full((1,), rep, device="cuda"),
                         frequency=torch.full((1,), 0.5, device="cuda"),
                         history=torch.arange(8, dtype=torch.int32, device="cuda").repeat(n))
    out, _ = mod().logits_process(torch.from_numpy(row).cuda(), r)
    want = x.astype(np.float64)
    with np.errstate(over="ignore", under="ignore"):
        for _ in range(n):
            want = np.where(want > 0, want / rep, want * rep)
        want = (want - 0.5 * n).astype(np.float32)
    assert np.array_equal(out.cpu().numpy()[0, :8], want)


def test_special_values_ties_and_empty_rows():
    torch = need_cuda()
    V = 3001
    x = np.zeros((6, V), np.float32)
    x[1] = -np.inf                                   # nothing to pick
    x[2, [77, 2500, 5]] = np.inf, np.inf, 9.0        # an infinity, twice
    x[3, :] = np.nan                                 # nothing that compares
    x[4, 100:] = np.nan
    x[4, 50] = 1.0
    x[5] = np.finfo(np.float32).min                  # the type's lowest value is above -inf
    mask = np.ones((6, V), bool)
    mask[0] = False                                  # a grammar that leaves nothing
    mask[3, :7] = False
    r = mod().LogitRules(mask=torch.from_numpy(pack(mask)).cuda())
    out, token = mod().logits_process(torch.from_numpy(x).cuda(), r)
    want = np.where(mask, x, -np.inf)
    assert np.array_equal(out.cpu().numpy(), want, equal_nan=True)
    assert token.cpu().tolist() == [-1, -1, 77, -1, 50, 0]
    tie = np.zeros((2, V), np.float32)
    tie[:, 3000] = tie[:, 1234] = tie[:, 1299] = 4.0
    _, token = mod().logits_process(torch.from_numpy(tie).cuda(), mod().LogitRules())
    assert token.cpu().tolist() == [1234, 1234]


def test_in_place_captured_and_on_a_side_stream():
    """In place, replayed with a history that grows between the replays, as a decode loop does
    it; against eager calls."""
    torch = need_cuda()
    rng = np.random.default_rng(8)
    R, V, cap = 3, 9999, 50
    x = torch.from_numpy((3 * rng.standard_normal((R, V))).astype(np.float32)).cuda()
    hist = torch.full((R, cap), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    rules = mod().LogitRules(repetition=torch.full((R,), 1.3, device="cuda"),
                             frequency=torch.full((R,), 0.5, device="cuda"), history=hist,
                             history_lens=lens)
    buf = torch.full((R * V + 9,), 5.0, device="cuda")
    y, tok = buf[:R * V].view(R, V), torch.empty(R, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y.copy_(x)
        mod().logits_process(y, rules, out=y, token=tok)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            y.copy_(x)
            mod().logits_process(y, rules, out=y, token=tok)
        for step in range(20):
            g.replay()
            side.synchronize()
            want, wt = mod().logits_process(x, rules)
            assert torch.equal(y, want) and torch.equal(tok, wt), step
            for r in range(R):
                hist[r, step] = tok[r]
            lens += 1
            side.synchronize()
    del g
    # a token picked again and again is pushed down until others win
    assert len(set(hist[0, :20].cpu().tolist())) > 1
    assert bool((buf[R * V:] == 5.0).all())
