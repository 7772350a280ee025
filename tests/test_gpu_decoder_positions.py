"""A decoder with 8-bit caches and positions on the device: sequences that are idle or past the
end of their cache, eager and in a captured loop that runs into the end."""
import importlib

import numpy as np
import pytest

from _util import need_cuda

pytestmark = pytest.mark.gpu


def decoder(B, ctx, **kw):
    d = importlib.import_module("0xbitnet_b200.decoder")
    cfg = d.DecoderConfig(layers=2, hidden=512, ffn=1024, heads=4, kv_heads=2, vocab=1000)
    m = d.BitNetDecoder(cfg, B, ctx, kv_bits=8, **kw)
    m.fill_caches(ctx - 1, seed=2)
    return m


def no_rules():
    return importlib.import_module("0xbitnet_b200.logits").LogitRules()


def tokens(torch, m, pos, ids):
    m.ids.copy_(torch.tensor(ids, dtype=torch.int32))
    logits = m.step(torch.tensor(pos, dtype=torch.int32, device="cuda"))
    return m.pick(logits, no_rules()).cpu().tolist()


def state(m):
    return [t.cpu().numpy().copy() for c in m.caches for t in (c.k, c.v, c.k_scale, c.v_scale)]


@pytest.mark.parametrize("outside", [33, 34, 1 << 20, 2147483647, -1, -2, -2147483648])
def test_positions_outside_the_cache_take_no_part(outside):
    """No token, no change of the sequence's cache, nothing for the other sequences."""
    torch = need_cuda()
    ctx = 33
    m, alone = decoder(3, ctx, seed=5), decoder(3, ctx, seed=5)
    got = tokens(torch, m, [7, outside, 32], [3, 4, 5])
    want = tokens(torch, alone, [7, -1, 32], [3, 4, 5])
    assert got == want and got[1] == -1 and got[0] >= 0 and got[2] >= 0
    for a, b in zip(state(m), state(alone)):
        assert np.array_equal(a, b, equal_nan=True)
    # a step with one position for all has a token for all again
    m.ids.copy_(torch.tensor([1, 2, 3], dtype=torch.int32))
    assert min(m.pick(m.step(9), no_rules()).cpu().tolist()) >= 0
    m.close()
    alone.close()


def test_captured_loop_that_runs_past_the_end():
    """Positions counted up on the device: each sequence has tokens until its cache is full and
    -1 from then on, as the calls made one by one give them."""
    torch = need_cuda()
    ctx, start, steps = 20, [17, 12, 19], 6
    seen = []
    for captured in (False, True):
        m = decoder(3, ctx, seed=6)
        pos = torch.tensor(start, dtype=torch.int32, device="cuda")
        rules = no_rules()

        def iteration():
            m.pick(m.step(pos), rules)
            pos.add_(1)

        m.ids.copy_(torch.tensor([1, 2, 3], dtype=torch.int32))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        got = []
        with torch.cuda.stream(stream):
            if captured:
                before = state(m)
                iteration()  # warm-up, undone
                for t, a in zip([t for c in m.caches for t in (c.k, c.v, c.k_scale, c.v_scale)],
                                before):
                    t.copy_(torch.from_numpy(a))
                pos.copy_(torch.tensor(start, dtype=torch.int32))
                m.ids.copy_(torch.tensor([1, 2, 3], dtype=torch.int32))
                stream.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    iteration()
            for _ in range(steps):
                g.replay() if captured else iteration()
                got.append(m.ids.cpu().tolist())
            if captured:
                del g
        seen.append(got)
        m.close()
    assert seen[0] == seen[1]
    for i, row in enumerate(seen[0]):
        for b, t in enumerate(row):
            assert (t >= 0) == (start[b] + i < ctx), (i, b)


def test_refused_positions_change_nothing():
    torch = need_cuda()
    m = decoder(2, 20, seed=1)
    before = state(m)
    for bad, err in ((torch.zeros(3, dtype=torch.int32, device="cuda"), ValueError),
                     (torch.zeros(2, dtype=torch.int64, device="cuda"), TypeError),
                     (torch.zeros(2, dtype=torch.int32), TypeError)):
        with pytest.raises(err):
            m.step(bad)
    for a, b in zip(before, state(m)):
        assert np.array_equal(a, b)
    assert min(tokens(torch, m, [[3], [4]], [1, 2])) >= 0  # any shape of B elements
    m.close()


def test_replayed_steps_between_steps_for_all():
    """A captured step with positions on the device and eager ones with a position for all, in
    turn, each followed by an eager pick: what was called last counts."""
    torch = need_cuda()
    m, ctx = decoder(2, 20, seed=3), 20
    pos = torch.tensor([4, ctx], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        m.ids.copy_(torch.tensor([1, 2], dtype=torch.int32))
        m.step(pos)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = m.step(pos)
        for _ in range(2):
            assert min(m.pick(m.step(5), no_rules()).cpu().tolist()) >= 0
            m.ids.copy_(torch.tensor([1, 2], dtype=torch.int32))
            g.replay()
            got = m.pick(out, no_rules()).cpu().tolist()
            assert got[0] >= 0 and got[1] == -1
            m.ids.copy_(torch.tensor([1, 2], dtype=torch.int32))
        del g
    m.close()
