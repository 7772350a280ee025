"""A BitNet decoder with 8-bit caches and logit rules: append, attention and rules as one run.

One step's logits against the oracle composition on the cache's own values (read back after the
step, so that the codes of the new position are the device's; their rounding has tests of its own),
within the end-to-end 2e-2 of the fp16 decoder's test. A run of steps at positions per sequence,
captured once and replayed, against the same calls made one by one: equal bit for bit.
"""
import importlib

import numpy as np
import pytest

import oracle as orc
from _util import need_cuda

pytestmark = pytest.mark.gpu


def dec():
    return importlib.import_module("0xbitnet_b200.decoder")


def rules_of(**kw):
    return importlib.import_module("0xbitnet_b200.logits").LogitRules(**kw)


def small(D_):
    return D_.DecoderConfig(layers=2, hidden=512, ffn=1024, heads=4, kv_heads=2, vocab=1000)


def oracle_logits(m, ids, values, pos):
    """The forward for one new token per sequence; values[layer] = (k, v) f32 [B, ctx, Hkv, d] of
    the caches after the step, pos[b] the token's position (-1: no token, no keys)."""
    cfg = m.cfg
    H, Hkv, d, D, F = cfg.heads, cfg.kv_heads, cfg.head_dim, cfg.hidden, cfg.ffn
    emb = m.embed.cpu().numpy()
    x = np.stack([emb[i] if i >= 0 else np.zeros(D, emb.dtype) for i in ids]).astype(np.float32)

    def lin(x, w, scales, rows, cols, norm):
        return orc.bitlinear_omp(x, w, scales, rows, cols, norm_w=norm.cpu().numpy(), eps=cfg.eps)

    for L, (k, v) in zip(m.layers, values):
        src = L.source
        sw = np.concatenate([np.full(n, s, np.float32) for n, s in
                             zip((H * d, Hkv * d, Hkv * d), L.qkv_scales)])
        qkv = lin(x, src["qkv"], sw, (H + 2 * Hkv) * d, D, L.attn_norm)
        a = np.zeros((len(ids), H * d), np.float32)
        for b, p in enumerate(pos):
            if p >= 0:
                q = orc.rope(qkv[b:b + 1, :H * d], H, d, p, cfg.rope_theta)
                a[b] = orc.attention(q, k[b, :p + 1].reshape(p + 1, -1),
                                     v[b, :p + 1].reshape(p + 1, -1), H, Hkv, d)[0]
        x = x + lin(a, src["o"], np.full(D, L.o_scale, np.float32), D, H * d, L.attn_sub_norm)
        gate = lin(x, src["gate"], np.full(F, L.gate_scale, np.float32), F, D, L.ffn_norm)
        up = lin(x, src["up"], np.full(F, L.up_scale, np.float32), F, D, L.ffn_norm)
        x = x + lin(orc.relu2_mul(gate, up), src["down"], np.full(D, L.down_scale, np.float32),
                    D, F, L.ffn_sub_norm)
    return orc.lm_head_f16(x.astype(np.float32), emb, m.final_norm.cpu().numpy(), cfg.eps)


@pytest.mark.parametrize("pos", [[10], [31, 31], [0, 15, 40, -1, 63]])
def test_step_matches_oracle(pos):
    torch = need_cuda()
    D_ = dec()
    B, ctx = len(pos), 64
    m = D_.BitNetDecoder(small(D_), B, ctx, seed=3, keep_source=True, kv_bits=8)
    m.fill_caches(ctx, seed=4)
    ids = [7, 999, 0, 5, 500][:B]
    m.ids.copy_(torch.tensor(ids, dtype=torch.int32))
    before = [c.read(0, ctx) for c in m.caches]
    same = len(set(pos)) == 1
    logits = m.step(pos[0] if same else torch.tensor(pos, dtype=torch.int32, device="cuda"))
    got = logits.cpu().numpy()
    values = [tuple(t.cpu().numpy() for t in c.read(0, ctx)) for c in m.caches]
    for (k0, v0), (k1, v1) in zip(before, values):
        for b, p in enumerate(pos):
            other = [i for i in range(ctx) if p < 0 or i // 16 != p // 16]
            assert np.array_equal(k0[b].cpu().numpy()[other], k1[b][other])
            assert np.array_equal(v0[b].cpu().numpy()[other], v1[b][other])
    err = np.abs(got - oracle_logits(m, ids, values, pos)).max()
    assert err <= 2e-2, err
    m.close()


def test_run_captured_and_replayed():
    """Steps and picks with positions, histories and a mask on the device: one captured iteration
    replayed against the calls made one by one, tokens, caches and logits bit for bit."""
    torch = need_cuda()
    D_ = dec()
    cfg, B, ctx, steps = small(D_), 3, 80, 6
    start = [5, 30, 0]
    m = D_.BitNetDecoder(cfg, B, ctx, seed=8, kv_bits=8)
    words = -(-cfg.vocab // 32)
    rng = np.random.default_rng(3)
    mask = torch.from_numpy(rng.integers(-2 ** 31, 2 ** 31, (B, words)).astype(np.int32)).cuda()
    rep = torch.tensor([1.0, 1.3, 2.0], device="cuda")
    pos = torch.empty(B, dtype=torch.int32, device="cuda")
    hist = torch.empty((B, steps), dtype=torch.int32, device="cuda")
    lens = torch.empty(B, dtype=torch.int32, device="cuda")
    rules = rules_of(repetition=rep, history=hist, history_lens=lens, mask=mask)
    stream = torch.cuda.Stream()

    def begin():
        for c in m.caches:
            for t in (c.k, c.v, c.k_scale, c.v_scale):
                t.zero_()
        m.fill_caches(40, seed=9)
        m.ids.copy_(torch.tensor([1, 2, 3], dtype=torch.int32))
        pos.copy_(torch.tensor(start, dtype=torch.int32))
        hist.fill_(-1)
        lens.zero_()

    def iteration():
        logits = m.step(pos)
        m.pick(logits, rules)
        hist.scatter_(1, lens.long().view(B, 1), m.ids.view(B, 1))
        pos.add_(1)
        lens.add_(1)
        return logits

    def run(call):
        begin()
        seen = []
        for i in range(steps):
            logits = call()
            seen.append((m.ids.cpu().numpy().copy(), logits.cpu().numpy().copy()))
        return seen, [t.cpu().numpy().copy() for c in m.caches
                      for t in (c.k, c.v, c.k_scale, c.v_scale)]

    with torch.cuda.stream(stream):
        eager, cache_eager = run(iteration)
        begin()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = iteration()

        def replay():
            g.replay()
            return out
        replayed, cache_replayed = run(replay)
        del g
    for (t0, l0), (t1, l1) in zip(eager, replayed):
        assert np.array_equal(t0, t1)
        assert np.array_equal(l0, l1)
        bits = mask.cpu().numpy().view(np.uint32)
        for b, t in enumerate(t0):
            assert bits[b, t // 32] >> (t % 32) & 1
            assert l0[b, t] == l0[b].max()
    for a, b in zip(cache_eager, cache_replayed):
        assert np.array_equal(a, b, equal_nan=True)
    m.close()


def test_refusals():
    torch = need_cuda()
    D_ = dec()
    with pytest.raises(ValueError):
        D_.BitNetDecoder(small(D_), 1, 16, kv_bits=4)
    m = D_.BitNetDecoder(small(D_), 1, 16)
    with pytest.raises(TypeError):
        m.step(torch.zeros(1, dtype=torch.int32, device="cuda"))
    m.close()
