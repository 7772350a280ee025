"""The cases of the 8-bit KV cache and of the logit rules: their inputs, plain forms and exact values.

Three operators of the decode path:

* append: RoPE of q and k and the append of k and v to a cache held in 8 bits, with one
  power-of-two scale for each block of 16 positions and KV head (``rope_kv_append_q8``),
  followed by the read-back of the rows it touched (``KVCacheQ8.read``);
* attend: causal grouped-query attention over that cache (``attention_q8``), from one new
  token per sequence to prefill chunks, with a length of its own for each sequence;
* logits: repetition, frequency and presence penalties, sparse biases and a grammar's bit
  mask on each row of the logits, and the row's greedy token (``logits_process``).

With ``own`` false every operator is computed by elementary torch operations.
"""
import importlib
import math

import torch

own = False
DEVICE = "cuda"
D = 128       # head size of the framework's attention
BLOCK = 16    # positions that share a scale
THETA = 500000.0


# ---- cases ------------------------------------------------------------------------------

def listed():
    return [
        # one conversation, one decode step (the 2B decoder's heads): latency
        dict(name="append-1", op="append", B=1, n=1, H=20, Hkv=5, pos=2047, ragged=False),
        # a full decode batch, every sequence at a position of its own
        dict(name="append-64", op="append", B=64, n=1, H=20, Hkv=5, pos=2000, ragged=True),
        # a long prompt's prefill chunk behind an earlier chunk that ended inside a block
        dict(name="append-2048", op="append", B=1, n=2048, H=20, Hkv=5, pos=1001, ragged=False),
        # one conversation, one decode step at the decoder benchmark's context: latency
        dict(name="attend-1", op="attend", B=1, n=1, H=20, Hkv=5, S=2048, ragged=False),
        # a full decode batch of conversations of every length up to 4095
        dict(name="attend-64", op="attend", B=64, n=1, H=20, Hkv=5, S=4095, ragged=True),
        # one very long document: work has to be split along the keys
        dict(name="attend-long", op="attend", B=1, n=1, H=20, Hkv=5, S=131072, ragged=False),
        # a few drafted tokens checked at once, eight query heads to a KV head
        dict(name="attend-draft", op="attend", B=8, n=4, H=32, Hkv=4, S=5000, ragged=True),
        # the model's prefill chunk over a context that is already there
        dict(name="attend-512", op="attend", B=1, n=512, H=20, Hkv=5, S=2100, ragged=False),
        # a long prompt in one piece behind an earlier one
        dict(name="attend-2048", op="attend", B=1, n=2048, H=20, Hkv=5, S=6144, ragged=False),
        # one conversation with a penalty window and a grammar: latency
        dict(name="logits-1", op="logits", R=1, V=128256, hist=64, bias=16, mask="rows"),
        # a decode batch with long histories, a grammar for each row
        dict(name="logits-64", op="logits", R=64, V=128256, hist=4096, bias=300, mask="rows"),
        # a large batch over a vocabulary whose rows end at odd addresses, one shared mask
        dict(name="logits-250", op="logits", R=250, V=32003, hist=513, bias=33, mask="shared"),
    ]


HEADS = [(20, 5), (32, 4), (8, 8), (16, 2), (12, 4), (16, 8), (4, 1), (14, 2), (5, 1)]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logits"])
    if op == "logits":
        V = _between(rng, 1000, 160000)
        R = _between(rng, 1, max(1, min(256, 8_000_000 // V)))
        return dict(op=op, R=R, V=V, hist=rng.choice([0, _between(rng, 1, 4096)]),
                    bias=rng.choice([0, _between(rng, 1, 300)]),
                    mask=rng.choice(["none", "rows", "shared"]))
    H, Hkv = rng.choice(HEADS)
    if op == "append":
        n = rng.choice([1, _between(rng, 1, 2048)])
        B = _between(rng, 1, max(1, min(64, 2048 * 20 // (n * H))))
        pos = _between(rng, 1, 4000 if B > 1 else 100000) - 1
        return dict(op=op, B=B, n=n, H=H, Hkv=Hkv, pos=pos, ragged=rng.random() < 0.5)
    kind = rng.choice(["decode", "decode", "few", "chunk"])
    if kind == "decode":
        n, B = 1, _between(rng, 1, 64)
        S = _between(rng, 1, max(64, min(131072, 64 * 4095 * 5 // (B * Hkv))))
    elif kind == "few":
        n = rng.randint(2, 24)
        B = _between(rng, 1, 16)
        S = n + _between(rng, 1, max(64, min(30000, 8 * 5000 * 32 // (B * H))))
    else:
        n = _between(rng, 25, 2048)
        S = n + _between(rng, 1, 4096) - 1
        B = max(1, min(4, 2048 * 4096 * 20 // (n * S * H)))
    return dict(op=op, B=B, n=n, H=H, Hkv=Hkv, S=S, ragged=rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)


def _cache(g, B, S, Hkv, sigma):
    """A cache of S positions (of which a block may be cut short by the end): int8 codes and
    block scales of rows with a few strong channels, as keys and values have."""
    blocks = -(-S // BLOCK)
    x = _normal(g, B, blocks * BLOCK, Hkv, D) * sigma
    x *= torch.exp(0.5 * _normal(g, 1, 1, Hkv, D))
    x = x.view(B, blocks, BLOCK, Hkv, D)
    amax = x.abs().amax(dim=(2, 4))
    scale = torch.exp2(torch.ceil(torch.log2(amax.double() / 127))).float()
    codes = torch.round(x / scale[:, :, None, :, None]).clamp_(-127, 127).to(torch.int8)
    return codes.view(B, blocks * BLOCK, Hkv, D)[:, :S].contiguous(), scale.contiguous()


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "logits":
        R, V = c["R"], c["V"]
        s = dict(case=c, logits=3 * _normal(g, R, V))
        u = torch.rand((3, R), generator=g, device=DEVICE)
        s["repetition"] = 1 + 0.5 * u[0]
        s["frequency"] = 0.7 * u[1]
        s["presence"] = 0.7 * u[2]
        if c["hist"]:
            # ids drawn with many repeats; each row's window has a length of its own
            u = torch.rand((R, c["hist"]), generator=g, device=DEVICE)
            s["history"] = (V * u ** 3).to(torch.int32).clamp_(max=V - 1)
            s["history_lens"] = torch.randint(c["hist"] // 2, c["hist"] + 1, (R,), generator=g,
                                              device=DEVICE, dtype=torch.int32)
        if c["bias"]:
            s["bias_ids"] = torch.randint(0, V, (R, c["bias"]), generator=g, device=DEVICE,
                                          dtype=torch.int32)
            s["bias_values"] = 2 * _normal(g, R, c["bias"])
        if c["mask"] != "none":
            rows, words = (R if c["mask"] == "rows" else 1), -(-V // 32)
            # grammars allow from almost nothing to almost everything
            keep = torch.rand((rows, 1, 1), generator=g, device=DEVICE) ** 2
            bits = torch.rand((rows, words, 32), generator=g, device=DEVICE) < keep
            bits[:, 0, 0] = True
            word = (bits.long() << torch.arange(32, device=DEVICE)).sum(-1)
            s["mask"] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)
        return s
    B, n, H, Hkv = c["B"], c["n"], c["H"], c["Hkv"]
    if c["op"] == "append":
        top = c["pos"] + n
        s = dict(case=c, S_max=top + 7)
        s["k"], s["v"] = _cache(g, B, s["S_max"], Hkv, 1.0), _cache(g, B, s["S_max"], Hkv, 0.5)
        qkv = _normal(g, B * n, H + 2 * Hkv, D)
        qkv[:, H + Hkv:] *= 0.5
        s["qkv"] = qkv.view(B * n, -1)
        if c["ragged"]:
            s["pos"] = torch.randint(0, c["pos"] + 1, (B,), generator=g, device=DEVICE,
                                     dtype=torch.int32)
            s["pos"][0] = c["pos"]
        # the first row of the block in which each sequence's append begins
        s["first"] = (s["pos"] // BLOCK * BLOCK) if c["ragged"] else c["pos"] // BLOCK * BLOCK
        s["rows"] = -(-(n + BLOCK - 1) // BLOCK) * BLOCK
        return s
    s = dict(case=c, S_max=c["S"] + 5)
    s["k"], s["v"] = _cache(g, B, s["S_max"], Hkv, 1.0), _cache(g, B, s["S_max"], Hkv, 0.5)
    s["q"] = 1.5 * _normal(g, B * n, H * D)
    if c["ragged"]:
        s["lens"] = torch.randint(n, c["S"] + 1, (B,), generator=g, device=DEVICE,
                                  dtype=torch.int32)
        s["lens"][0] = c["S"]
    return s


# ---- one pass -----------------------------------------------------------------------------

def run(s):
    return {"append": _append, "attend": _attend, "logits": _logits}[s["case"]["op"]](s)


def _kept(s):
    """The cache object that a program keeps, over the state's buffers."""
    if "cache" not in s:
        att = importlib.import_module("0xbitnet_b200.attention")
        s["cache"] = att.KVCacheQ8.wrap(*s["k"], *s["v"])
    return s["cache"]


def _append(s):
    c = s["case"]
    if own:
        att = importlib.import_module("0xbitnet_b200.attention")
        cache = _kept(s)
        q = att.rope_kv_append_q8(s["qkv"], cache, c["H"], c["n"], THETA,
                                  pos=s["pos"] if c["ragged"] else c["pos"])
        k, v = cache.read(s["first"], s["rows"])
        return dict(q=q, k=k, v=v)
    B, n, H, Hkv, W = c["B"], c["n"], c["H"], c["Hkv"], s["rows"]
    pos = s["pos"].long() if c["ragged"] else torch.full((B,), c["pos"], device=DEVICE)
    # RoPE in 64 bits: far positions have large angles, and codes sit next to borders
    x = s["qkv"].view(B, n, H + 2 * Hkv, D)
    p = pos[:, None] + torch.arange(n, device=DEVICE)
    freq = THETA ** (-torch.arange(0, D, 2, device=DEVICE, dtype=torch.float64) / D)
    ang = p[:, :, None, None].double() * freq
    cos, sin = torch.cos(ang), torch.sin(ang)
    a, b = x[:, :, :H + Hkv, 0::2].double(), x[:, :, :H + Hkv, 1::2].double()
    rot = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).view(B, n, H + Hkv, D)
    first = pos // BLOCK * BLOCK
    rows = first[:, None] + torch.arange(W, device=DEVICE)          # positions of the window
    at = rows.clamp(max=s["S_max"] - 1)
    seq = torch.arange(B, device=DEVICE)[:, None]
    blocks = W // BLOCK
    blk = (at.view(B, blocks, BLOCK)[:, :, 0] // BLOCK)
    is_old = (rows < pos[:, None])[:, :, None, None]
    is_new = ((rows >= pos[:, None]) & (rows < pos[:, None] + n))[:, :, None, None]
    src = (rows - pos[:, None]).clamp(0, n - 1)
    out = dict(q=rot[:, :, :H].float().reshape(B * n, H * D))
    for name, new in (("k", rot[:, :, H:]), ("v", x[:, :, H + Hkv:].double())):
        codes, scales = s[name]
        new = new[seq, src] * is_new                                  # [B, W, Hkv, D]
        amax = new.view(B, blocks, BLOCK, Hkv, D).abs().amax(dim=(2, 4))
        need = torch.exp2(torch.ceil(torch.log2(amax / 127)).clamp(min=-126))
        need = torch.where(amax > 0, need, 0.0)
        was = scales[seq, blk].double()
        has_old = is_old.view(B, blocks, BLOCK).any(-1)[:, :, None]
        has_new = is_new.view(B, blocks, BLOCK).any(-1)[:, :, None]
        now = torch.maximum(torch.where(has_old, was, 0.0), need)
        safe = torch.where(now > 0, now, 1.0).repeat_interleave(BLOCK, 1)[..., None]
        old = codes[seq, at].double() * was.repeat_interleave(BLOCK, 1)[..., None]
        code = torch.round(torch.where(is_new, new, old) / safe).to(torch.int8)
        touched = (is_new | is_old) & has_new.repeat_interleave(BLOCK, 1)[..., None]
        code = torch.where(touched, code, codes[seq, at])
        inside = rows < s["S_max"]
        codes[seq.expand_as(at)[inside], at[inside]] = code[inside]
        keep = (blk * BLOCK == rows.view(B, blocks, BLOCK)[:, :, 0])
        value = torch.where(has_new, now, was).float()
        scales[seq.expand_as(blk)[keep], blk[keep]] = value[keep]
        got = codes[seq, at].float() * scales[seq, at // BLOCK][..., None]
        out[name] = got * inside[:, :, None, None]
    return out


def _attend(s):
    c = s["case"]
    B, n, H, Hkv, S = c["B"], c["n"], c["H"], c["Hkv"], s["S_max"]
    if own:
        att = importlib.import_module("0xbitnet_b200.attention")
        cache = _kept(s)
        if "workspace" not in s:
            s["workspace"] = att.attention_q8_workspace(cache, H, n)
        return att.attention_q8(s["q"], cache, H, n, s["lens"] if c["ragged"] else c["S"],
                                workspace=s["workspace"])
    lens = s["lens"].long() if c["ragged"] else torch.full((B,), c["S"], device=DEVICE)

    def plain(part):
        codes, scales = part
        wide = scales.repeat_interleave(BLOCK, 1)[:, :S]
        return (codes.float() * wide[..., None]).permute(0, 2, 1, 3)   # [B, Hkv, S, D]

    q = s["q"].view(B, n, Hkv, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    score = torch.matmul(q, plain(s["k"]).transpose(2, 3)) * (1.0 / math.sqrt(D))
    limit = lens[:, None] - n + torch.arange(n, device=DEVICE)         # last key of each row
    seen = torch.arange(S, device=DEVICE) <= limit[:, :, None]         # [B, n, S]
    seen = seen[:, None, :, None].expand(B, 1, n, H // Hkv, S).reshape(B, 1, -1, S)
    top = torch.where(seen, score, -torch.inf).amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(score - torch.where(top > -torch.inf, top, 0.0)), 0.0)
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, plain(s["v"])) / torch.where(total > 0, total, 1.0)
    return out.view(B, Hkv, n, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B * n, H * D)


def _logits(s):
    if own:
        mod = importlib.import_module("0xbitnet_b200.logits")
        if "rules" not in s:
            s["rules"] = mod.LogitRules(
                repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                history=s.get("history"), history_lens=s.get("history_lens"),
                bias_ids=s.get("bias_ids"), bias_values=s.get("bias_values"),
                mask=s.get("mask"))
        out, token = mod.logits_process(s["logits"], s["rules"])
        return dict(logits=out, token=token)
    x = s["logits"].double()   # each value is rounded once: a greedy choice hangs on it
    R, V = x.shape
    if "history" in s:
        h = s["history"].long()
        live = torch.arange(h.shape[1], device=DEVICE) < s["history_lens"][:, None]
        count = torch.zeros_like(x).scatter_add_(1, h, live.double())
        factor = s["repetition"].double()[:, None] ** count
        x = torch.where(x > 0, x / factor, x * factor)
        x = x - (s["frequency"].double()[:, None] * count
                 + s["presence"].double()[:, None] * (count > 0))
    if "bias_ids" in s:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias_values"].double())
    if "mask" in s:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=DEVICE, dtype=torch.int32)) & 1
        x = torch.where(bits.view(bits.shape[0], -1)[:, :V] > 0, x, -torch.inf)
    out = x.float()
    top = out.amax(1, keepdim=True)
    token = torch.where(out == top, torch.arange(V, device=DEVICE), V).amin(1)
    return dict(logits=out, token=torch.where(top[:, 0] > -torch.inf, token, -1).to(torch.int32))


# ---- work -------------------------------------------------------------------------------

def work(case):
    c = dict(case)
    if c["op"] == "logits":
        cells = c["R"] * c["V"]
        masks = {"none": 0, "rows": c["R"], "shared": 1}[c["mask"]]
        bytes_ = 8 * cells + masks * -(-c["V"] // 32) * 4
        bytes_ += c["R"] * (4 * c["hist"] * 3 // 4 + 8 * c["bias"] + 4)
        return {"bytes": bytes_, "flops": 2 * cells}
    B, n, H, Hkv = c["B"], c["n"], c["H"], c["Hkv"]
    if c["op"] == "append":
        rows = -(-(n + BLOCK - 1) // BLOCK) * BLOCK
        bytes_ = B * n * D * 4 * (2 * H + 2 * Hkv)               # qkv in, q out
        bytes_ += 2 * B * n * Hkv * D                            # codes written
        bytes_ += 2 * B * rows * Hkv * D * (1 + 4)               # the read-back
        return {"bytes": bytes_, "flops": 6 * B * n * (H + Hkv) * D}
    # ragged lengths are uniform over [n, S], but for the first
    keys = c["S"] + (B - 1) * ((c["S"] + n) / 2 if c["ragged"] else c["S"])
    bytes_ = 2 * keys * Hkv * D + 2 * keys / BLOCK * Hkv * 4 + 2 * 4 * B * n * H * D
    pairs = H * n * (keys - B * (n - 1) / 2)
    return {"bytes": bytes_, "flops": 4 * D * pairs}


# ---- exact values -------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logits": _exact_logits}[
        case["op"]](s)


def _exact_append(s):
    """Sequence by sequence and block by block, the rotation as a complex product."""
    c = s["case"]
    B, n, H, Hkv, W = c["B"], c["n"], c["H"], c["Hkv"], s["rows"]
    if B * W > 40000:
        return None
    x = s["qkv"].double().view(B, n, H + 2 * Hkv, D // 2, 2)
    i = torch.arange(D // 2, device=DEVICE, dtype=torch.float64)
    rate = torch.exp(-2 * i / D * math.log(THETA))
    q_all = torch.empty((B, n, H, D), dtype=torch.float64, device=DEVICE)
    back = {m: torch.zeros((B, W, Hkv, D), dtype=torch.float64, device=DEVICE) for m in "kv"}
    for b in range(B):
        pos = int(s["pos"][b]) if c["ragged"] else c["pos"]
        t = torch.arange(pos, pos + n, device=DEVICE, dtype=torch.float64)
        turn = torch.polar(torch.ones((n, D // 2), dtype=torch.float64, device=DEVICE),
                           torch.outer(t, rate))
        z = torch.view_as_complex(x[b, :, :H + Hkv].contiguous()) * turn[:, None]
        z = torch.view_as_real(z).reshape(n, H + Hkv, D)
        q_all[b] = z[:, :H]
        first = pos // BLOCK * BLOCK
        for m, new in (("k", z[:, H:]), ("v", x[b, :, H + Hkv:].reshape(n, Hkv, D))):
            codes, scales = s[m][0][b].double(), s[m][1][b].double()
            rows = min(W, s["S_max"] - first)
            # the window's blocks: its values, its new rows, what is behind them
            value = torch.zeros((W, Hkv, D), dtype=torch.float64, device=DEVICE)
            kind = torch.zeros(W, dtype=torch.int64, device=DEVICE)   # 0 old, 1 new, 2 behind
            old_scale = torch.zeros((W // BLOCK, Hkv), dtype=torch.float64, device=DEVICE)
            have = scales[first // BLOCK:first // BLOCK + W // BLOCK]
            old_scale[:have.shape[0]] = have
            wide = old_scale.repeat_interleave(BLOCK, 0)[..., None]
            value[:rows] = codes[first:first + rows] * wide[:rows]
            value[pos - first:pos - first + n] = new
            kind[pos - first:] = 1
            kind[pos - first + n:] = 2
            big = (value * (kind == 1)[:, None, None]).view(-1, BLOCK, Hkv, D).abs().amax((1, 3))
            mant, exp = torch.frexp(big / 127)
            need = torch.ldexp(torch.ones_like(big), exp - (mant == 0.5).int())
            need = torch.where(big > 0, need, 0)
            any_new = (kind == 1).view(-1, BLOCK).any(1)[:, None]
            any_old = (kind == 0).view(-1, BLOCK).any(1)[:, None]
            step = torch.maximum(need, old_scale * any_old)
            step = torch.where(any_new, step, old_scale).repeat_interleave(BLOCK, 0)[..., None]
            held = torch.round(value / torch.where(step > 0, step, 1)) * step
            behind = torch.zeros_like(value)
            behind[:rows] = codes[first:first + rows] * step[:rows]
            held = torch.where((kind == 2)[:, None, None], behind, held)
            untouched = ~any_new.repeat_interleave(BLOCK, 0)[..., None]
            back[m][b] = torch.where(untouched, value, held)
            back[m][b, rows:] = 0
    return dict(q=q_all.view(B * n, H * D), k=back["k"], v=back["v"])


def _exact_attend(s):
    """Head by head, a slice of the rows at a time, by the logarithm of the softmax's sum."""
    c = s["case"]
    B, n, H, Hkv = c["B"], c["n"], c["H"], c["Hkv"]
    if B * Hkv > 1200:
        return None
    out = torch.zeros((B, n, H, D), dtype=torch.float64, device=DEVICE)
    q = s["q"].double().view(B, n, H, D)
    for b in range(B):
        S = int(s["lens"][b]) if c["ragged"] else c["S"]
        block = torch.arange(S, device=DEVICE) // BLOCK
        for h in range(Hkv):
            K = s["k"][0][b, :S, h].double() * s["k"][1][b, block, h].double()[:, None]
            V = s["v"][0][b, :S, h].double() * s["v"][1][b, block, h].double()[:, None]
            for t in range(0, n, 256):
                rows = q[b, t:t + 256, h * (H // Hkv):(h + 1) * (H // Hkv)]
                z = torch.einsum("tgd,sd->tgs", rows, K) / math.sqrt(D)
                last = S - n + t + torch.arange(rows.shape[0], device=DEVICE)
                hidden = torch.arange(S, device=DEVICE)[None] > last[:, None]
                z = z.masked_fill(hidden[:, None], -torch.inf)
                z = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
                out[b, t:t + 256, h * (H // Hkv):(h + 1) * (H // Hkv)] = \
                    torch.einsum("tgs,sd->tgd", z, V)
    return out.view(B * n, H * D)


def _exact_logits(s):
    """Row by row, over the ids that the rules name only."""
    R, V = s["logits"].shape
    out = s["logits"].double().clone()
    for r in range(R):
        if "history" in s:
            ids, times = torch.unique(s["history"][r, :int(s["history_lens"][r])].long(),
                                      return_counts=True)
            v, t = out[r, ids], times.double()
            grow = torch.exp(t * torch.log(s["repetition"][r].double()))
            v = torch.where(v > 0, v / grow, v * grow)
            out[r, ids] = v - s["presence"][r].double() - t * s["frequency"][r].double()
        if "bias_ids" in s:
            ids, back = torch.unique(s["bias_ids"][r].long(), return_inverse=True)
            add = torch.zeros(ids.numel(), dtype=torch.float64, device=DEVICE)
            add.index_add_(0, back, s["bias_values"][r].double())
            out[r, ids] += add
        if "mask" in s:
            word = s["mask"][r % s["mask"].shape[0]].long()
            i = torch.arange(V, device=DEVICE)
            out[r].masked_fill_((word[i // 32] >> (i % 32)) % 2 == 0, -torch.inf)
    return dict(logits=out, token=None)
