"""CPU checks of the 8-bit cache's and the logit rules' argument checks, and of the 64-bit
restatements that the GPU tests compare with. No kernel runs: every call is refused on the
host, before any pointer is used."""
import ctypes

import numpy as np
import pytest

from _util import obn
from oracle import q8_ref as ref

P = 4096  # an aligned address that is never read


def call(name, **over):
    base = {
        "obn_rope_kv_append_q8": dict(qkv=P, B=1, n=1, H=4, Hkv=2, d=128, pos=0, pos_dev=None,
                                      base=1e4, q=P, k=P, v=P, ks=P, vs=P, S=64, st=None),
        "obn_kv_read_q8": dict(k=P, v=P, ks=P, vs=P, B=1, Hkv=2, d=128, S=64, first=0, fd=None,
                               count=1, ko=P, vo=P, st=None),
        "obn_attention_q8": dict(q=P, k=P, v=P, ks=P, vs=P, B=1, n=1, H=4, Hkv=2, d=128, S=64,
                                 L=10, ld=None, scale=1.0, out=P, ws=P, wb=1 << 40, st=None),
    }[name]
    assert set(over) <= set(base)
    return getattr(obn().lib(), name)(*dict(base, **over).values())


INV, UNS = -1, -2


@pytest.mark.parametrize("name,over,code", [
    ("obn_rope_kv_append_q8", dict(qkv=None), INV), ("obn_rope_kv_append_q8", dict(q=None), INV),
    ("obn_rope_kv_append_q8", dict(ks=None), INV), ("obn_rope_kv_append_q8", dict(B=0), INV),
    ("obn_rope_kv_append_q8", dict(n=0), INV), ("obn_rope_kv_append_q8", dict(pos=-1), INV),
    ("obn_rope_kv_append_q8", dict(pos=64), INV), ("obn_rope_kv_append_q8", dict(n=65), INV),
    ("obn_rope_kv_append_q8", dict(pos=2147483647), INV),
    ("obn_rope_kv_append_q8", dict(d=64), UNS), ("obn_rope_kv_append_q8", dict(H=5), UNS),
    ("obn_rope_kv_append_q8", dict(H=65536), UNS), ("obn_rope_kv_append_q8", dict(qkv=P + 8), INV),
    ("obn_rope_kv_append_q8", dict(q=P + 4), INV), ("obn_rope_kv_append_q8", dict(k=P + 8), INV),
    ("obn_rope_kv_append_q8", dict(base=0.0), INV),
    ("obn_rope_kv_append_q8", dict(base=float("nan")), INV),
    ("obn_rope_kv_append_q8", dict(pos_dev=P + 2), INV),
    ("obn_rope_kv_append_q8", dict(n=1 << 29, pos_dev=P), UNS),
    ("obn_rope_kv_append_q8", dict(B=65536), UNS),
    ("obn_rope_kv_append_q8", dict(S=(1 << 30) + 1), UNS),
    ("obn_kv_read_q8", dict(ko=None, vo=None), INV), ("obn_kv_read_q8", dict(count=0), INV),
    ("obn_kv_read_q8", dict(ko=P + 8), INV), ("obn_kv_read_q8", dict(v=None), INV),
    ("obn_kv_read_q8", dict(d=256), UNS), ("obn_kv_read_q8", dict(fd=P + 1), INV),
    ("obn_attention_q8", dict(q=None), INV), ("obn_attention_q8", dict(ws=None), INV),
    ("obn_attention_q8", dict(wb=0), INV), ("obn_attention_q8", dict(ws=P + 128), INV),
    ("obn_attention_q8", dict(L=65), INV), ("obn_attention_q8", dict(L=-1), INV),
    ("obn_attention_q8", dict(H=3), UNS), ("obn_attention_q8", dict(H=65536), UNS),
    ("obn_attention_q8", dict(scale=-0.5), INV),
    ("obn_attention_q8", dict(scale=float("nan")), INV),
    ("obn_attention_q8", dict(scale=float("inf")), INV),
    ("obn_attention_q8", dict(d=96), UNS), ("obn_attention_q8", dict(q=P + 8), INV),
    ("obn_attention_q8", dict(out=P + 4), INV), ("obn_attention_q8", dict(Hkv=0), INV),
    ("obn_attention_q8", dict(n=-1), INV), ("obn_attention_q8", dict(ld=P + 2), INV),
    ("obn_attention_q8", dict(vs=P + 2), INV),
])
def test_cache_refusals(name, over, code):
    assert call(name, **over) == code
    assert obn().lib().obn_error_message()


@pytest.mark.parametrize("args,zero", [
    ((1, 1, 20, 5, 128, 2048), False), ((0, 1, 20, 5, 128, 2048), True),
    ((1, 1, 20, 6, 128, 2048), True), ((1, 1, 20, 5, 64, 2048), True),
    ((1, 1, 20, 5, 128, 0), True),
])
def test_workspace_bytes(args, zero):
    assert (obn().lib().obn_attention_q8_workspace_bytes(*args) == 0) == zero


@pytest.mark.parametrize("over,rules,code", [
    (dict(logits=None), {}, INV), (dict(out=None), {}, INV), (dict(rows=0), {}, INV),
    (dict(vocab=0), {}, INV), (dict(vocab=(1 << 24) + 1), {}, UNS), (dict(rows=65536), {}, UNS),
    (dict(logits=P + 2), {}, INV), (dict(token=P + 1), {}, INV),
    ({}, dict(history=P, history_cap=65536), UNS), ({}, dict(history=P, history_cap=-1), UNS),
    ({}, dict(bias_ids=P, bias_values=P, bias_cap=1025), UNS),
    ({}, dict(bias_ids=P, bias_cap=4), INV), ({}, dict(bias_values=P, bias_cap=4), INV),
    ({}, dict(history=P, history_cap=8, history_ld=7), INV),
    ({}, dict(bias_ids=P, bias_values=P, bias_cap=8, bias_ld=4), INV),
    ({}, dict(mask=P, mask_ld=3), INV), ({}, dict(mask=P + 2), INV),
    ({}, dict(history=P, history_cap=8, history_ld=-1), INV),
    ({}, dict(repetition=P + 1), INV), ({}, dict(history=P, history_lens=P + 3), INV),
])
def test_logit_refusals(over, rules, code):
    lib_ = obn()._lib
    s = lib_.LogitRulesStruct(**rules)
    a = dict(dict(logits=P, rows=2, vocab=100, rules=ctypes.addressof(s), out=P, token=P,
                  st=None), **over)
    assert lib_.lib().obn_logits_process(*a.values()) == code
    assert lib_.lib().obn_error_message()


def test_null_rules_are_refused():
    assert obn().lib().obn_logits_process(P, 1, 10, None, P, P, None) == INV


def test_host_wrappers_refuse_cpu_tensors():
    import importlib
    import torch
    att = importlib.import_module("0xbitnet_b200.attention")
    lg = importlib.import_module("0xbitnet_b200.logits")
    k = torch.zeros((1, 16, 2, 128), dtype=torch.int8)
    s = torch.zeros((1, 1, 2))
    with pytest.raises(TypeError):
        att.KVCacheQ8.wrap(k, s, k, s)
    with pytest.raises(TypeError):
        lg.LogitRules(history=torch.zeros((1, 4), dtype=torch.int32))
    with pytest.raises(ValueError):
        lg.LogitRules(bias_ids=torch.zeros((1, 4), dtype=torch.int32))
    with pytest.raises(TypeError):
        lg.logits_process(torch.zeros((1, 4)), lg.LogitRules())


def test_rules_struct_matches_the_header():
    """Field order of obn_logit_rules in include/obn.h and in the binding."""
    import os
    import re
    from _util import ROOT
    text = open(os.path.join(ROOT, "include", "obn.h")).read()
    body = re.search(r"typedef struct obn_logit_rules \{(.*?)\} obn_logit_rules;", text, re.S)[1]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [re.search(r"(\w+)\s*$", f)[1] for f in body.split(";") if f.strip()]
    assert names == [f[0] for f in obn()._lib.LogitRulesStruct._fields_]


# ---- the restatements themselves ---------------------------------------------------------

def test_need_scale():
    assert ref.need_scale(np.zeros(3)) == 0.0
    assert ref.need_scale(np.array([127.0])) == 1.0
    assert ref.need_scale(np.array([np.nextafter(127.0, 200.0)])) == 2.0
    assert ref.need_scale(np.array([1e-45])) == 2.0 ** -126
    assert np.isnan(ref.need_scale(np.array([1.0, np.inf])))


def test_append_bounds_the_error_of_a_growing_block():
    rng = np.random.default_rng(0)
    codes, scales = np.zeros((16, 1, 8), np.int64), np.zeros((1, 1))
    rows = [rng.standard_normal((1, 1, 8)) * 1.4 ** t for t in range(16)]
    for t, r in enumerate(rows):
        ref.append(codes, scales, r, t)
    err = np.abs(ref.values(codes, scales) - np.concatenate(rows))
    assert err.max() <= scales[0, 0] and np.abs(codes).max() <= 127


def test_attention_restatement_against_a_direct_softmax():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((3, 4, 8)), rng.standard_normal((9, 2, 8)), \
        rng.standard_normal((9, 2, 8))
    out, bound = ref.attention(q, k, v, 7, 0.3)
    s = np.exp(k[:6, 1] @ q[1, 3] * 0.3)
    np.testing.assert_allclose(out[1, 3], (s[:, None] * v[:6, 1]).sum(0) / s.sum(), rtol=1e-13)
    assert (bound > 0).all()
    out, _ = ref.attention(q, k, v, 1, 0.3)  # three queries, one position: two see nothing
    assert not out[:2].any() and np.array_equal(out[2, 0], v[0, 0])


def test_logits_restatement():
    x = np.array([2.0, -2.0, 0.0, 1.0], np.float32)
    y = ref.logits(x, 2.0, 0.5, 0.25, [0, 1, 1, 9, -1], [(3, 1.0), (3, 2.0)],
                   np.array([True, True, False, True]))
    assert y.tolist() == [1.0 - 0.75, -8.0 - 1.25, -np.inf, 4.0]
