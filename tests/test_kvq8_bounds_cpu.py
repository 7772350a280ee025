"""CPU check that the row bound of the 8-bit cache's attention tests notices what it is for."""
import numpy as np
import pytest

from oracle import q8_ref as ref

D = 128
SCALE = float(np.float32(1.0) / np.sqrt(np.float32(D)))


def ratio(got, want, tol):
    return (np.sqrt(((got - want) ** 2).mean(-1)) / tol).max()


@pytest.mark.parametrize("n,S", [(1, 40000), (4, 3000), (64, 2100)])
def test_the_bound_notices_what_it_is_for(n, S):
    """In the oracle: one key left out, or added, weights in one f16, queries in one f16."""
    rng = np.random.default_rng(n)
    H, Hkv = 2, 1
    k, v = rng.standard_normal((S + 1, Hkv, D)), rng.standard_normal((S + 1, Hkv, D))
    q = rng.standard_normal((n, H, D)).astype(np.float32)
    want, tol = ref.attention_rms(q, k, v, S, SCALE)

    def softmax(q, lo, hi, cut=lambda p: p):
        out = np.zeros((n, H, D))
        for t in range(n):
            last = S - n + t + 1 + hi
            p = np.exp((s := q[t].astype(np.float64) @ k[lo:last, 0].T * SCALE) - s.max(1, keepdims=True))
            out[t] = cut(p) @ v[lo:last, 0] / p.sum(1, keepdims=True)
        return out
    assert ratio(softmax(q, 0, 0), want, tol) < 1e-6
    f16 = lambda x: x.astype(np.float16).astype(np.float64)
    assert ratio(softmax(q, 1, 0), want, tol) > 20       # the first key lost
    assert ratio(softmax(q, 0, -1), want, tol) > 20      # the last one
    assert ratio(softmax(q, 0, 1), want, tol) > 20       # one key too many
    assert ratio(softmax(q, 0, 0, lambda p: f16(256 * p) / 256), want, tol) > 10
    assert ratio(softmax(f16(q), 0, 0), want, tol) > 10
