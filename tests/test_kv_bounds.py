"""The bound that fp32 results of the paged cache's attention are held to tells fp32's precision from less.  Needs no GPU."""
import numpy as np
import pytest

import kv_ref as ref


def parts(x, n):
    """x in n fp16 parts."""
    kept = np.zeros_like(x)
    for _ in range(n):
        kept = kept + (x - kept).astype(np.float16).astype(np.float64)
    return kept


def attention_in_parts(q, keys, values, scale, q_parts, p_parts, leave_out=None):
    """One row's attention with queries and probabilities in so many fp16 parts, a token left out."""
    s = keys @ parts(q, q_parts).T * scale
    p = np.exp(s - s.max(0)) * 16
    if leave_out is not None:
        p[leave_out] = 0
    total = p.sum(0)
    return (parts(p, p_parts).T @ values) / total[:, None]


@pytest.mark.parametrize("fmt", [ref.F16, ref.Q4_0, ref.Q8_0])
@pytest.mark.parametrize("hd,n", [(64, 20), (64, 700), (128, 500), (128, 2500), (96, 333), (256, 90)])
def test_what_the_norm_tells_apart(fmt, hd, n):
    rng = np.random.default_rng(hd + n)
    k, v = (ref.stored(rng.standard_normal((n, hd)).astype(np.float32), fmt) for _ in range(2))
    q = (rng.standard_normal((4, hd)) * 2).astype(np.float32).astype(np.float64)
    want = ref.attention(q[None].astype(np.float32), k[:, None], v[:, None], n, hd ** -0.5)[0]

    def off(*how):
        return np.linalg.norm(attention_in_parts(q, k, v, hd ** -0.5, *how) - want) / np.linalg.norm(want)

    bound = ref.fp32_norm_bound(2.0)
    assert off(2, 2) <= bound / 4                       # 22 bits
    assert off(1, 2) > 4 * bound and off(2, 1) > 4 * bound  # 11 bits of queries, of probabilities
    assert off(2, 2, n // 2) > 4 * bound                # a token that was lost
