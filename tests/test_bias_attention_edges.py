"""Where the bias attention's definition is easy to lose: keys that the causal rule hides from every query, values that
are not finite, buckets without a pair, rows with a single key, gradients far from one in magnitude.

Tolerances are those of test_bias_attention.py (derived there); the bias gradient's is `_tight` below."""

import pytest
import torch

import oracle.text as ot
from tests.test_bias_attention import DTS, GRAD, OUT, _case, _check, _near, _run

NAN, INF = float("nan"), float("inf")


def _infer(q, k, v, table, m, **kw):
    import torch_vulkan_b200 as tv

    with torch.no_grad():
        return tv.bucket_bias_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), key_mask=None if m is None else m.cuda(), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("Sq", [9, 100, 200])
@pytest.mark.parametrize("D", [64, 128, 20])
def test_keys_past_the_last_query_may_hold_anything(dt, Sq, D):
    """A prompt chunk in a preallocated cache: the slots after it are not written yet."""
    Sk, off = 700, 150
    q, k, v, go, table, _ = _case(2, 4, 2, Sq, Sk, D, dt, Sq + D)
    kw = dict(causal=True, bidirectional=False, q_offset=off)
    clean, plain = _check(q, k, v, go, table, None, **kw), _infer(q, k, v, table, None, **kw)
    for bad in (NAN, INF, -torch.finfo(dt).max):
        k2, v2 = k.clone(), v.clone()
        k2[:, :, off + Sq:], v2[:, :, off + Sq:] = bad, bad
        got = _run(q, k2, v2, table, None, go, **kw)
        for n in clean:
            assert torch.equal(got[n], clean[n]), (n, bad)
        assert not got["dk"][:, :, off + Sq:].any() and not got["dv"][:, :, off + Sq:].any()
        assert torch.equal(_infer(q, k2, v2, table, None, **kw), plain), bad
        some = torch.ones(2, Sk, dtype=torch.bool)  # the same with a mask that leaves the slots in
        some[1, 40:60] = False
        k2[1, :, 40:60] = bad
        a, b = _run(q, k2, v2, table, some, go, **kw), _run(q, k, v, table, some, go, **kw)
        for n in a:
            assert torch.equal(a[n], b[n]), (n, bad)
