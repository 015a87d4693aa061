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


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("Sq", [1, 8, 9, 130])
@pytest.mark.parametrize("Sk", [50, 5000])
def test_a_nan_is_not_taken_for_a_row_without_keys(dt, Sq, Sk):
    """A query or a visible key that holds a NaN gives NaN, in its rows and heads alone, whatever the number of key splits."""
    q, k, v, go, table, _ = _case(2, 4, 2, Sq, Sk, 64, dt, Sq + Sk)
    ref = ot.bias_attention(q, k, v, table)
    q2, k2 = q.clone(), k.clone()
    q2[0, 1, 0, 3] = NAN  # one row
    k2[1, 1, 7, 2] = NAN  # every row of the two heads that read it
    want = torch.zeros(2, 4, Sq, dtype=torch.bool)
    want[0, 1, 0] = want[1, 2] = want[1, 3] = True
    got = _run(q2, k2, v, table, None, go)
    for o in (got["o"], _infer(q2, k2, v, table, None)):
        nan = torch.isnan(o.cpu())
        assert torch.equal(nan.all(-1), want) and torch.equal(nan.any(-1), want)
        _near(o.cpu()[~want].cuda(), ref[~want], OUT[dt], "o")
    assert torch.equal(torch.isnan(got["dq"].cpu()).any(-1), want)
    for n in ("dk", "dv"):  # both of the rows' key heads
        assert torch.isnan(got[n].cpu()[0, 0]).any() and torch.isnan(got[n].cpu()[1, 1]).any()
        assert torch.isfinite(got[n].cpu()[0, 1]).all() and torch.isfinite(got[n].cpu()[1, 0]).all()
    assert torch.isnan(got["dtable"].cpu()).any(0).tolist() == [False, True, True, True]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("Sq", [1, 9])
def test_an_infinite_score_is_nan_and_rows_without_keys_stay_zero(dt, Sq):
    q, k, v, go, table, _ = _case(2, 2, 2, Sq, 300, 64, dt, Sq)
    table[:, 1] = INF
    m = torch.ones(2, 300, dtype=torch.bool)
    m[1] = False
    for o in (_run(q, k, v, table, m, go)["o"], _infer(q, k, v, table, m)):
        assert torch.isnan(o[0, 1]).all() and torch.isfinite(o[0, 0]).all() and not o[1].any()
