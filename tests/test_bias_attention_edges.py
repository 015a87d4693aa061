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


def _pairs(table, keep, max_distance, bidirectional, q_offset):
    """Visible pairs of each bucket, keep [B, Sq, Sk]."""
    Sq, Sk = keep.shape[1:]
    rel = torch.arange(Sk)[None, :] - torch.arange(Sq)[:, None] - q_offset
    lo = int(rel.min())
    lut = torch.tensor([ot.bucket(r, table.shape[0], max_distance, bidirectional) for r in range(lo, int(rel.max()) + 1)])
    return torch.bincount(lut[rel - lo].flatten(), weights=keep.sum(0).flatten().double(), minlength=table.shape[0])


def _tight(got, ref, far):
    """The bias gradient is a sum of fp32 dS. delta comes from an output good to 2^-16 + 2^-17 of itself (1024 keys are 64
    truncating steps of P's two halves; P is good to 2^-17), the two exponentials and dP move dS by 2^-16 of itself. A far bucket
    may be taken as minus the sum of the others, and then has their errors."""
    own = (2.0 ** -16 + 2.0 ** -17) * ref["dtable_abs"] + 2.0 ** -16 * ref["ds_abs"] + 1e-9
    bound = own.clone()
    bound[far] = own.sum(0)
    err = (got["dtable"].cpu().double() - ref["dtable"]).abs()
    assert bool((err <= bound).all()), f"dtable: {(err / bound).max().item():.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", ["left", "left_causal", "far", "all_far", "before_the_keys", "none"])
def test_a_bucket_without_a_pair_has_no_gradient(dt, D, case):
    """Padding and the causal rule leave some buckets without a pair: their gradient is exactly zero, the others' is right."""
    Sq, Sk, dist, kw = 1024, 1024, 128, {}
    keep = torch.ones(1, Sk, dtype=torch.bool)
    if case.startswith("left"):  # left padding: no two of the keys that are left are far apart
        keep[:, :941] = False
        if case == "left_causal":
            kw = dict(causal=True, bidirectional=False)
    elif case == "far":  # every key well after the queries is masked, and most before
        Sq, kw = 300, dict(q_offset=724)
        keep[:, :700] = keep[:, 760:] = False
    elif case == "all_far":
        Sq, Sk, kw = 200, 40, dict(q_offset=700)
        keep = keep[:, :Sk]
    elif case == "before_the_keys":  # the first queries see nothing, and no query sees a key after it
        Sq, Sk, dist, kw = 140, 100, 4, dict(causal=True, bidirectional=True, q_offset=-100)
        keep = keep[:, :Sk]
    q, k, v, go, table, _ = _case(1, 2, 2, Sq, Sk, D, dt, D + Sq, nb=4 if dist == 4 else 32)
    kw["max_distance"] = dist
    m = None if bool(keep.all()) else keep
    ref = ot.bias_attention(q, k, v, table, key_mask=m, go=go, **kw)
    got = _run(q, k, v, table, m, go, **kw)
    rel = torch.arange(Sk)[None, :] - torch.arange(Sq)[:, None] - kw.get("q_offset", 0)
    seen = keep[:, None, :] & ((rel <= 0) if kw.get("causal") else torch.ones_like(rel, dtype=torch.bool))
    bidir = kw.get("bidirectional", True)
    pairs = _pairs(table, seen, dist, bidir, kw.get("q_offset", 0))
    assert int((pairs == 0).sum()) >= (1 if case == "none" else 2)  # two-sided: the place of distance 0 after the query
    assert not got["dtable"].cpu()[pairs == 0].any()
    side = table.shape[0] // (2 if bidir else 1)
    _tight(got, ref, [side - 1, table.shape[0] - 1, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
def test_a_nan_in_a_block_of_one_far_bucket_reaches_the_bias_gradient(dt):
    q, k, v, go, table, _ = _case(1, 2, 2, 130, 40, 64, dt, 3)
    v = v.clone()
    v[0, 1, 5, 6] = NAN
    got = _run(q, k, v, table, None, go, q_offset=900)
    assert torch.isnan(got["dtable"][15, 1]) and torch.isfinite(got["dtable"][:, 0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Sq,Sk,D,mask,causal", [(150, 290, 64, "tail", False), (150, 290, 128, "head", True), (700, 700, 128, "random", False),
                                                 (700, 700, 64, "none", True), (33, 1000, 40, "tail", True), (1000, 60, 96, "none", False)])
def test_bias_gradient_is_as_good_as_its_output(dt, Sq, Sk, D, mask, causal):
    q, k, v, go, table, m = _case(2, 4, 2, Sq, Sk, D, dt, Sq + D, mask)
    kw = dict(causal=causal, bidirectional=not causal, q_offset=Sk - Sq if causal else 0)
    ref = ot.bias_attention(q, k, v, table, key_mask=m, go=go, **kw)
    _tight(_run(q, k, v, table, m, go, **kw), ref, [31] if causal else [15, 31])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("D", [64, 128, 20])
def test_a_row_with_one_key_has_no_gradient_of_its_scores(dt, D):
    """P is 1 there whatever the score: dq and the bias gradient are exactly zero, and a NaN is not lost."""
    Sq, Sk = 200, 300
    q, k, v, go, table, _ = _case(2, 4, 2, Sq, Sk, D, dt, D)
    m = torch.zeros(2, Sk, dtype=torch.bool)
    m[0, 123] = m[1, 299] = True
    got = _check(q, k, v, go, table, m)
    assert not got["dq"].any() and not got["dtable"].any()
    m[1, 7] = True  # the second sample's queries choose between two keys
    got = _check(q, k, v, go, table, m)
    assert not got["dq"][0].any() and got["dq"][1].any() and got["dtable"].any()
    kw = dict(causal=True, bidirectional=False, q_offset=0)
    m[0, 5:] = True
    got = _check(q, k, v, go, table, m, **kw)  # none for rows 0..4 of the first sample, one for row 5; one for the second's rows 7..
    assert not got["dq"][0, :, :6].any() and got["dq"][0, :, 6:].any(-1).all() and not got["dq"][1].any()
    got = _check(q, k, v, go, table, None, **kw)
    assert not got["dq"][:, :, 0].any() and got["dq"][:, :, 1:].any(-1).all()
    v = v.clone()
    v[0, 0, 0, 1] = NAN
    got = _run(q, k, v, table, None, go, **kw)
    assert torch.isnan(got["dq"][0, 0, 0]).any() and torch.isnan(got["dtable"][:, 0]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("up", [-24, -16, -12, 0, 9])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_half_gradients_of_any_magnitude(up, D, causal):
    """Gradients of an f16 call are as good for a loss that was not scaled as for one that was: relative to their norm, and to
    half a step of f16's smallest numbers."""
    Sq, Sk, dt = 260, 900, torch.float16
    q, k, v, go, table, m = _case(2, 4, 2, Sq, Sk, D, dt, D + 100, "tail")
    if up > 0:  # rows that look at one key: dS as large as dP
        q, v = q * 6, v * 4
    go = torch.ldexp(go.float(), torch.tensor(up)).to(dt)
    kw = dict(causal=causal, bidirectional=not causal, q_offset=Sk - Sq if causal else 0)
    ref = ot.bias_attention(q, k, v, table, key_mask=m, go=go, **kw)
    got = _run(q, k, v, table, m, go, **kw)
    for n in ("dq", "dk", "dv"):
        assert ref[n].abs().max() < 60000
        mags = 0.0 if n == "dv" else 2.0 ** -20 * ref[n + "_abs"].norm().item()
        _near(got[n], ref[n], GRAD[dt], n, 1e-9 * 2.0 ** up + mags + 2.0 ** -25 * ref[n].numel() ** 0.5)
    _tight(got, ref, [15, 31])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("Sq,D", [(1, 64), (8, 128), (150, 64), (150, 128), (150, 20)])
@pytest.mark.parametrize("low", [-torch.finfo(torch.float32).max, -INF])
def test_a_bucket_of_the_lowest_bias_is_left_out(dt, Sq, D, low):
    """A table entry of fp32's lowest value hides its keys as -inf does; a row that has no others gets zeros."""
    q, k, v, go, table, _ = _case(2, 2, 2, Sq, 300, D, dt, D)
    table[3], table[7, 0], table[12:16], table[20:] = low, low, low, low
    kw = dict(q_offset=40)
    ref = ot.bias_attention(q, k, v, table.clamp(min=-INF if low == -INF else -1e30), go=go, **kw)
    got = _run(q, k, v, table, None, go, **kw)
    _near(got["o"], ref["o"], OUT[dt], "o")
    _near(_infer(q, k, v, table, None, **kw), ref["o"], OUT[dt], "o")
    for n in ("dq", "dk", "dv"):
        _near(got[n], ref[n], GRAD[dt], n, 1e-9 if n == "dv" else 1e-9 + 2.0 ** -20 * ref[n + "_abs"].norm().item())
    for i in [3, *range(12, 16), *range(20, 32)]:
        assert not got["dtable"][i].any()
    table[:, 1] = low
    got = _run(q, k, v, table, None, go, **kw)
    assert not got["o"][:, 1].any() and not got["dq"][:, 1].any() and not got["dk"][:, 1].any() and not got["dv"][:, 1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bidirectional,off", [(True, 1300), (True, 0), (False, 1300)])
def test_a_far_bucket_of_little_weight_keeps_its_own_accuracy(dt, D, bidirectional, off):
    """A table that has learned to look nearby: the far buckets hold most keys and almost no weight, and their small gradients
    are not made from the large ones."""
    Sq, Sk = 200, 1500
    q, k, v, go, table, _ = _case(1, 2, 2, Sq, Sk, D, dt, D)
    table[[15, 31] if bidirectional else [31]] = -16.0
    kw = dict(q_offset=off, bidirectional=bidirectional, causal=not bidirectional)
    ref = ot.bias_attention(q, k, v, table, go=go, **kw)
    _tight(_run(q, k, v, table, None, go, **kw), ref, [])
