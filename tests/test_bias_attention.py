"""Attention with a bucketed relative position bias against float64, forward and backward.

Tolerances (relative L2): an output passes at most two roundings to its type (P and the output), a gradient three
(P or dS, an operand made from them, the output), each at most u = 2^-8 (bf16) or 2^-11 (f16); fp32 sums over these
lengths and two exponentials stay within 3e-5. dq and dk are made from the difference dP - delta, whose two fp32 sums
are off by up to 2^-20 of their magnitudes even where it cancels (a row with a single key). The bias gradient is summed in fp32 from fp32 dS, but delta is made from
the rounded output, which moves it by at most u sum(P |dO||O|) in each bucket; the rest is 2^-14 of the magnitudes."""

import itertools

import pytest
import torch

import oracle.text as ot
from tests.helpers import rel_err

U = {torch.float32: 2.0 ** -22, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
OUT = {torch.float32: 3e-5, torch.bfloat16: 2 * 2.0 ** -8, torch.float16: 2 * 2.0 ** -11}
GRAD = {torch.float32: 3e-5, torch.bfloat16: 3 * 2.0 ** -8, torch.float16: 3 * 2.0 ** -11}


def _case(B, H, Hk, Sq, Sk, D, dt, seed, mask="none", nb=32, bshd=True):
    g = torch.Generator().manual_seed(seed)

    def mk(heads, s, std=1.0):
        t = (torch.randn(B, s, heads, D, generator=g) * std).to(dt)
        return t.transpose(1, 2) if bshd else t.transpose(1, 2).contiguous()

    q, k, v, go = mk(H, Sq, D ** -0.25), mk(Hk, Sk, D ** 0.25), mk(Hk, Sk), mk(H, Sq)
    table = torch.randn(nb, H, generator=g)
    m = None
    if mask == "tail":
        lens = torch.randint(1, Sk + 1, (B,), generator=g)
        m = torch.arange(Sk)[None, :] < lens[:, None]
    elif mask == "head":  # padding on the left
        m = torch.arange(Sk)[None, :] >= torch.randint(0, Sk, (B,), generator=g)[:, None]
    elif mask == "random":
        m = torch.rand(B, Sk, generator=g) > 0.4
        m[-1] = False  # one sample without a key
    return q, k, v, go, table, m


def _run(q, k, v, table, m, go, **kw):
    import torch_vulkan_b200 as tv

    leaf = [t.cuda().detach().requires_grad_(True) for t in (q, k, v, table)]
    o = tv.bucket_bias_attention(*leaf, key_mask=None if m is None else m.cuda(), **kw)
    grads = torch.autograd.grad(o, leaf, go.cuda())
    return dict(zip(("o", "dq", "dk", "dv", "dtable"), (o.detach(), *grads)))


def _near(got, ref, tol, what, floor=1e-9):
    assert got.shape == ref.shape
    assert torch.isfinite(got).all(), what
    err = (got.cpu().double() - ref).norm()
    assert err <= tol * ref.norm() + floor, f"{what}: {(err / ref.norm()).item():.3g} > {tol:.3g}"


def _check(q, k, v, go, table, m, **kw):
    ref = ot.bias_attention(q, k, v, table, key_mask=m, go=go, **kw)
    got = _run(q, k, v, table, m, go, **kw)
    dt = q.dtype
    _near(got["o"], ref["o"], OUT[dt], "o")
    for n in ("dq", "dk", "dv"):
        _near(got[n], ref[n], GRAD[dt], n, 1e-9 if n == "dv" else 1e-9 + 2.0 ** -20 * ref[n + "_abs"].norm().item())
    bound = U[dt] * ref["dtable_abs"] + 2.0 ** -14 * ref["ds_abs"] + 1e-7
    err = (got["dtable"].cpu().double() - ref["dtable"]).abs()
    assert bool((err <= bound).all()), f"dtable: {(err / bound).max().item():.3g} of the bound"
    return got


DTS = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("Sq,Sk,D", [(1, 1, 64), (1, 130, 64), (5, 3, 64), (64, 64, 64), (77, 77, 64), (128, 128, 64), (129, 257, 64),
                                     (200, 129, 128), (384, 384, 128), (300, 511, 40), (33, 65, 80), (130, 100, 20), (257, 130, 7)])
def test_lengths_and_head_dims(dt, Sq, Sk, D):
    _check(*_case(2, 2, 2, Sq, Sk, D, dt, Sq * 7 + Sk + D))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("mask,causal", list(itertools.product(["none", "tail", "head", "random"], [False, True])))
def test_masks(dt, mask, causal):
    Sq, Sk = 150, 290
    kw = dict(causal=causal, bidirectional=not causal, q_offset=Sk - Sq if causal else 0)
    q, k, v, go, table, m = _case(3, 2, 2, Sq, Sk, 64, dt, 11, mask)
    got = _check(q, k, v, go, table, m, **kw)
    if mask == "random":  # the sample whose keys are all masked: zeros throughout
        for n in ("o", "dq", "dk", "dv"):
            assert not got[n][-1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
def test_causal_rows_before_the_first_key(dt):
    """A negative offset leaves the first queries without a key; two directions and one-sided buckets."""
    for bidir in (False, True):
        got = _check(*_case(2, 2, 1, 140, 100, 64, dt, 5), causal=True, bidirectional=bidir, q_offset=-30)
        assert not got["o"][:, :, :30].any() and not got["dq"][:, :, :30].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("H,Hk", [(6, 3), (4, 1), (8, 2)])
def test_shared_heads(dt, H, Hk):
    _check(*_case(2, H, Hk, 140, 200, 64, dt, H * 10 + Hk, "tail"))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nb,dist,bidir", [(32, 128, True), (32, 128, False), (4, 2, True), (2, 2, False), (64, 1024, True), (128, 1000, False), (8, 300, True)])
def test_bucket_parameters(dt, nb, dist, bidir):
    _check(*_case(1, 2, 2, 330, 700, 64, dt, nb + dist, nb=nb), max_distance=dist, bidirectional=bidir)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("off", [-400, -131, 1, 200, 5000])
def test_offsets(dt, off):
    _check(*_case(1, 2, 2, 140, 270, 64, dt, 3), q_offset=off)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
def test_values_at_masked_positions_are_never_used(dt):
    q, k, v, go, table, m = _case(2, 2, 2, 150, 300, 64, dt, 21, "tail")
    m[1, 130:140] = False
    clean = _run(q, k, v, table, m, go)
    for bad in (float("nan"), float("inf"), -torch.finfo(dt).max):
        k2, v2 = k.clone(), v.clone()
        hide = ~m[:, None, :, None].expand_as(k)
        k2[hide], v2[hide] = bad, bad
        got = _run(q, k2, v2, table, m, go)
        for n in clean:
            assert torch.equal(got[n], clean[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
def test_strides_views_and_expanded_inputs(dt):
    B, H, S, D = 2, 3, 100, 64
    g = torch.Generator().manual_seed(2)
    big = torch.randn(B, S, 3, H, D, generator=g).to(dt)
    q, k, v = (big[:, :, i].transpose(1, 2) for i in range(3))  # column blocks of one projection's output
    go = torch.randn(B, H, S, D, generator=g).to(dt)
    table = torch.randn(32, H, generator=g)
    _check(q, k, v, go, table, None)
    base = torch.randn(B, H, S, D + 1, generator=g).to(dt)
    _check(base[..., 1:], k, v, go, table, None)  # rows off every alignment
    _check(q, k[:1].expand(B, H, S, D), v[:1].expand(B, H, S, D), go, table, None)
    _check(q, k.flip(2).flip(2), v.transpose(2, 3).contiguous().transpose(2, 3), go, table, None)
    _check(q, k, v, go[:, :, :1].expand(B, H, S, D), table, None)
    _check(q, k, v, go, table.t().contiguous().t(), torch.ones(B, 2 * S, dtype=torch.bool)[:, ::2])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("B,H,Hk,Sq,Sk", [(1, 1, 1, 1, 5000), (2, 4, 2, 1, 4097), (1, 16, 16, 3, 2000), (8, 16, 16, 1, 300), (1, 2, 2, 130, 3001)])
def test_few_rows_against_a_long_cache(dt, B, H, Hk, Sq, Sk):
    import torch_vulkan_b200 as tv

    q, k, v, _, table, m = _case(B, H, Hk, Sq, Sk, 64, dt, Sk, "head")
    kw = dict(causal=True, bidirectional=False, q_offset=Sk - Sq)
    o = tv.bucket_bias_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), key_mask=m.cuda(), **kw)
    _near(o, ot.bias_attention(q, k, v, table, key_mask=m, **kw), OUT[dt], "o")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_one_token_at_a_time_matches_the_whole_sequence(dt):
    import torch_vulkan_b200 as tv

    S = 40
    q, k, v, _, table, _ = (t.cuda() if t is not None else None for t in _case(2, 2, 1, S, S, 64, dt, 9))
    whole = tv.bucket_bias_attention(q, k, v, table, causal=True, bidirectional=False)
    for i in range(S):
        one = tv.bucket_bias_attention(q[:, :, i:i + 1], k[:, :, :i + 1], v[:, :, :i + 1], table, causal=True,
                                       bidirectional=False, q_offset=i)
        assert rel_err(one, whole[:, :, i:i + 1]) <= 2 * OUT[dt]


@pytest.mark.gpu
def test_large_scores_and_bias():
    """Scores of +-3000 and a bias of -1e30: no overflow, and a masked-out bucket stays out."""
    q, k, v, go, table, m = _case(1, 2, 2, 200, 200, 64, torch.float32, 4)
    table[5], table[20] = -1e30, 50.0
    ref = ot.bias_attention(q * 20, k * 20, v, table)
    import torch_vulkan_b200 as tv

    o = tv.bucket_bias_attention((q * 20).cuda(), (k * 20).cuda(), v.cuda(), table.cuda())
    # scores of 3000 carry 3000 * 2^-23 of absolute error into the exponent, a handful of times
    _near(o, ref, 5e-3, "o")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
def test_no_keys_no_queries(dt):
    q, k, v, go, table, _ = _case(2, 2, 2, 5, 0, 64, dt, 1)
    got = _run(q, k, v, table, None, go)
    assert not got["o"].any() and not got["dq"].any() and got["dk"].shape == (2, 2, 0, 64) and not got["dtable"].any()
    q, k, v, go, table, _ = _case(2, 2, 2, 0, 5, 64, dt, 1)
    got = _run(q, k, v, table, None, go)
    assert got["o"].numel() == 0 and not got["dk"].any() and not got["dv"].any() and not got["dtable"].any()


@pytest.mark.gpu
def test_gradients_against_differences():
    import torch_vulkan_b200 as tv

    q, k, v, go, table, m = _case(1, 2, 1, 70, 90, 16, torch.float32, 6, "tail")
    got = _run(q, k, v, table, m, go)
    f = lambda *a: (ot.bias_attention(*a, key_mask=m) * go.double()).sum().item()  # noqa: E731
    base = [q.double(), k.double(), v.double(), table.double()]
    g = torch.Generator().manual_seed(1)
    for i, n in enumerate(("dq", "dk", "dv", "dtable")):
        d = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        up = [t + (1e-5 * d if j == i else 0) for j, t in enumerate(base)]
        dn = [t - (1e-5 * d if j == i else 0) for j, t in enumerate(base)]
        num = (f(*up) - f(*dn)) / 2e-5
        ana = (got[n].cpu().double() * d).sum().item()
        # the central difference is good to ~1e-9 relative of f's curvature, the kernel to 3e-5 of the norms
        assert abs(num - ana) <= 3e-5 * (got[n].cpu().double().norm() * d.norm()).item() + 1e-6
    assert tv.validation_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
def test_same_bits_on_every_call_and_on_another_stream(dt):
    q, k, v, go, table, m = _case(2, 4, 2, 300, 420, 64, dt, 8, "random")
    first = _run(q, k, v, table, m, go)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for i in range(3):
        with torch.cuda.stream(s if i % 2 else torch.cuda.current_stream()):
            again = _run(q, k, v, table, m, go)
        torch.cuda.synchronize()
        for n in first:
            assert torch.equal(first[n], again[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_gradients_wanted_one_at_a_time(dt):
    import torch_vulkan_b200 as tv

    q, k, v, go, table, m = _case(2, 2, 2, 150, 150, 64, dt, 8, "tail")
    every = _run(q, k, v, table, m, go)
    for i, n in enumerate(("dq", "dk", "dv", "dtable")):
        leaf = [t.cuda().detach().requires_grad_(j == i) for j, t in enumerate((q, k, v, table))]
        o = tv.bucket_bias_attention(*leaf, key_mask=m.cuda())
        (g,) = torch.autograd.grad(o, leaf[i], go.cuda())
        assert torch.equal(g, every[n]), n
    half = table.to(torch.bfloat16).cuda().requires_grad_(True)
    o = tv.bucket_bias_attention(q.cuda(), k.cuda(), v.cuda(), half, key_mask=m.cuda())
    (g,) = torch.autograd.grad(o, half, go.cuda())
    assert g.dtype == torch.bfloat16 and g.shape == table.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S", [200, 512])
def test_bias_gradient_keeps_fp32_accuracy(dt, S):
    """With 16-bit tensors the bias gradient is still a sum of fp32 dS: the two exponent terms carry |x| 2^-23 each
    (|x| < 16 here) and delta is a sum of D fp32 products, so it is within 2^-17 of the magnitudes of dP - delta's sums."""
    q, k, v, go, table, m = _case(2, 4, 4, S, S, 64, dt, S, "tail")
    ref = ot.bias_attention(q, k, v, table, key_mask=m, go=go)
    got = _run(q, k, v, table, m, go)["dtable"].cpu().double()
    assert bool(((got - ref["dtable"]).abs() <= 2.0 ** -17 * (ref["dtable_abs"] + ref["ds_abs"]) + 1e-9).all())


@pytest.mark.gpu
def test_refusals():
    import torch_vulkan_b200 as tv

    q, k, v, _, table, _ = (t.cuda() if t is not None else None for t in _case(2, 4, 2, 8, 9, 64, torch.bfloat16, 1))
    f = tv.bucket_bias_attention
    ok = torch.ones(2, 9, dtype=torch.bool, device="cuda")
    f(q, k, v, table, key_mask=ok)
    wide = torch.zeros(2, 4, 8, 136, device="cuda", dtype=torch.bfloat16)
    bad = [lambda: f(q.cpu(), k, v, table), lambda: f(q.cpu(), k.cpu(), v.cpu(), table.cpu()), lambda: f(q.float(), k, v, table),
           lambda: f(q.double(), k.double(), v.double(), table), lambda: f(q[0], k, v, table), lambda: f(q[:1], k, v, table),
           lambda: f(q, k, v[:, :, :8], table), lambda: f(q[:, :3], k, v, table[:, :3]), lambda: f(q, k, v, table[:, :3]),
           lambda: f(q, k, v, table.int()), lambda: f(q, k, v, table[:31]), lambda: f(q, k, v, table[:2]),
           lambda: f(q, k, v, torch.zeros(130, 4, device="cuda")), lambda: f(q, k, v, table, max_distance=8),
           lambda: f(q, k, v, table, max_distance=1025), lambda: f(q, k, v, table, key_mask=ok.int()),
           lambda: f(q, k, v, table, key_mask=ok[:, :8]), lambda: f(q, k, v, table, key_mask=ok.cpu()),
           lambda: f(q, k, v, table, q_offset=1 << 40), lambda: f(wide, wide, wide, table),
           lambda: tv.relative_position_bucket(3, num_buckets=31), lambda: tv.relative_position_bucket(3, num_buckets=256)]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
            pytest.fail(f"refusal {i} did not happen")
    assert tv.validation_errors() == 0


def test_buckets_equal_whole_number_arithmetic():
    """Every distance of many parameter sets: the library's thresholds against exact powers."""
    import torch_vulkan_b200 as tv

    sets = [(32, 128, True), (32, 128, False), (2, 2, False), (4, 2, True), (64, 256, True), (16, 64, False), (128, 1024, False),
            (128, 1024, True), (6, 17, True), (7, 100, False), (10, 81, True), (24, 1000, False), (12, 27, True), (96, 729, True)]
    for nb, dist, bidir in sets:
        for rel in list(range(-dist - 3, dist + 4)) + [-(1 << 29), 1 << 29]:
            assert tv.relative_position_bucket(rel, nb, dist, bidir) == ot.bucket(rel, nb, dist, bidir), (nb, dist, bidir, rel)


def test_bucket_known_values():
    import torch_vulkan_b200 as tv

    assert [tv.relative_position_bucket(-d) for d in (0, 7, 8, 11, 12, 16, 64, 127, 128, 4000)] == [0, 7, 8, 8, 9, 10, 14, 15, 15, 15]
    assert [tv.relative_position_bucket(d) for d in (1, 8, 4000)] == [17, 24, 31]
    assert tv.relative_position_bucket(5, bidirectional=False) == 0


def test_c_entry_points_refuse_bad_arguments():
    import ctypes

    import torch_vulkan_b200 as tv

    lib = ctypes.CDLL(tv._LIB_PATH)
    assert lib.b2_bias_attn_fwd(None, None) < 0 and lib.b2_bias_attn_bwd(None, None) < 0
    assert lib.b2_bias_bucket(ctypes.c_int64(3), 31, 128, 1) == -1 and lib.b2_bias_bucket(ctypes.c_int64(3), 32, 2000, 1) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", [(2, 16, 2, 1, 700, 128), (1, 12, 1, 1, 130, 40), (1, 10, 2, 3, 515, 96), (2, 8, 1, 7, 1000, 64),
                                            (1, 40, 1, 1, 65, 8), (1, 6, 2, 8, 2049, 80), (3, 3, 3, 5, 17, 64)])
def test_few_queries_of_heads_that_share_their_keys(dt, B, H, Hk, Sq, Sk, D):
    """Rows of several heads and queries side by side, causal and not, with one sample that sees no key."""
    import torch_vulkan_b200 as tv

    q, k, v, _, table, m = _case(B, H, Hk, Sq, Sk, D, dt, H + Sk, "random")
    for mask, kw in ((m, {}), (None, dict(causal=True, bidirectional=False, q_offset=Sk - Sq)),
                     (m, dict(causal=True, q_offset=2))):  # most keys lie past the last query
        o = tv.bucket_bias_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), key_mask=None if mask is None else mask.cuda(), **kw)
        _near(o, ot.bias_attention(q, k, v, table, key_mask=mask, **kw), OUT[dt], "o")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
def test_a_masked_key_of_a_cache_may_hold_anything(dt):
    import torch_vulkan_b200 as tv

    q, k, v, _, table, m = _case(2, 8, 2, 2, 300, 64, dt, 21, "tail")
    ref = ot.bias_attention(q, k, v, table, key_mask=m)
    k, v = k.clone(), v.clone()
    k.masked_fill_(~m[:, None, :, None], float("nan"))
    v.masked_fill_(~m[:, None, :, None], float("inf"))
    o = tv.bucket_bias_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), key_mask=m.cuda())
    _near(o, ref, OUT[dt], "o")


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 100])
def test_in_a_graph(Sq):
    """Captured once, replayed on new values: the same bits as the call itself."""
    import torch_vulkan_b200 as tv

    q, k, v, _, table, _ = (t.cuda() if t is not None else None for t in _case(2, 4, 2, Sq, 1500, 64, torch.bfloat16, 3))
    kw = dict(causal=True, bidirectional=False, q_offset=1500 - Sq)
    tv.bucket_bias_attention(q, k, v, table, **kw)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = tv.bucket_bias_attention(q, k, v, table, **kw)
    q.copy_(torch.randn_like(q))
    table.add_(1.0).mul_(0.5)
    g.replay()
    assert torch.equal(o, tv.bucket_bias_attention(q, k, v, table, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [40, 64, 128])
def test_long_rows_keep_their_sum(dt, D):
    """Long rows in one piece (enough blocks that the keys are not split), with values of one sign: a sum that is cut short at every
    step would show. A 16-wide step of the product may lose 2^-23 of the sum; 1024 keys are 64 steps of P's two halves, 2^-16,
    and P is good to 2^-17."""
    q, k, v, go, table, m = _case(4, 70, 70, 40, 2048, D, dt, D, "tail")
    v = v.abs()
    ref = ot.bias_attention(q, k, v, table, key_mask=m, go=go)
    got = _run(q, k, v, table, m, go)
    _near(got["o"], ref["o"], OUT[dt], "o")
    err = (got["dtable"].cpu().double() - ref["dtable"]).abs()
    bound = (2.0 ** -16 + 2.0 ** -17) * ref["dtable_abs"] + 2.0 ** -14 * ref["ds_abs"] + 1e-7
    assert bool((err <= bound).all()), f"dtable: {(err / bound).max().item():.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("Sq,Sk,causal", [(1500, 14, False), (300, 1, False), (7, 1200, True), (260, 700, False)])
def test_bias_gradient_where_one_bucket_has_most_keys(dt, Sq, Sk, causal):
    """Many rows have all their keys in the bucket beyond max_distance, where the row's dS cancels: the bound of every bucket still
    holds, and a single key, whose P is 1, gives no gradient at all."""
    q, k, v, go, table, m = _case(2, 4, 2, Sq, Sk, 64, dt, Sq + Sk, "tail")
    for bidirectional in (True, False):
        kw = dict(causal=causal, bidirectional=bidirectional, q_offset=Sk - Sq if causal else 0)
        got = _check(q, k, v, go, table, m, **kw)
        if Sk == 1:
            assert not got["dtable"].any()
