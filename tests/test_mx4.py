"""MXFP4 quantisation, read-back and the 4-bit linear against float64: codes and scales bit for bit, products within
the bounds that their roundings give.

Bounds of the products (bf16 outputs, element products exact, fp32 sums): one rounding of the output is at most
2^-8 |y|, a sum of magnitudes A that is accumulated in fp32 in any order and alignment moves by at most 2^-20 A at these
lengths, and the LoRA term reads its hidden activation rounded to bf16, 2^-8 of its own magnitudes."""

import ctypes
import os

import pytest
import torch

import oracle.text as ot

BF = torch.bfloat16


def _x(rows, cols, dt, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * std
    x *= torch.exp2(torch.randint(-6, 7, (rows, (cols + 31) // 32), generator=g).float()).repeat_interleave(32, 1)[:, :cols]
    return x.to(dt)


def _scale_index(rows, cols):
    r, j = torch.arange(rows)[:, None], torch.arange((cols + 31) // 32)[None, :]
    return (r // 128, j // 4, r % 32, r % 128 // 32, j % 4)


def _unpack(w):
    rows, cols = w.shape
    c = w.codes.cpu().long()
    codes = torch.stack([c & 15, c >> 4], -1).reshape(rows, -1)
    scales = w.scales.cpu().long()[_scale_index(rows, cols)]
    return codes, scales


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, BF, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 33), (5, 7), (128, 128), (129, 160), (257, 1000), (64, 2048)])
def test_quantize_bits(dt, rows, cols):
    import torch_vulkan_b200 as tv

    x = _x(rows, cols, dt, rows * 1000 + cols)
    w = tv.mx4_quantize(x.cuda())
    codes, scales = _unpack(w)
    rc, rs = ot.mx4_quantize(x)
    assert torch.equal(codes[:, :cols], rc) and torch.equal(scales, rs)
    assert not codes[:, cols:].any()  # columns of padding hold zero codes
    used = torch.zeros(w.scales.shape, dtype=torch.bool)
    used[_scale_index(rows, cols)] = True
    assert not w.scales.cpu()[~used].any()  # and unused scales are zero
    for out in (torch.float32, BF):
        assert torch.equal(tv.mx4_dequantize(w, out).cpu().double(), ot.mx4_values(rc, rs))
    assert w.shape == (rows, cols)


@pytest.mark.gpu
def test_quantize_every_rounding_case():
    """Every tie and its neighbours in units of the scale, with the largest magnitude 4 so that the scale is 1, at
    three scales; a zero block; the largest and smallest numbers of fp32."""
    import torch_vulkan_b200 as tv

    t = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 4.0])
    near = torch.cat([t, torch.nextafter(t, torch.zeros(1)), torch.nextafter(t[:6], torch.full((1,), 9.0)), torch.zeros(12)])
    big = torch.tensor([5.0, 5.0000005, 4.9999995, 6.0, 7.0, 7.9999995] + [0.0] * 26)
    rows = [near, -near, near * 2.0 ** 100, near * 2.0 ** -100, big, -big, torch.zeros(32),
            torch.full((32,), torch.finfo(torch.float32).max), torch.full((32,), 2.0 ** -149),
            torch.cat([torch.tensor([2.0 ** -126, 2.0 ** -127, 2.0 ** -128, 2.0 ** -129, 2.0 ** -130]), torch.zeros(27)])]
    x = torch.stack(rows)
    codes, scales = _unpack(tv.mx4_quantize(x.cuda()))
    rc, rs = ot.mx4_quantize(x)
    assert torch.equal(codes, rc) and torch.equal(scales, rs)


@pytest.mark.gpu
def test_quantize_non_finite_blocks_read_back_as_nan():
    import torch_vulkan_b200 as tv

    x = _x(4, 96, torch.float32, 3)
    x[0, 40], x[1, 5], x[3, 95] = float("inf"), float("nan"), -float("inf")
    w = tv.mx4_quantize(x.cuda())
    codes, scales = _unpack(w)
    rc, rs = ot.mx4_quantize(x)
    assert torch.equal(codes, rc) and torch.equal(scales, rs)
    back = tv.mx4_dequantize(w, torch.float32).cpu()
    assert torch.equal(torch.isnan(back), (rs == 255).repeat_interleave(32, 1))
    # and a product with such a block is NaN in its row alone
    y = tv.mx4_linear(x.to(BF).cuda(), tv.mx4_quantize(_x(64, 96, BF, 4).cuda()))
    assert torch.equal(torch.isnan(y).any(1).cpu(), torch.tensor([True, True, False, True]))
    assert torch.equal(torch.isnan(y).all(1).cpu(), torch.tensor([True, True, False, True]))


@pytest.mark.gpu
def test_quantize_strided_rows_and_offsets():
    import torch_vulkan_b200 as tv

    x = _x(40, 200, BF, 7)
    for view in (lambda t: t[:, 8:136], lambda t: t[:, 3:70], lambda t: t[::2, :64], lambda t: t.t(), lambda t: t[1:2].expand(6, 200)):
        codes, scales = _unpack(tv.mx4_quantize(view(x.cuda())))
        rc, rs = ot.mx4_quantize(view(x))
        assert torch.equal(codes[:, :rc.shape[1]], rc) and torch.equal(scales, rs)


def _linear_case(m, k, n, seed, r=0):
    x = _x(m, k, BF, seed, 0.5)
    w = _x(n, k, BF, seed + 1, 0.02)
    g = torch.Generator().manual_seed(seed + 2)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    bias, gy = (rnd(n)).to(BF), (rnd(m, n) * 0.1).to(BF)
    a = (rnd(r, k) * k ** -0.5).to(BF) if r else None
    b = (rnd(n, r) * 0.1).to(BF) if r else None
    return x, w, bias, gy, a, b


def _close(got, ref, mags, rounded=0.0):
    err = (got.detach().cpu().double() - ref).abs()
    tol = 2.0 ** -8 * ref.abs() + 2.0 ** -20 * mags + 2.0 ** -8 * rounded + 1e-30
    assert got.shape == ref.shape and bool((err <= tol).all()), f"worst {(err / tol).max().item():.3g} of the bound"


SHAPES = [(1, 32, 8), (1, 2048, 512), (2, 1000, 1111), (5, 64, 130), (8, 96, 257), (9, 4096, 96), (17, 33, 40), (64, 160, 128),
          (128, 256, 256), (130, 640, 300), (231, 1000, 1111), (300, 2048, 520), (512, 512, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_forward_and_dx(m, k, n):
    import torch_vulkan_b200 as tv

    x, w, bias, gy, _, _ = _linear_case(m, k, n, m + k + n)
    xq, wq = ot.mx4_round(x), ot.mx4_round(w)
    xd = x.cuda().requires_grad_(True)
    bd = bias.cuda().requires_grad_(True)
    wd = tv.mx4_quantize(w.cuda())
    y = tv.mx4_linear(xd, wd, bd)
    _close(y, xq @ wq.t() + bias.double(), xq.abs() @ wq.abs().t() + bias.double().abs())
    y.backward(gy.cuda())
    _close(xd.grad, gy.double() @ wq, gy.double().abs() @ wq.abs())
    # torch's own bf16 sum makes the bias gradient
    assert torch.allclose(bd.grad.cpu().double(), gy.double().sum(0), rtol=2e-2, atol=2e-2 * m ** 0.5 * 0.1)
    with torch.no_grad():
        _close(tv.mx4_linear(xd, wd), xq @ wq.t(), xq.abs() @ wq.abs().t())
        lead = tv.mx4_linear(xd.view(1, m, k), wd)
        assert lead.shape == (1, m, n) and torch.equal(lead[0], tv.mx4_linear(xd, wd))


@pytest.mark.gpu
@pytest.mark.parametrize("r", [8, 16, 48, 64])
@pytest.mark.parametrize("m,k,n", [(1, 64, 48), (77, 256, 512), (200, 136, 264), (512, 1024, 640), (33, 100, 50)])
def test_lora_forward_and_gradients(m, k, n, r):
    import torch_vulkan_b200 as tv

    x, w, bias, gy, a, b = _linear_case(m, k, n, m + k + n + r, r)
    xq, wq = ot.mx4_round(x), ot.mx4_round(w)
    xd, ad, bd = (t.cuda().requires_grad_(True) for t in (x, a, b))
    y = tv.mx4_lora_linear(xd, tv.mx4_quantize(w.cuda()), bias.cuda(), ad, bd)
    X, A, Bm, G = (t.double() for t in (x, a, b, gy))
    h, dh = X @ A.t(), G @ Bm
    lo = (X.abs() @ A.abs().t()) @ Bm.abs().t()
    _close(y, xq @ wq.t() + bias.double() + h @ Bm.t(), xq.abs() @ wq.abs().t() + lo, h.abs() @ Bm.abs().t())
    y.backward(gy.cuda())
    ldx = (G.abs() @ Bm.abs()) @ A.abs()
    _close(xd.grad, G @ wq + dh @ A, G.abs() @ wq.abs() + ldx, dh.abs() @ A.abs())
    _close(ad.grad, dh.t() @ X, (G.abs() @ Bm.abs()).t() @ X.abs(), dh.abs().t() @ X.abs())
    _close(bd.grad, G.t() @ h, G.abs().t() @ (X.abs() @ A.abs().t()), G.abs().t() @ h.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 4, 7, 8, 9])
@pytest.mark.parametrize("k,n", [(2048, 700), (40, 33), (4096, 130), (9000, 64)])
def test_few_rows(m, k, n):
    """One to nine rows (the weight-stream kernel and the first size past it), with bias, LoRA and strided rows."""
    import torch_vulkan_b200 as tv

    x, w, bias, _, a, b = _linear_case(m, k, n, m * 7 + k + n, 16)
    xq, wq = ot.mx4_round(x), ot.mx4_round(w)
    wd = tv.mx4_quantize(w.cuda())
    h = x.double() @ a.double().t()
    ref = xq @ wq.t() + bias.double()
    _close(tv.mx4_linear(x.cuda(), wd, bias.cuda()), ref, xq.abs() @ wq.abs().t() + bias.double().abs())
    _close(tv.mx4_lora_linear(x.cuda(), wd, bias.cuda(), a.cuda(), b.cuda()), ref + h @ b.double().t(),
           xq.abs() @ wq.abs().t() + (x.double().abs() @ a.double().abs().t()) @ b.double().abs().t(), h.abs() @ b.double().abs().t())
    wide = torch.randn(m, k + 3).to(BF).cuda()
    assert torch.equal(tv.mx4_linear(wide[:, 3:], wd), tv.mx4_linear(wide[:, 3:].contiguous(), wd))


@pytest.mark.gpu
def test_few_rows_extreme_scales():
    """Blocks with scales from 2^-120 to 2^100, zero blocks and a NaN row."""
    import torch_vulkan_b200 as tv

    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(3, 256, generator=g), torch.randn(50, 256, generator=g)
    e = torch.randint(-60, 50, (1, 8), generator=g).float()
    x *= torch.exp2(e).repeat_interleave(32, 1)
    w *= torch.exp2(-e - 3).repeat_interleave(32, 1)
    w[:, 64:96] = 0
    x, w = x.to(BF), w.to(BF)
    x[1, 7] = float("nan")
    y = tv.mx4_linear(x.cuda(), tv.mx4_quantize(w.cuda()))
    assert torch.isnan(y[1]).all()
    xq, wq = ot.mx4_round(x)[[0, 2]], ot.mx4_round(w)
    _close(y[[0, 2]], xq @ wq.t(), xq.abs() @ wq.abs().t())


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,r", [(2100, 288, 2500, 24), (2100, 2500, 288, 16), (4096, 160, 1300, 8)])
def test_many_tiles(m, k, n, r):
    """Enough 256 x 256 tiles for CTA pairs, ragged in every direction, several tiles a pair."""
    import torch_vulkan_b200 as tv

    x, w, bias, gy, a, b = _linear_case(m, k, n, m + k + n, r)
    xq, wq = ot.mx4_round(x), ot.mx4_round(w)
    xd = x.cuda().requires_grad_(True)
    wd = tv.mx4_quantize(w.cuda())
    X, A, Bm, G = (t.double() for t in (x, a, b, gy))
    h, dh = X @ A.t(), G @ Bm
    _close(tv.mx4_linear(xd, wd, bias.cuda()), xq @ wq.t() + bias.double(), xq.abs() @ wq.abs().t() + bias.double().abs())
    if k % 8 == 0:
        y = tv.mx4_lora_linear(xd, wd, bias.cuda(), a.cuda(), b.cuda())
        _close(y, xq @ wq.t() + bias.double() + h @ Bm.t(), xq.abs() @ wq.abs().t() + (X.abs() @ A.abs().t()) @ Bm.abs().t(),
               h.abs() @ Bm.abs().t())
        y.backward(gy.cuda())
        _close(xd.grad, G @ wq + dh @ A, G.abs() @ wq.abs() + (G.abs() @ Bm.abs()) @ A.abs(), dh.abs() @ A.abs())
    else:
        tv.mx4_linear(xd, wd).backward(gy.cuda())
        _close(xd.grad, G @ wq, G.abs() @ wq.abs())


@pytest.mark.gpu
def test_dx_is_the_derivative_along_the_weight():
    """y is linear in the quantised activation, so replacing Q(x) by another quantised x' moves sum(gy * y) by exactly
    (x' - x) . dx: a difference test at inputs that quantisation leaves as they are."""
    import torch_vulkan_b200 as tv

    m, k, n = 24, 96, 72
    x, w, _, gy, _, _ = _linear_case(m, k, n, 5)
    x0 = ot.mx4_round(x).to(BF)
    x1 = (2.0 * ot.mx4_round(_x(m, k, BF, 99, 0.5))).to(BF)
    wd = tv.mx4_quantize(w.cuda())
    xd = x0.cuda().requires_grad_(True)
    y0 = tv.mx4_linear(xd, wd)
    (dx,) = torch.autograd.grad(y0, xd, gy.cuda())
    y1 = tv.mx4_linear(x1.cuda(), wd)
    lhs = (gy.double() * (y1.cpu().double() - y0.detach().cpu().double())).sum()
    rhs = (dx.cpu().double() * (x1.double() - x0.double())).sum()
    # three bf16-rounded factors of random sign: 2^-8 of the magnitudes, shrunk by the square root of the terms
    tol = 2.0 ** -8 * ((gy.double().abs() * (y1.cpu().double().abs() + y0.cpu().double().abs())).pow(2).sum().sqrt()
                       + (dx.cpu().double() * (x1.double() - x0.double())).pow(2).sum().sqrt()) * 4
    assert abs(lhs - rhs) <= tol


@pytest.mark.gpu
def test_linear_empty_strides_streams_and_repeatability():
    import torch_vulkan_b200 as tv

    w = tv.mx4_quantize(_x(40, 64, BF, 1).cuda())
    assert tv.mx4_linear(torch.empty(0, 64, device="cuda", dtype=BF), w).shape == (0, 40)
    x = _x(70, 128, BF, 2).cuda()
    v = x[:, 64:]
    assert torch.equal(tv.mx4_linear(v, w), tv.mx4_linear(v.contiguous(), w))
    t = _x(64, 70, BF, 3).cuda().t()
    assert torch.equal(tv.mx4_linear(t, w), tv.mx4_linear(t.contiguous(), w))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = tv.mx4_linear(v, w)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        assert torch.equal(y, tv.mx4_linear(v, w))
    # a captured graph replays on new inputs
    xs = v.contiguous()
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        ys = tv.mx4_linear(xs, w)
    new = _x(70, 64, BF, 8).cuda()
    xs.copy_(new)
    g.replay()
    assert torch.equal(ys, tv.mx4_linear(new, w))
    assert tv.validation_errors() == 0


@pytest.mark.gpu
def test_gradients_wanted_one_at_a_time_and_leading_dimensions():
    import torch_vulkan_b200 as tv

    m, k, n, r = 40, 64, 72, 8
    x, w, bias, gy, a, b = (t.cuda() for t in _linear_case(m, k, n, 3, r))
    wd = tv.mx4_quantize(w)
    for with_bias in (True, False):
        args = dict(x=x.view(2, 20, k), bias=bias if with_bias else None, a=a, b=b)
        names = [t for t in args if args[t] is not None]

        def run(wanted):
            leaf = {t: (args[t].detach().requires_grad_(t in wanted) if args[t] is not None else None) for t in args}
            y = tv.mx4_lora_linear(leaf["x"], wd, leaf["bias"], leaf["a"], leaf["b"])
            assert y.shape == (2, 20, n)
            return dict(zip(wanted, torch.autograd.grad(y, [leaf[t] for t in wanted], gy.view(2, 20, n))))

        every = run(names)
        for t in names:
            assert every[t].shape == args[t].shape
            assert torch.equal(run([t])[t], every[t]), t
        for t in names[:2]:
            leaf = {u: args[u].detach().requires_grad_(u == t) if u in names[:2] else None for u in args}
            y = tv.mx4_linear(leaf["x"], wd, leaf["bias"]) if with_bias else tv.mx4_linear(args["x"].detach().requires_grad_(True), wd)
            if with_bias:
                (g,) = torch.autograd.grad(y, leaf[t], gy.view(2, 20, n))
                assert g.shape == args[t].shape
    with torch.no_grad():
        assert not tv.mx4_lora_linear(x, wd, bias, a.requires_grad_(True), b).requires_grad


@pytest.mark.gpu
def test_refusals():
    import torch_vulkan_b200 as tv

    w = tv.mx4_quantize(_x(40, 64, BF, 1).cuda())
    x = _x(8, 64, BF, 2).cuda()
    bad = [lambda: tv.mx4_quantize(x.cpu()), lambda: tv.mx4_quantize(x[0]), lambda: tv.mx4_quantize(x.int()),
           lambda: tv.mx4_dequantize(w, torch.float64), lambda: tv.mx4_dequantize(w._replace(cols=65)),
           lambda: tv.mx4_dequantize(w._replace(scales=w.scales[:0])), lambda: tv.mx4_linear(x.float(), w),
           lambda: tv.mx4_linear(x[:, :32], w), lambda: tv.mx4_linear(x, w, torch.zeros(39, device="cuda", dtype=BF)),
           lambda: tv.mx4_linear(x, w, torch.zeros(40, device="cuda")), lambda: tv.mx4_linear(x, w._replace(codes=w.codes.cpu())),
           lambda: tv.mx4_linear(x, w._replace(codes=w.codes.int())),
           lambda: tv.mx4_lora_linear(x, w, None, torch.zeros(12, 64, device="cuda", dtype=BF), torch.zeros(40, 12, device="cuda", dtype=BF)),
           lambda: tv.mx4_lora_linear(x, w, None, torch.zeros(72, 64, device="cuda", dtype=BF), torch.zeros(40, 72, device="cuda", dtype=BF)),
           lambda: tv.mx4_lora_linear(x, w, None, torch.zeros(8, 64, device="cuda", dtype=BF), torch.zeros(39, 8, device="cuda", dtype=BF))]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()
            pytest.fail(f"refusal {i} did not happen")
    assert tv.validation_errors() == 0


def test_c_entry_points_refuse_bad_arguments():
    lib = ctypes.CDLL(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch_vulkan_b200", "libb2rt.so"))
    lib.b2_mx4_code_bytes.restype = lib.b2_mx4_scale_bytes.restype = ctypes.c_int64
    lib.b2_mx4_code_bytes.argtypes = [ctypes.c_int64]
    lib.b2_mx4_scale_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64]
    for f in (lib.b2_mx4_quantize, lib.b2_mx4_dequantize, lib.b2_mx4_gemm):
        assert f(None, None) < 0
    assert [lib.b2_mx4_code_bytes(c) for c in (0, 1, 32, 33)] == [0, 16, 16, 32]
    assert [lib.b2_mx4_scale_bytes(*c) for c in ((0, 5), (1, 1), (128, 128), (129, 129))] == [0, 512, 512, 2048]


def test_oracle_values():
    """The oracle's own rounding, by hand: scale 2^(2 - 2) for a block whose largest magnitude is 4.x."""
    x = torch.zeros(1, 32)
    x[0, :8] = torch.tensor([4.0, 0.25, -0.75, 1.25, 1.75, 2.5, -3.5, 5.0])
    assert ot.mx4_round(x)[0, :8].tolist() == [4.0, 0.0, -1.0, 1.0, 2.0, 2.0, -4.0, 4.0]
    assert ot.mx4_round(torch.full((1, 32), 7.9))[0, 0].item() == 6.0
