"""The 4-bit linears at the ends of their ranges."""

import pytest
import torch

import oracle.text as ot
from tests.test_mx4 import BF, _close, _linear_case


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 3, 8, 40])
def test_the_largest_activations(m):
    """Sums of products whose scale alone passes fp32's range: the weight's scale brings them back, for few rows as for many."""
    import torch_vulkan_b200 as tv

    x, w, _, _, _, _ = _linear_case(m, 256, 96, m)
    x = (x.float() / x.float().abs().max() * 3e38).to(BF)
    y = tv.mx4_linear(x.cuda(), tv.mx4_quantize((w.float() * 2.0 ** -10).to(BF).cuda()))
    xq, wq = ot.mx4_round(x), ot.mx4_round((w.float() * 2.0 ** -10).to(BF))
    assert (xq.abs() @ wq.abs().t()).max() < 3e38
    _close(y, xq @ wq.t(), xq.abs() @ wq.abs().t())


@pytest.mark.gpu
def test_no_output_features_and_no_rows():
    import torch_vulkan_b200 as tv

    for m, n in ((5, 0), (0, 40), (0, 0)):
        w = tv.mx4_quantize(torch.randn(n, 64, device="cuda"))
        x = torch.randn(m, 64, device="cuda").bfloat16().requires_grad_(True)
        a, b, bias = (torch.randn(*s, device="cuda").bfloat16().requires_grad_(True) for s in ((8, 64), (n, 8), (n,)))
        for y, leaf in ((tv.mx4_linear(x, w, bias), (x, bias)), (tv.mx4_lora_linear(x, w, bias, a, b), (x, a, b, bias))):
            assert y.shape == (m, n)
            for t, g in zip(leaf, torch.autograd.grad(y, leaf, torch.ones_like(y))):
                assert g.shape == t.shape and not g.any()


def test_lora_ranks_that_do_not_fit_are_refused_by_the_constructors():
    """Before anything is built: on the CPU."""
    from torch_vulkan_b200.dit import DiTBlock, LoRAMx4Linear
    from torch_vulkan_b200.text_encoder import TextEncoder

    for rank in (0, 4, 12, 24, 32, 128):
        with pytest.raises(ValueError, match="at most 16 where 3"):
            DiTBlock(hidden=256, heads=2, text_dim=128, mlp=512, rank=rank, base="mx4", device="cpu")
    for rank in (4, 40, 64):
        with pytest.raises(ValueError, match="at most 32 where 2"):
            TextEncoder(blocks=1, hidden=256, heads=4, mlp=512, rank=rank, device="cpu")
    for rank in (4, 72):
        with pytest.raises(ValueError, match="at most 64"):
            LoRAMx4Linear(64, 64, rank=rank, device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 16])
def test_lora_ranks_that_fit(rank):
    from torch_vulkan_b200.dit import DiTBlock, synthetic_batch
    from torch_vulkan_b200.text_encoder import TextEncoder

    x, text, cond, _ = synthetic_batch(tokens=64, text_tokens=32, hidden=256, text_dim=128, seed=7)
    assert torch.isfinite(DiTBlock(hidden=256, heads=2, text_dim=128, mlp=512, rank=rank, base="mx4")(x, text, cond)).all()
    assert torch.isfinite(TextEncoder(blocks=1, hidden=256, heads=4, mlp=512, rank=2 * rank)(x)).all()


def test_lowered_scales_keep_a_nan():
    from torch_vulkan_b200.text_encoder import _shift_scales

    s = torch.tensor([0, 1, 2, 3, 4, 100, 252, 255], dtype=torch.uint8)
    assert _shift_scales(s, 64).tolist() == [0, 0, 0, 0, 1, 97, 249, 255]
    assert _shift_scales(s, 16).tolist() == [0, 0, 0, 1, 2, 98, 250, 255]
