"""What the embeddings of padded tokens hold, NaN included, reaches neither the encoder's output nor a gradient."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 7.0])
def test_padding_may_hold_anything(bad):
    from torch_vulkan_b200.text_encoder import TextEncoder

    enc = TextEncoder(blocks=2, hidden=256, heads=4, mlp=512, seed=3)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 50, 256, generator=g).to(torch.bfloat16).cuda()
    go = torch.randn(3, 50, 256, generator=g).to(torch.bfloat16).cuda()
    mask = torch.arange(50, device="cuda")[None, :] < torch.tensor([50, 23, 0], device="cuda")[:, None]

    def run(x):
        enc.zero_grad(set_to_none=True)
        xs = x.clone().requires_grad_(True)
        y = enc(xs, mask)
        y.backward(go)
        return [y.detach(), xs.grad] + [p.grad for p in enc.trainable_parameters()]

    clean = run(x)
    assert not clean[0][~mask].any() and not clean[1][~mask].any() and all(torch.isfinite(t).all() for t in clean)
    dirty = run(x.masked_fill(~mask.unsqueeze(-1), bad))
    assert all(torch.equal(a, b) for a, b in zip(clean, dirty))
