"""4-bit blocks under activation checkpointing and block swap: both point the buffers that a product's backward reads at other
memory, and neither may change a bit of the loss or of a gradient."""

import pytest
import torch
import torch.nn.functional as F

BF = torch.bfloat16


@pytest.mark.gpu
def test_checkpointing_changes_nothing():
    from torch_vulkan_b200.dit import DiTStack, synthetic_batch

    x, text, cond, target = synthetic_batch(tokens=128, text_tokens=64, hidden=256, text_dim=128, seed=7)
    grads = []
    for checkpoint in (False, True):
        model = DiTStack(blocks=2, seed=0, hidden=256, heads=2, text_dim=128, mlp=512, base="mx4", checkpoint=checkpoint)
        F.mse_loss(model(x, text, cond).float(), target.float()).backward()
        grads.append([p.grad for p in model.lora_parameters()])
    assert all(torch.equal(a, b) and a.any() for a, b in zip(*grads))


@pytest.mark.gpu
@pytest.mark.parametrize("swap,ring", [(2, 1), (3, 2)])
def test_swapped_blocks_equal_resident_ones(swap, ring):
    from torch_vulkan_b200.dit import DiTStack, synthetic_batch

    kw = dict(blocks=3, seed=0, hidden=256, heads=2, text_dim=128, mlp=512, base="mx4")
    x, text, cond, target = synthetic_batch(tokens=128, text_tokens=64, hidden=256, text_dim=128, seed=7)

    def run(model):
        res = []
        for _ in range(2):
            for p in model.lora_parameters():
                p.grad = None
            loss = F.mse_loss(model(x, text, cond).float(), target.float())
            loss.backward()
            res.append((loss.item(), [p.grad.detach().clone() for p in model.lora_parameters()]))
        return res

    ref = run(DiTStack(checkpoint=True, **kw))
    model = DiTStack(**kw)
    off = model.enable_block_swap(swap, ring_size=ring)
    for (lr, gr), (lg, gg) in zip(ref, run(model)):
        assert lr == lg and all(torch.equal(a, b) for a, b in zip(gr, gg))
    assert off.h2d_copies >= 2 * swap


@pytest.mark.gpu
def test_a_checkpointed_encoder_block_changes_nothing():
    from torch.utils.checkpoint import checkpoint

    from torch_vulkan_b200.text_encoder import TextEncoderBlock

    blk = TextEncoderBlock(hidden=256, heads=4, mlp=512, seed=2)
    x = torch.randn(2, 70, 256, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    table = torch.randn(32, 4, generator=torch.Generator().manual_seed(2)).cuda()
    mask = torch.arange(70, device="cuda")[None, :] < torch.tensor([70, 41], device="cuda")[:, None]
    grads = []
    for on in (False, True):
        xs, ts = x.clone().requires_grad_(True), table.clone().requires_grad_(True)
        blk.zero_grad(set_to_none=True)
        y = checkpoint(blk, xs, ts, mask, use_reentrant=False) if on else blk(xs, ts, mask)
        y.float().pow(2).sum().backward()
        grads.append([xs.grad, ts.grad] + [p.grad for p in blk.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
