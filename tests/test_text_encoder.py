"""The 4-bit DiT block and the 4-bit text encoder on this package's operators: against a plain float64 restatement with the
same quantised weights, the stacked products against the modules one by one, masking, and joint training steps.

Quantising an activation is a step function: where the kernels' bf16 activations and the restatement's differ by their
rounding (2^-9 relative), about one element in a hundred falls on the other side of a step and moves by up to a third of
itself. sqrt(0.01) / 3, some ten quantised products in a row, adds up to sqrt(10) * 0.033 = 0.1 of the branch outputs."""

import math

import pytest
import torch
import torch.nn.functional as F

import oracle.text as ot

pytestmark = pytest.mark.gpu


def d(t):
    return t.detach().cpu().double()


def ste(x):
    """Q(x) with the straight-through gradient."""
    flat = x.detach().reshape(-1, x.shape[-1]).to(torch.bfloat16)
    return x + (ot.mx4_round(flat).view(x.shape) - x).detach()


def values(base):
    import torch_vulkan_b200 as tv

    return d(tv.mx4_dequantize(base.weight, torch.float32))


def lin(base, x):
    return ste(x) @ values(base).t() + d(base.bias)


def lora(mod, x, p):
    return lin(mod.base, x) + (x @ p[mod, "down"].t()) @ p[mod, "up"].t() * mod.scale


def params_of(mods):
    p = {}
    for m in mods:
        p[m, "down"] = d(m.lora_down).requires_grad_(True)
        p[m, "up"] = d(m.lora_up).requires_grad_(True)
    return p


def rel(a, b):
    return ((d(a) - d(b)).norm() / d(b).norm()).item()


def test_encoder_block_against_float64():
    from torch_vulkan_b200.text_encoder import TextEncoderBlock

    blk = TextEncoderBlock(hidden=256, heads=4, mlp=512, seed=2)
    g = torch.Generator().manual_seed(1)
    B, S = 2, 70
    x = torch.randn(B, S, 256, generator=g).to(torch.bfloat16)
    table = torch.randn(32, 4, generator=g)
    mask = torch.arange(S)[None, :] < torch.tensor([S, 41])[:, None]
    go = (torch.randn(B, S, 256, generator=g) * mask[..., None]).to(torch.bfloat16)
    xd, td = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
    y = blk(xd, td, mask.cuda())
    y.backward(go.cuda())

    p = params_of((blk.q, blk.k, blk.v, blk.o))
    X, T = d(x).requires_grad_(True), d(table).requires_grad_(True)
    h = F.layer_norm(X, (256,), eps=1e-6)
    split = lambda t: t.view(B, S, 4, 64).transpose(1, 2)  # noqa: E731
    q, k, v = (split(lora(m, h, p)) for m in (blk.q, blk.k, blk.v))
    bk = torch.tensor([[ot.bucket(j - i, 32, 128, True) for j in range(S)] for i in range(S)])
    s = q @ k.transpose(-1, -2) + T[bk].permute(2, 0, 1)
    a = torch.softmax(s.masked_fill(~mask[:, None, None, :], -math.inf), -1) @ v
    z = X + lora(blk.o, a.transpose(1, 2).reshape(B, S, 256), p)
    ref = z + lin(blk.fc2, F.gelu(lin(blk.fc1, F.layer_norm(z, (256,), eps=1e-6)), approximate="tanh"))
    ref.backward(d(go))
    live = mask[..., None].expand_as(x)
    assert rel(y.cpu()[live], ref[live]) <= 0.05  # the residual stream carries most of it
    assert rel(xd.grad, X.grad) <= 0.1
    for m in (blk.q, blk.k, blk.v, blk.o):
        assert rel(m.lora_down.grad, p[m, "down"].grad) <= 0.1 and rel(m.lora_up.grad, p[m, "up"].grad) <= 0.1
    assert rel(td.grad, T.grad) <= 0.1


def test_encoder_ignores_padding_and_zeroes_it():
    from torch_vulkan_b200.text_encoder import TextEncoder

    enc = TextEncoder(blocks=2, hidden=256, heads=4, mlp=512, seed=3)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 50, 256, generator=g).to(torch.bfloat16).cuda()
    mask = torch.arange(50, device="cuda")[None, :] < torch.tensor([50, 23], device="cuda")[:, None]
    y = enc(x, mask)
    x2 = x.clone()
    x2[1, 23:] = 7.0
    assert torch.equal(enc(x2, mask), y)
    assert not y[1, 23:].any() and y[1, :23].any()
    short = enc(x[1:, :23].contiguous(), None)
    assert rel(short[0], y[1, :23]) <= 0.02  # other tiles, other rounding of the same sums


def test_dit_block_stacked_products_equal_the_modules():
    from torch_vulkan_b200.dit import DiTBlock, synthetic_batch

    blk = DiTBlock(hidden=256, heads=2, text_dim=128, mlp=512, seed=3, base="mx4")
    x, _, _, _ = synthetic_batch(tokens=128, text_tokens=64, hidden=256, text_dim=128, seed=4)
    q, k, v = blk._stacked("qkv", x, (blk.q, blk.k, blk.v))
    for got, m in zip((q, k, v), (blk.q, blk.k, blk.v)):
        # the block-diagonal up-projection adds zeros to the same sums: fp32 order apart, then one bf16 rounding
        assert torch.allclose(got.float(), m(x).float(), rtol=2.0 ** -7, atol=1e-3)
    go = torch.randn(128, 3 * 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda().view(1, 128, 768)
    blk.zero_grad(set_to_none=True)
    xs = x.clone().requires_grad_(True)
    blk._stacked("qkv", xs, (blk.q, blk.k, blk.v), whole=True).backward(go)
    got = {n: p.grad.clone() for n, p in blk.named_parameters() if p.grad is not None}
    blk.zero_grad(set_to_none=True)
    xm = x.clone().requires_grad_(True)
    torch.cat([m(xm) for m in (blk.q, blk.k, blk.v)], -1).backward(go)
    assert rel(xs.grad, xm.grad) <= 0.02  # three rounded dX added in bf16 against one sum
    for n, p in blk.named_parameters():
        if p.grad is not None:
            assert rel(got[n], p.grad) <= 2.0 ** -6, n


def test_dit_block_against_float64():
    from tests.test_dit import oracle
    from torch_vulkan_b200.dit import DiTBlock, synthetic_batch

    blk = DiTBlock(hidden=256, heads=2, text_dim=128, mlp=512, seed=3, base="mx4")
    x, text, cond, target = synthetic_batch(tokens=128, text_tokens=64, hidden=256, text_dim=128, seed=4)
    out = blk(x, text, cond)
    p = params_of((blk.q, blk.k, blk.v, blk.o, blk.cq, blk.ck, blk.cv, blk.co))
    X, T, C = d(x), d(text), d(cond)
    sh1, sc1, g1, sh2, sc2, g2, sh3, sc3, g3 = lin(blk.ada, F.silu(C)).unsqueeze(1).chunk(9, -1)
    ln = lambda t, sh, sc: F.layer_norm(t, (256,), eps=1e-6) * (1 + sc) + sh  # noqa: E731

    def attn(tq, tk, qm, km, vm, om):
        hd = lambda t: t.view(1, t.shape[1], 2, 128).transpose(1, 2)  # noqa: E731
        o, _ = oracle.sdpa_fwd(hd(lora(qm, tq, p)), hd(lora(km, tk, p)), hd(lora(vm, tk, p)))
        return lora(om, o.transpose(1, 2).reshape(1, -1, 256), p)

    with torch.no_grad():
        h = ln(X, sh1, sc1)
        z = X + g1 * attn(h, h, blk.q, blk.k, blk.v, blk.o)
        z = z + g2 * attn(ln(z, sh2, sc2), T, blk.cq, blk.ck, blk.cv, blk.co)
        z = z + g3 * lin(blk.fc2, F.gelu(lin(blk.fc1, ln(z, sh3, sc3)), approximate="tanh"))
    assert rel(out, z) <= 0.05
    with pytest.raises(ValueError):
        DiTBlock(hidden=192, heads=2, text_dim=128, mlp=512, base="mx4")
    with pytest.raises(ValueError):
        DiTBlock(hidden=256, heads=2, text_dim=128, mlp=512, base="int2")


@pytest.mark.parametrize("base", ["int8", "mx4"])
def test_joint_training_steps_reduce_the_loss(base):
    import torch_vulkan_b200 as tv
    from torch_vulkan_b200.dit import DiTStack, synthetic_batch
    from torch_vulkan_b200.text_encoder import ConditionedTrainer, TextEncoder

    enc = TextEncoder(blocks=2, hidden=256, heads=4, mlp=512, seed=5)
    model = DiTStack(blocks=1, seed=6, hidden=256, heads=2, text_dim=256, mlp=512, base=base)
    tokens, _, cond, _ = synthetic_batch(tokens=64, text_tokens=8, hidden=256, text_dim=256, seed=7)
    x, _, _, target = synthetic_batch(tokens=128, text_tokens=8, hidden=256, text_dim=256, seed=8)
    mask = torch.arange(64, device="cuda")[None, :] < 50
    before = enc.table.detach().clone()
    up = enc.blocks[0].q.lora_up.detach().clone()
    tv.reset_counts()
    tr = ConditionedTrainer(enc, model, lr=3e-3)
    losses = [tr.step(tokens, mask, x, cond, target).item() for _ in range(12)]
    assert all(math.isfinite(v) for v in losses) and min(losses[-3:]) < losses[0] - 1e-4
    assert not torch.equal(enc.table, before) and not torch.equal(enc.blocks[0].q.lora_up, up)
    kc = tv.kernel_counts()
    for op in ("b2::bias_attn_fwd", "b2::bias_attn_bwd", "b2::mx4_lora_linear", "b2::mx4_lora_dx", "b2::mx4_linear", "b2::mx4_linear_dx"):
        assert kc.get(op, 0) >= 1, (op, kc)
    assert tv.validation_errors() == 0
