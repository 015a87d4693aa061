"""Text encoder with frozen 4-bit weights, LoRA on its attention projections and a learned relative position bias, and a
training step that trains it together with the DiT it conditions.

Layer layout: LayerNorm, q / k / v / o projections (LoRAMx4Linear, k and v stacked in one product), attention without a score
scale whose positions enter as one learned scalar per head and bucket of distances (tv.bucket_bias_attention; the table is
shared by all layers), LayerNorm, MLP with tanh-GELU (Mx4Linear). The input is the token embeddings [B, S, hidden] with a
mask of the tokens that exist; padded positions come out as zeros, which the DiT's cross-attention reads as they are."""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

import torch_vulkan_b200 as tv

from .dit import LoRAGroup, LoRAMx4Linear, Mx4Linear, check_mx4_rank, make_optimizer, stacked_mx4_lora_forward


class TextEncoderBlock(nn.Module):
    def __init__(self, hidden=1024, heads=16, mlp=4096, rank=16, alpha=16.0, max_distance=128, seed=0, device="cuda"):
        super().__init__()
        if hidden % heads or hidden % 128:
            raise ValueError(f"TextEncoderBlock: hidden {hidden} must be a multiple of 128 and of the {heads} heads")
        check_mx4_rank(rank, 2)  # k and v share a product
        g = torch.Generator(device=device).manual_seed(seed)
        mk = lambda: LoRAMx4Linear(hidden, hidden, rank, alpha, generator=g, device=device)  # noqa: E731
        self.h, self.heads, self.d, self.max_distance = hidden, heads, hidden // heads, max_distance
        self.q, self.k, self.v, self.o = mk(), mk(), mk(), mk()
        self.fc1 = Mx4Linear(hidden, mlp, generator=g, device=device)
        self.fc2 = Mx4Linear(mlp, hidden, generator=g, device=device)
        self.register_buffer("ln1", torch.ones(hidden, dtype=torch.bfloat16, device=device))
        self.register_buffer("ln2", torch.ones(hidden, dtype=torch.bfloat16, device=device))
        for part in ("codes", "scales", "bias"):  # k and v read the same input: one stacked weight, the modules hold views
            full = torch.cat([getattr(m.base, part) for m in (self.k, self.v)], 0)
            self.register_buffer(f"kv_{part}", full)
            half = full.shape[0] // 2
            setattr(self.k.base, part, full[:half])
            setattr(self.v.base, part, full[half:])
        self._kv = LoRAGroup((self.k, self.v))

    def _heads(self, t):
        return t.view(t.shape[0], t.shape[1], self.heads, self.d).transpose(1, 2)

    def forward(self, x, table, key_mask=None):
        h = F.layer_norm(x, (self.h,), weight=self.ln1, eps=1e-6)
        q = self.q(h)
        k, v = stacked_mx4_lora_forward(h, self.kv_codes, self.kv_scales, self.kv_bias, self._kv)
        o = tv.bucket_bias_attention(self._heads(q), self._heads(k), self._heads(v), table, key_mask=key_mask,
                                     max_distance=self.max_distance, scale=1.0)
        x = x + self.o(o.transpose(1, 2).reshape(x.shape))
        h = F.layer_norm(x, (self.h,), weight=self.ln2, eps=1e-6)
        return x + self.fc2(F.gelu(self.fc1(h), approximate="tanh"))


class TextEncoder(nn.Module):
    """A stack of TextEncoderBlock with one trainable bias table [num_buckets, heads] (fp32)."""

    def __init__(self, blocks=2, hidden=1024, heads=16, num_buckets=32, seed=0, device="cuda", **kw):
        super().__init__()
        self.blocks = nn.ModuleList([TextEncoderBlock(hidden, heads, seed=seed + i, device=device, **kw) for i in range(blocks)])
        g = torch.Generator().manual_seed(seed + 1000)
        self.table = nn.Parameter((0.1 * torch.randn(num_buckets, heads, generator=g)).to(device))
        self.register_buffer("ln", torch.ones(hidden, dtype=torch.bfloat16, device=device))
        # an encoder without a score scale carries 1 / sqrt(d) in its query weights: here a power of two near it, which the scales
        # of a 4-bit weight take exactly (1/8 for a head dim from 64 to 255)
        for b in self.blocks:
            with torch.no_grad():
                b.q.base.scales.copy_(_shift_scales(b.q.base.scales, b.d))
                b.q.lora_up.mul_(2.0 ** -_half_log2(b.d))

    def forward(self, x, key_mask=None):
        # what a padded position holds (it may be anything) reaches neither the other positions nor, times zero, a gradient
        pad = None if key_mask is None else ~key_mask.unsqueeze(-1)
        if pad is not None:
            x = x.masked_fill(pad, 0.0)
        for b in self.blocks:
            x = b(x, self.table, key_mask)
        x = F.layer_norm(x, (x.shape[-1],), weight=self.ln, eps=1e-6)
        return x if pad is None else x.masked_fill(pad, 0.0)

    def trainable_parameters(self):
        return [p for n, p in self.named_parameters() if "lora_" in n] + [self.table]


def _half_log2(d: int) -> int:
    return (d.bit_length() - 1) // 2


def _shift_scales(scales: torch.Tensor, d: int) -> torch.Tensor:
    """MXFP4 scale codes of W / 2^_half_log2(d): the exponents lowered (not below 2^-127); the NaN scale (255) stays."""
    lower = (scales.to(torch.int16) - _half_log2(d)).clamp_(min=0).to(torch.uint8)
    return torch.where(scales == 255, scales, lower)


class ConditionedTrainer:
    """One training step of a DiTStack and the text encoder that conditions it: encode, denoise, MSE loss, backward
    through both, AdamW on every LoRA matrix and the position-bias table."""

    def __init__(self, encoder: TextEncoder, model, lr=1e-4, fused_optimizer=False):
        self.encoder, self.model = encoder, model
        self.params = model.lora_parameters() + [p for n, p in encoder.named_parameters() if "lora_" in n]
        self.opt = make_optimizer(self.params, lr=lr, fused=fused_optimizer)
        self.opt_table = make_optimizer([encoder.table], lr=lr, fused=fused_optimizer)

    def step(self, tokens, key_mask, x, cond, target):
        text = self.encoder(tokens, key_mask)
        loss = tv.mse_loss(self.model(x, text, cond), target)
        loss.backward()
        for o in (self.opt, self.opt_table):
            o.step()
            o.zero_grad(set_to_none=True)
        return loss.detach()


def main(steps=5):
    """A few joint steps on synthetic data: python -m torch_vulkan_b200.text_encoder"""
    from .dit import DiTStack, synthetic_batch

    enc = TextEncoder(blocks=2)
    model = DiTStack(blocks=1, base="mx4")
    x, tokens, cond, target = synthetic_batch()
    mask = torch.arange(tokens.shape[1], device=tokens.device)[None, :] < 300
    trainer = ConditionedTrainer(enc, model, lr=1e-3)
    for i in range(steps):
        print(f"step {i}: loss {trainer.step(tokens, mask, x, cond, target).item():.5f}")


if __name__ == "__main__":
    main()
