"""The 4-bit linears and the bias attention under autograd's modes: without gradients, and differentiated twice."""

import pytest
import torch

from tests.test_bias_attention import _case
from tests.test_mx4 import _linear_case

pytestmark = pytest.mark.gpu


def _peak(f):
    f()
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = f()
    return out, torch.cuda.max_memory_allocated() - base


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 700, 64), (300, 300, 64), (300, 400, 128), (1024, 1024, 128)])
def test_a_trainable_table_without_gradients_runs_the_inference_kernel(dt, Sq, Sk, D):
    """no_grad and inference_mode give a Parameter's call the bits and the memory of its detached copy's: no unrounded output."""
    import torch_vulkan_b200 as tv

    q, k, v, _, table, m = _case(2, 4, 4, Sq, Sk, D, dt, D, "tail")
    q, k, v, m = (t.cuda() for t in (q, k, v, m))
    plain, param = table.cuda(), torch.nn.Parameter(table.cuda())
    f = lambda t, x=q: tv.bucket_bias_attention(x, k, v, t, key_mask=m)  # noqa: E731
    want, peak = _peak(lambda: f(plain))
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            got, used = _peak(lambda: f(param))
            assert not got.requires_grad and torch.equal(got, want) and used == peak
            got, used = _peak(lambda: f(param, q.detach().requires_grad_(True)))
            assert torch.equal(got, want) and used == peak
    assert f(param).requires_grad


def _calls():
    import torch_vulkan_b200 as tv

    x, w, bias, gy, a, b = (t.cuda() for t in _linear_case(40, 64, 72, 3, 8))
    wd = tv.mx4_quantize(w)
    q, k, v, go, table, m = (t.cuda() if t is not None else None for t in _case(2, 4, 2, 40, 60, 64, torch.bfloat16, 1, "tail"))
    f32 = [t.float() for t in (q, k, v)]
    return {"linear": (lambda x, bias: tv.mx4_linear(x, wd, bias), (x, bias), gy),
            "lora": (lambda x, bias, a, b: tv.mx4_lora_linear(x, wd, bias, a, b), (x, bias, a, b), gy),
            "attention": (lambda *t: tv.bucket_bias_attention(*t, key_mask=m), (q, k, v, table), go),
            "attention_f32": (lambda *t: tv.bucket_bias_attention(*t), (*f32, table), go.float())}


@pytest.mark.parametrize("name", ["linear", "lora", "attention", "attention_f32"])
def test_a_second_differentiation_is_refused(name):
    """create_graph gives the first derivatives as ever; differentiating one of them along what it depends on, alone or in a
    larger sum, is an error. A bias gradient is a sum of the incoming one and can be; dx of the plain 4-bit linear depends on
    that alone."""
    f, args, go = _calls()[name]
    leaf = [t.detach().requires_grad_(True) for t in args]
    first = torch.autograd.grad(f(*leaf), leaf, go)
    weight = go.detach().requires_grad_(True)
    exact = {"linear": (1,), "lora": (1,)}.get(name, ())
    for i in range(len(leaf)):
        for w in (go, weight):
            got = torch.autograd.grad(f(*leaf), leaf, w, create_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, first))
            total = got[i].float().pow(2).sum() + sum(t.float().sum() for t in leaf)
            wanted = leaf + [w] if w is weight else leaf
            if i in exact or (name == "linear" and w is go):
                *rest, dw = torch.autograd.grad(total, leaf + [weight], allow_unused=True)
                assert all(bool((t == 1).all()) for t in rest)
                if w is weight:
                    assert torch.equal(dw, (2 * got[i].float()).bfloat16().expand_as(go))
            else:
                with pytest.raises(RuntimeError, match="twice"):
                    torch.autograd.grad(total, wanted, allow_unused=True)


def test_a_second_differentiation_of_the_stacked_projections_is_refused():
    from torch_vulkan_b200.dit import DiTBlock

    blk = DiTBlock(hidden=256, heads=2, text_dim=128, mlp=512, base="mx4")
    x = torch.randn(1, 64, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = blk._stacked("qkv", x, (blk.q, blk.k, blk.v), whole=True)
    (gx,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(gx.float().pow(2).sum() + x.float().sum(), x)
