"""The 4-bit linears and the bias attention under autograd's modes."""

import pytest
import torch

from tests.test_bias_attention import _case

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
