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
