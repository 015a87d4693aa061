"""Operands of the 4-bit linears on another GPU than x."""

import pytest
import torch

from tests.test_mx4 import BF, _linear_case

pytestmark = pytest.mark.gpu


class _Elsewhere(torch.Tensor):
    """A tensor that says it is on the second GPU and has no memory there."""

    @staticmethod
    def __new__(cls, *size):
        return torch.Tensor._make_wrapper_subclass(cls, size, dtype=BF, device="cuda:1")

    __torch_dispatch__ = None


def _case():
    import torch_vulkan_b200 as tv

    x, w, bias, gy, a, b = (t.cuda() for t in _linear_case(5, 64, 72, 3, 8))
    return tv, x, tv.mx4_quantize(w), bias, gy, a, b


def test_a_bias_or_lora_matrix_elsewhere_is_refused():
    tv, x, w, bias, gy, a, b = _case()
    skip = torch._C._ExcludeDispatchKeyGuard(torch._C.DispatchKeySet(torch._C.DispatchKey.Python)
                                             | torch._C.DispatchKeySet(torch._C.DispatchKey.PythonTLSSnapshot))
    with torch.no_grad(), skip:
        for f in (lambda: tv.mx4_linear(x, w, _Elsewhere(72)), lambda: tv.mx4_lora_linear(x, w, _Elsewhere(72), a, b),
                  lambda: tv.mx4_lora_linear(x, w, bias, _Elsewhere(8, 64), b),
                  lambda: tv.mx4_lora_linear(x, w, bias, a, _Elsewhere(72, 8)),
                  lambda: torch.ops.b2.mx4_lora_dx(gy, w.codes, w.scales, 64, _Elsewhere(5, 8), a),
                  lambda: torch.ops.b2.mx4_lora_dx(gy, w.codes, w.scales, 64, torch.mm(gy, b), _Elsewhere(8, 64))):
            with pytest.raises(RuntimeError, match="on x's device"):
                f()
    tv.mx4_lora_linear(x, w, bias, a, b)
    assert tv.validation_errors() == 0


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
def test_operands_on_a_second_gpu_are_refused():
    tv, x, w, bias, gy, a, b = _case()
    for f in (lambda: tv.mx4_linear(x, w, bias.to(1)), lambda: tv.mx4_lora_linear(x, w, bias, a.to(1), b),
              lambda: tv.mx4_lora_linear(x, w, bias, a, b.to(1)), lambda: tv.mx4_linear(x.to(1), w)):
        with pytest.raises(RuntimeError, match="device"):
            f()
