"""Two host threads that call one kernel with different sizes of shared memory."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _both(calls, steps):
    """calls[i](step) for every step in a thread of its own, each step begun by all together; the first error is raised."""
    gate, errors = threading.Barrier(len(calls)), []

    def work(call):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(steps):
                    gate.wait(60)
                    call(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
            gate.abort()

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for e in errors:
        if not isinstance(e, threading.BrokenBarrierError):
            raise e
    assert not errors


@pytest.mark.parametrize("dt,D,Sq", [(torch.float32, 40, 33), (torch.float32, 128, 33), (torch.bfloat16, 20, 33), (torch.bfloat16, 64, 33),
                                     (torch.float16, 128, 33), (torch.float32, 72, 2), (torch.float16, 96, 2), (torch.bfloat16, 32, 2)])
def test_bias_attention_of_growing_max_distances(dt, D, Sq):
    """The bias vector's length sets a kernel's shared memory: both threads ask for more at every step, one always for less
    than the other."""
    import torch_vulkan_b200 as tv

    t = [torch.randn(1, 2, n, D, device="cuda").to(dt) for n in (Sq, 50, 50)]
    table = torch.randn(4, 2, device="cuda")
    torch.cuda.synchronize()
    call = lambda extra: lambda i: tv.bucket_bias_attention(*t, table, max_distance=20 + 8 * i + extra)  # noqa: E731
    _both([call(0), call(4), call(6)], 120)
    assert tv.validation_errors() == 0


def test_few_rows_of_growing_widths():
    import torch_vulkan_b200 as tv

    ks = [[32 * (3 * i + e + 1) for i in range(60)] for e in range(3)]
    ws = [[tv.mx4_quantize(torch.randn(16, k, device="cuda")) for k in row] for row in ks]
    xs = [[torch.randn(2, k, device="cuda").bfloat16() for k in row] for row in ks]
    torch.cuda.synchronize()
    _both([lambda i, e=e: tv.mx4_linear(xs[e][i], ws[e][i]) for e in range(3)], 60)
    assert tv.validation_errors() == 0
