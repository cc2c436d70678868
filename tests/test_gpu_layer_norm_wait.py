"""The bounded waits of layer norm's gradient: a stage that nothing fills is given up, reported, and the next call is right."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import ssm_reference as ref  # noqa: E402
from anygpu_b200 import capi  # noqa: E402
from test_gpu_selective_scan import F16, ops, rn  # noqa: E402,F401


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", [(1, 1024), (5, 2048), (3001, 4096), (901, 8192)])  # one CTA and all of them, two rows at a time and one
def test_a_stage_that_never_fills(ops, rows, dim):
    lib = capi.load()
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x, dy = rn(gen, rows, dim, dtype=F16), rn(gen, rows, dim, dtype=F16)
    _, mean, rstd = ops.tensor_layer_norm(x, None, None, 1e-5, want_stats=True)
    dx = torch.empty_like(x)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.b200_last_device_error(stream, None) == 0
    rc = lib.b200_debug_layer_norm_backward_starved(dy.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), rows, dim, 20000,
                                                    stream)
    assert rc == 0  # the launch itself succeeds
    detail = ctypes.c_uint32(0)
    assert lib.b200_last_device_error(stream, ctypes.byref(detail)) == -4 and detail.value >> 16 == 6, hex(detail.value)
    assert lib.b200_last_device_error(stream, None) == 0  # reading the error word clears it
    torch.cuda.synchronize()
    got = ops.tensor_layer_norm_backward(dy, x, None, mean, rstd)
    want = ref.layer_norm_backward(dy, x, None, mean, rstd)
    for a, w, bound, name in zip(got, want[:3], want[3:], ("dx", "dw", "db")):
        ref.assert_within(a, w, bound, name)
    assert lib.b200_last_device_error(stream, None) == 0


def test_refusals():
    f, one, odd = capi.load().b200_debug_layer_norm_backward_starved, 256, 264
    assert f(None, one, one, one, one, 1, 1024, 1000, None) == -7 and f(one, one, one, one, None, 1, 1024, 1000, None) == -7
    assert f(one, one, one, one, one, 1, 1000, 1000, None) == -1 and f(one, one, one, one, one, 1, 8200, 1000, None) == -1
    assert f(one, one, one, one, one, 0, 1024, 1000, None) == -1 and f(one, one, one, one, one, 1, 1024, 0, None) == -1
    assert f(one, one, one, one, one, 1, 1024, 1 << 22, None) == -1 and f(odd, one, one, one, one, 1, 1024, 1000, None) == -2
