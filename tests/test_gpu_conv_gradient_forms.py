"""The gradient of the short convolution in each form of its channel accesses (four, two and single ones), over several runs and blocks
of tokens and blocks of channels, for every width, with and without an initial state. Tolerances: tests/ssm_reference.py."""
import pytest

torch = pytest.importorskip("torch")

import ssm_reference as ref  # noqa: E402
from test_gpu_selective_scan import F16, F32, ops, rn  # noqa: E402,F401

pytestmark = pytest.mark.gpu


# off, in elements, and channels: fours; pairs (even channels, rows on two elements); pairs of single loads (odd channels, or odd rows)
@pytest.mark.parametrize("b,l,d,off", [(2, 300, 132, 0), (2, 300, 130, 0), (1, 1030, 38, 0), (1, 1030, 38, 2), (2, 67, 260, 2), (3, 1, 6, 0), (1, 2, 70, 2),
                                       (2, 300, 130, 1), (1, 517, 67, 0), (4, 3, 2, 0)])
@pytest.mark.parametrize("width", [1, 2, 3, 4])
@pytest.mark.parametrize("with_init", [True, False])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_forms(ops, b, l, d, off, width, with_init, dtype):
    gen = torch.Generator(device="cuda").manual_seed(b * 1000 + l + d + off)
    x = rn(gen, b, l, d + 16, dtype=dtype)[..., off:off + d]
    w, bias, dy = rn(gen, d, width, dtype=dtype, std=0.5), rn(gen, d, dtype=dtype, std=0.2), rn(gen, b, l, d + 8, dtype=dtype)[..., off:off + d]
    init = rn(gen, b, d, width - 1, dtype=dtype) if with_init else None
    got = ops.tensor_causal_conv1d_tokens_backward(dy, x, w, bias, init, want_dinitial=True)
    want, bounds = ref.conv_tokens_backward(dy, x, w, bias, init)
    for name, a, e, bd in zip(("dx", "dw", "db", "dinit"), got, want, bounds):
        ref.assert_within(a, e, bd, name)
    again = ops.tensor_causal_conv1d_tokens_backward(dy, x, w, bias, init)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("b,l,d", [(2, 300, 132), (3, 2, 6), (1, 517, 67)])
@pytest.mark.parametrize("width", [1, 2, 4])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_each_gradient_alone_and_in_wider_rows(ops, b, l, d, width, dtype):
    """Through the C ABI: each output with the others null equals that of the full call; dx in wider rows leaves what lies between them."""
    import ctypes
    from anygpu_b200 import capi
    gen = torch.Generator(device="cuda").manual_seed(b + l + d)
    x, dy = rn(gen, b, l, d, dtype=dtype), rn(gen, b, l, d, dtype=dtype)
    w, bias, init = rn(gen, d, width, dtype=dtype, std=0.5), rn(gen, d, dtype=dtype), rn(gen, b, d, width - 1, dtype=dtype)
    full = ops.tensor_causal_conv1d_tokens_backward(dy, x, w, bias, init, want_dinitial=True)
    ws = torch.empty(capi.load().b200_causal_conv1d_tokens_backward_workspace_bytes(b, l, d, width), dtype=torch.uint8, device="cuda")
    ptr = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr() or 256)

    def call(dx, dxs, dw, db, dinit):
        capi.call("b200_causal_conv1d_tokens_backward", capi.F16 if dtype == F16 else capi.F32, ptr(dy), d, ptr(x), d, ptr(w), ptr(bias), ptr(init), dx, dxs,
                  ptr(dw), ptr(db), ptr(dinit), b, l, d, width, ptr(ws), ws.numel(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))

    for i in range(4):
        out = [torch.full_like(t, 7.0) if i == j else None for j, t in enumerate(full)]
        call(ptr(out[0]), d, out[1], out[2], out[3])
        assert torch.equal(out[i], full[i]), i
    wide = torch.full((b, l, d + 9), 3.0, device="cuda", dtype=dtype)
    call(ctypes.c_void_p(wide.data_ptr() + 4 * wide.element_size()), d + 9, None, None, None)
    assert torch.equal(wide[..., 4:4 + d], full[0]) and (wide[..., :4] == 3).all() and (wide[..., 4 + d:] == 3).all()
