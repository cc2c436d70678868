"""Parameters of the selective scan that start off 16 bytes (one layer's row of a tensor for all layers) give the bits of aligned ones."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_selective_scan import F16, F32, inputs, ops, rn  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2, 40, 20, 1, 16), (1, 37, 6, 2, 5), (1, 700, 8, 1, 4), (3, 20, 12, 1, 100)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [1, 2])
def test_parameters_off_16_bytes(ops, shape, dtype, n):
    b, l, d, g, s = shape
    p, gen = inputs(sum(shape), b, l, d, g, s, dtype)
    dy = rn(gen, b, l, d, dtype=dtype)

    def off(t):
        flat = torch.full((t.numel() + n,), float("nan"), device="cuda")
        flat[n:] = t.reshape(-1)
        return flat[n:].view(t.shape)

    def everything(q):
        y, fin, ck = ops.tensor_selective_scan(**q, want_checkpoints=True)
        state = q["initial_states"].clone()
        one = {k: (v[:, 3] if k in ("x", "dt", "B", "C", "z") else v) for k, v in q.items() if k != "initial_states"}
        step = ops.tensor_selective_scan_update(state, **one)
        return (y, fin, step, state) + tuple(ops.tensor_selective_scan_backward(dy, checkpoints=ck, **q))

    want = everything(p)
    got = everything({**p, **{k: off(p[k]) for k in ("A", "D", "dt_bias")}})
    assert all(torch.equal(a, c) for a, c in zip(got, want))
