"""The selective scan split along the tokens, for every number of lanes that share a channel (1 to 32: up to 4, 8, 16, 32, 64 and 128
states), at lengths that end inside a tile, against the 64-bit forms of tests/ssm_reference.py (tolerances there)."""
import pytest

torch = pytest.importorskip("torch")

import ssm_reference as ref  # noqa: E402
from test_gpu_selective_scan import F16, F32, GRADS, inputs, ops, reference_args, rn  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(1, 701, 8, 1, 4), (2, 1111, 40, 1, 3), (1, 1500, 24, 1, 7), (1, 701, 12, 2, 16), (1, 701, 40, 2, 24), (1, 1235, 12, 1, 32),
                                   (1, 1111, 14, 2, 64), (1, 701, 10, 1, 100), (1, 999, 6, 1, 128)])
@pytest.mark.parametrize("dtype,off", [(F16, 0), (F16, 2), (F16, 1), (F32, 0)])
def test_segments(ops, shape, dtype, off):
    """off: f16 rows on 16 bytes (or fewer), on 4 and on 2."""
    from anygpu_b200 import capi
    b, l, d, g, n = shape
    assert capi.load().b200_selective_scan_workspace_bytes(b, l, d, g, n) > 0, "one segment only"
    p, gen = inputs(l + n, b, l, d, g, n, dtype, off=off)
    dy, dfin = rn(gen, b, l, d, dtype=dtype), rn(gen, b, d, n)
    y, fin, ck = ops.tensor_selective_scan(**p, want_checkpoints=True)
    grads = ops.tensor_selective_scan_backward(dy, checkpoints=ck, dfinal_states=dfin, **p)
    leaves = {k: v.requires_grad_() for k, v in reference_args(p).items()}
    wy, wfin = ref.scan(**leaves)
    ((wy * dy.double()).sum() + (wfin * dfin.double()).sum()).backward()
    bounds = ref.scan_bounds(**reference_args(p), dy=dy.double(), dfin=dfin.double())
    ref.assert_within(y, wy.detach(), bounds[0], "y")
    ref.assert_within(fin, wfin.detach(), bounds[1], "final_states")
    for i, (name, leaf) in enumerate(GRADS):
        ref.assert_within(getattr(grads, name), leaves[leaf].grad, bounds[2 + i], name)
    y2, fin2 = ops.tensor_selective_scan(**p)
    assert torch.equal(y, y2) and torch.equal(fin, fin2)


@pytest.mark.parametrize("n", [4, 8, 16, 32, 64, 128])
def test_checkpoints_are_the_states(ops, n):
    """checkpoints[b, t / 16] is the state before token t, whichever segment it lies in: that which a call on the tokens before it ends in."""
    b, l, d, g = 2, 701, 8, 1
    p, _ = inputs(n, b, l, d, g, n, F32)
    _, _, ck = ops.tensor_selective_scan(**p, want_checkpoints=True)
    ck = ck.view(b, -1, d, n)
    assert ck.shape[1] == (l + 15) // 16
    assert torch.equal(ck[:, 0], p["initial_states"])
    for k in (1, 2, 3, 21, 22, ck.shape[1] - 1):
        part = {name: (v[:, :16 * k] if name in ("x", "dt", "B", "C", "z") else v) for name, v in p.items()}
        part = {name: v.contiguous() for name, v in part.items()}
        _, want = ref.scan(**reference_args(part))
        ref.assert_within(ck[:, k], want, ref.scan_bounds(**reference_args(part))[1], f"checkpoint {k}")


@pytest.mark.parametrize("shape", [(2, 33, 6, 6, 16), (1, 40, 8, 8, 4), (1, 700, 3, 3, 16), (2, 20, 4, 4, 100), (1, 35, 66, 33, 16)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_groups_of_one_and_two_channels(ops, shape, dtype):
    b, l, d, g, n = shape
    p, gen = inputs(l + n, b, l, d, g, n, dtype)
    dy, dfin = rn(gen, b, l, d, dtype=dtype), rn(gen, b, d, n)
    y, fin, ck = ops.tensor_selective_scan(**p, want_checkpoints=True)
    grads = ops.tensor_selective_scan_backward(dy, checkpoints=ck, dfinal_states=dfin, **p)
    leaves = {k: v.requires_grad_() for k, v in reference_args(p).items()}
    wy, wfin = ref.scan(**leaves)
    ((wy * dy.double()).sum() + (wfin * dfin.double()).sum()).backward()
    bounds = ref.scan_bounds(**reference_args(p), dy=dy.double(), dfin=dfin.double())
    ref.assert_within(y, wy.detach(), bounds[0], "y")
    ref.assert_within(fin, wfin.detach(), bounds[1], "final_states")
    for i, (name, leaf) in enumerate(GRADS):
        ref.assert_within(getattr(grads, name), leaves[leaf].grad, bounds[2 + i], name)
    state = p["initial_states"].clone()
    one = {k: (v[:, 0] if k in ("x", "dt", "B", "C", "z") else v) for k, v in p.items() if k != "initial_states"}
    first = {k: (v[:, :1].contiguous() if k in ("x", "dt", "B", "C", "z") else v) for k, v in p.items()}
    wy, wfin = ref.scan(**reference_args(first))
    bounds = ref.scan_bounds(**reference_args(first))
    ref.assert_within(ops.tensor_selective_scan_update(state, **one), wy[:, 0], bounds[0][:, 0], "single token")
    ref.assert_within(state, wfin, bounds[1], "state")
