"""The selective scan and its gradients where the decays leave the range of fp32: A at the type's lowest value, infinite or past the
range of exp, against the 64-bit forms of tests/ssm_reference.py (tolerances there)."""
import pytest

torch = pytest.importorskip("torch")

import ssm_reference as ref  # noqa: E402
from test_gpu_selective_scan import F16, F32, GRADS, inputs, ops, reference_args, rn  # noqa: E402,F401

pytestmark = pytest.mark.gpu
LOWEST = torch.finfo(F32).min


def check_all(got, p, dy, dfin, **form):
    """y, the last state and every gradient against the 64-bit form."""
    y, fin, grads = got
    leaves = {k: v.requires_grad_() for k, v in reference_args(p).items()}
    wy, wfin = ref.scan(**leaves, **form)
    ((wy * dy.double()).sum() + (wfin * dfin.double()).sum()).backward()
    bounds = ref.scan_bounds(**reference_args(p), **form, dy=dy.double(), dfin=dfin.double())
    ref.assert_within(y, wy.detach(), bounds[0], "y")
    ref.assert_within(fin, wfin.detach(), bounds[1], "final_states")
    for i, (name, leaf) in enumerate(GRADS):
        ref.assert_within(getattr(grads, name), leaves[leaf].grad, bounds[2 + i], name)


@pytest.mark.parametrize("shape", [(2, 40, 20, 1, 16), (1, 37, 12, 2, 5), (2, 33, 8, 1, 100), (1, 700, 8, 1, 16)])  # the last: token segments
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("low", [-1e30, -1e36, LOWEST, -float("inf")])
def test_gradients_of_decays_that_forget(ops, shape, dtype, low):
    """exp(delta A) is zero there, and so is A exp(delta A) h: nothing of it reaches ddt, ddt_bias or dA, whatever A is."""
    b, l, d, g, n = shape
    p, gen = inputs(l + d + n, b, l, d, g, n, dtype)
    p["A"][3], p["A"][5, 2] = low, low
    dy, dfin = rn(gen, b, l, d, dtype=dtype), rn(gen, b, d, n)
    y, fin, ck = ops.tensor_selective_scan(**p, want_checkpoints=True)
    grads = ops.tensor_selective_scan_backward(dy, checkpoints=ck, dfinal_states=dfin, **p)
    # an infinite A counts as the lowest finite one, whose exponential is zero in 64 bits too
    check_all((y, fin, grads), {**p, "A": p["A"].clamp_min(LOWEST)}, dy, dfin)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("log", [80.0, 88.5, 95.0])
def test_gradients_of_a_log_past_the_range_of_exp(ops, dtype, log):
    """The same for A = -exp(A_log) that overflows fp32 (above 88.7): dA is zero, not infinity times zero."""
    b, l, d, g, n = 2, 45, 20, 1, 16
    p, gen = inputs(7, b, l, d, g, n, dtype, log=True)
    p["A"][3], p["A"][5, 2] = log, log
    dy, dfin = rn(gen, b, l, d, dtype=dtype), rn(gen, b, d, n)
    y, fin, ck = ops.tensor_selective_scan(**p, a_is_log=True, want_checkpoints=True)
    grads = ops.tensor_selective_scan_backward(dy, checkpoints=ck, dfinal_states=dfin, **p, a_is_log=True)
    check_all((y, fin, grads), p, dy, dfin, log=True)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_single_tokens_forget(ops, dtype):
    """A state whose decay is zero starts anew with the token, in the single-token call as in the sequence."""
    b, l, d, g, n = 3, 9, 16, 1, 16
    p, _ = inputs(9, b, l, d, g, n, dtype)
    p["A"][3] = LOWEST
    p["initial_states"][:, 3] = 1e38  # 2^-126 of it would still be 0.9
    p["x"][:, 4, 3] = 0
    one = {k: (v[:, 4] if k in ("x", "dt", "B", "C", "z") else v) for k, v in p.items() if k != "initial_states"}
    state = p["initial_states"].clone()
    ops.tensor_selective_scan_update(state, **one)
    assert not state[:, 3].any()
    cut = {k: (v[:, 4:5] if k in ("x", "dt", "B", "C", "z") else v) for k, v in p.items()}
    assert not ops.tensor_selective_scan(**cut)[1][:, 3].any()


@pytest.mark.parametrize("shape", [(2, 50, 24, 1, 16), (1, 700, 8, 1, 16), (2, 37, 6, 1, 5)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("mask", ["inf", "max"])
def test_masked_tokens_of_channels_that_forget(ops, shape, dtype, mask):
    """A step of zero passes state and adjoint on whatever A is, and its own gradient is zero: A g h, which overflows where A is the
    type's lowest value, comes with softplus' = 0."""
    b, l, d, g, n = shape
    p, gen = inputs(17 + l, b, l, d, g, n, dtype)
    p["A"][3], p["A"][5, 2] = LOWEST, LOWEST
    masked = torch.rand(b, l, device="cuda", generator=gen) < 0.4
    masked[:, -1] = False
    p["dt"][masked] = -float("inf") if mask == "inf" else torch.finfo(dtype).min
    p["initial_states"] *= 100
    dy, dfin = rn(gen, b, l, d, dtype=dtype) * 8, rn(gen, b, d, n) * 100
    y, fin, ck = ops.tensor_selective_scan(**p, want_checkpoints=True)
    grads = ops.tensor_selective_scan_backward(dy, checkpoints=ck, dfinal_states=dfin, **p)
    for name, _ in GRADS:
        assert torch.isfinite(getattr(grads, name)).all(), name
    assert not grads.ddt[masked].any() and not grads.dB[masked].any()
    # where dy is zero too, a masked token is as good as not there
    dy[masked] = 0
    grads = ops.tensor_selective_scan_backward(dy, checkpoints=ck, dfinal_states=dfin, **p)
    for i in range(b):
        kept = ~masked[i]
        row = lambda k, v: v[i:i + 1, kept].contiguous() if k in ("x", "dt", "B", "C", "z") else (v[i:i + 1] if k == "initial_states" else v)
        one = {k: row(k, v) for k, v in p.items()}
        leaves = {k: v.requires_grad_() for k, v in reference_args(one).items()}
        wy, wfin = ref.scan(**leaves)
        dyi, dfi = dy[i:i + 1, kept].double(), dfin[i:i + 1].double()
        ((wy * dyi).sum() + (wfin * dfi).sum()).backward()
        bounds = ref.scan_bounds(**reference_args(one), dy=dyi, dfin=dfi)
        for j, (name, leaf) in enumerate(GRADS):
            if leaf in ("x", "dt", "B", "C", "z"):
                ref.assert_within(getattr(grads, name)[i:i + 1, kept], leaves[leaf].grad, bounds[2 + j], name)
            elif leaf == "init":
                ref.assert_within(grads.dinitial_states[i:i + 1], leaves[leaf].grad, bounds[2 + j], name)


@pytest.mark.parametrize("shape", [(2, 40, 20, 1, 16), (1, 33, 12, 2, 5), (1, 31, 9, 1, 3), (2, 17, 8, 1, 100), (1, 3, 16, 1, 16), (1, 700, 8, 1, 16)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("log", [False, True])
def test_a_decay_that_is_not_a_number_reaches_what_it_should(ops, shape, dtype, log):
    """NaN in one element of A, sequences that end inside a tile: results and gradients are NaN exactly where the 64-bit form's are, the last
    token's (which no decay separates from the final state) among them."""
    b, l, d, g, n = shape
    p, gen = inputs(l + d, b, l, d, g, n, dtype, log=log)
    p["A"][5, 2] = float("nan")
    dy, dfin = rn(gen, b, l, d, dtype=dtype), rn(gen, b, d, n)
    y, fin, ck = ops.tensor_selective_scan(**p, a_is_log=log, want_checkpoints=True)
    grads = ops.tensor_selective_scan_backward(dy, checkpoints=ck, dfinal_states=dfin, **p, a_is_log=log)
    leaves = {k: v.requires_grad_() for k, v in reference_args(p).items()}
    wy, wfin = ref.scan(**leaves, log=log)
    ((wy * dy.double()).sum() + (wfin * dfin.double()).sum()).backward()
    assert not torch.isnan(leaves["x"].grad[:, -1]).any() and not torch.isnan(leaves["B"].grad[:, -1]).any()
    for name, got, want in [("y", y, wy), ("final_states", fin, wfin)] + [(name, getattr(grads, name), leaves[leaf].grad) for name, leaf in GRADS]:
        assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: {int(torch.isnan(got).sum())} against {int(torch.isnan(want).sum())}"
        assert torch.isfinite(got[~torch.isnan(got)]).all(), name
