"""Relative accuracy of the step sizes, of softplus' and of the gate over their whole range, read off calls of one token and one state
in which nothing else rounds.

Tolerances, with u = 2^-24 and first order throughout. e^v: the argument is split exactly, the polynomial and its evaluation are off by 1.9 u
(its last addition u, the ones before 0.4 u, the fraction 0.4 u, the fit 2^-28.9), the scale is exact. softplus = max(v, 0) + 2 artanh(s), s =
w / (2 + w): 1.9 u of w, u of 2 + w, 2 u of the reciprocal and u of the product in s; the odd series u, its argument 0.5 u, its end 0.5 u, the
last operation u: 8.9 u of softplus. sigmoid: 1.9 u, u of 1 + e, 2 u: 4.9 u, and one product in silu and one with the sum: 6.9 u."""
import pytest

torch = pytest.importorskip("torch")

import ssm_reference as ref  # noqa: E402
from test_gpu_selective_scan import F16, F32, ops  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def values(dtype, lo, hi, n=4096):
    gen = torch.Generator(device="cuda").manual_seed(n)
    v = torch.rand(n - 8, device="cuda", generator=gen) * (hi - lo) + lo
    v = torch.cat([v, torch.tensor([lo, hi, 0.0, -0.5, 0.5, -1e-3, -20.0, 20.0], device="cuda").clamp(lo, hi)])
    return v.to(dtype).view(1, 1, n)


def ones(d, dtype):
    one = torch.ones(1, 1, d, device="cuda", dtype=dtype)
    bc = torch.ones(1, 1, 1, 1, device="cuda", dtype=dtype)
    return dict(x=one, A=torch.zeros(d, 1, device="cuda"), B=bc, C=bc)


def check(got, want, steps, what):
    err = (got.double() - want).abs() / (want.abs() + 1e-30)
    bound = steps * ref.U + (ref.HALF_STEP[got.dtype] if got.dtype == F16 else 0)
    if got.dtype == F16:
        err = ((got.double() - want).abs() - ref.HALF_TINY[F16]).clamp_min(0) / (want.abs() + 1e-30)
    assert float(err.max()) <= bound, f"{what}: off by {float(err.max()) / ref.U:.1f} u relative, allowed {bound / ref.U:.1f}"


@pytest.mark.parametrize("dtype", [F16, F32])
def test_step_sizes(ops, dtype):
    """final_state = delta x B from a state of zero: softplus(dt) itself."""
    dt = values(dtype, -80.0, 80.0)
    p = ones(dt.shape[-1], dtype)
    want = torch.nn.functional.softplus(dt.double(), threshold=1000.0)[0, 0, :, None]
    _, fin = ops.tensor_selective_scan(dt=dt, **p)
    check(fin[0], want, 8.9, "sequence")
    state = torch.zeros(1, dt.shape[-1], 1, device="cuda")
    ops.tensor_selective_scan_update(state, dt=dt[:, 0], **{k: (v if k == "A" else v[:, 0]) for k, v in p.items()})
    check(state[0], want, 8.9, "single token")


@pytest.mark.parametrize("dtype", [F16, F32])
def test_step_gradient(ops, dtype):
    """y = delta, so ddt = softplus'(dt) and, in fp32 whatever the type, ddt_bias is the same."""
    dt = values(dtype, -80.0, 80.0)
    p = ones(dt.shape[-1], dtype)
    bias = torch.zeros(dt.shape[-1], device="cuda")
    _, _, ck = ops.tensor_selective_scan(dt=dt, dt_bias=bias, **p, want_checkpoints=True)
    g = ops.tensor_selective_scan_backward(torch.ones_like(dt), dt=dt, dt_bias=bias, checkpoints=ck, **p)
    want = torch.sigmoid(dt.double())
    check(g.ddt, want, 4.9, "ddt")
    check(g.ddt_bias, want[0, 0], 4.9, "ddt_bias")


@pytest.mark.parametrize("dtype", [F16, F32])
def test_gate(ops, dtype):
    """y = 1 silu(z), in the sequence and in the single-token call."""
    z = values(dtype, -80.0, 80.0)
    p = ones(z.shape[-1], dtype)
    want = z.double() * torch.sigmoid(z.double())
    y, _ = ops.tensor_selective_scan(dt=p["x"], z=z, **p, dt_softplus=False)
    check(y, want, 6.9, "sequence")
    one = {k: (v if k == "A" else v[:, 0]) for k, v in p.items()}
    state = torch.zeros(1, z.shape[-1], 1, device="cuda")
    check(ops.tensor_selective_scan_update(state, dt=one["x"], z=z[:, 0], **one, dt_softplus=False), want[:, 0], 6.9, "single token")
