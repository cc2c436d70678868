"""Which parameters the selective scan's Python front-end takes (no GPU: what it takes goes on to the check of the device)."""
import pytest

torch = pytest.importorskip("torch")

from anygpu_b200 import ops  # noqa: E402


def off(t, n):
    """t's values n elements into a buffer of its own: one layer's row of parameters that are kept in one tensor for all layers."""
    flat = torch.zeros(t.numel() + n, dtype=t.dtype)
    assert flat.data_ptr() % 16 == 0
    return flat[n:].view(t.shape)


def calls(**over):
    x, BC = torch.zeros(2, 5, 6), torch.zeros(2, 5, 1, 3)
    p = {**dict(x=x, dt=x, A=torch.zeros(6, 3), B=BC, C=BC, D=torch.zeros(6), dt_bias=torch.zeros(6)), **over}
    ops_args = dict(p)
    step = {k: (v[:, 0] if k in ("x", "dt", "B", "C") else v) for k, v in p.items()}
    ck = torch.zeros(2 * 1 * 6 * 3)
    init = p.get("initial_states")
    step.pop("initial_states", None)
    yield lambda: ops.tensor_selective_scan(**ops_args)
    yield lambda: ops.tensor_selective_scan_backward(x, checkpoints=ck, **ops_args)
    yield lambda: ops.tensor_selective_scan_update(torch.zeros(2, 6, 3) if init is None else init, **step)


@pytest.mark.parametrize("n", [1, 2, 3])
@pytest.mark.parametrize("name,shape", [("A", (6, 3)), ("D", (6,)), ("dt_bias", (6,))])
def test_parameters_may_start_on_any_element(name, shape, n):
    for call in calls(**{name: off(torch.zeros(shape), n)}):
        with pytest.raises(AssertionError, match="no CPU path"):
            call()


def test_states_start_on_16_bytes():
    for call in calls(initial_states=off(torch.zeros(2, 6, 3), 1)):
        with pytest.raises(AssertionError, match="16-byte boundary"):
            call()
