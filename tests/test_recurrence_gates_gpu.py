"""GPU: both gates of the recurrence to a few steps of fp32 however far apart they are.

The smaller gate is 1 / (1 + e^|g|).  Its roundings (U = 2^-24): 4 U of ex2.approx, 1 U of the correction of its argument,
1 U of the sum, 2 U of rcp.approx, and 1 U of the product it goes into: 9 U, relative, down to the smallest normal number,
below which it comes out as 0."""
import pytest
import torch

from policy_reference import U, within
from test_policy_ops_gpu import BF16, F16, F32

pytestmark = pytest.mark.gpu
TINY = 2.0 ** -126


def gate_values(dtype, n=4096):
    """0 to 90 and beyond, both spread evenly and over the logarithm; values of `dtype`."""
    v = torch.cat([torch.linspace(0, 90, n // 2, device="cuda"), torch.logspace(-6, 2.2, n // 2, device="cuda")])
    return v.to(dtype)


def smaller(g):
    """1 / (1 + e^|g|) in 64 bits."""
    return torch.sigmoid(-g.double().abs())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_the_smaller_gate_of_a_step(dtype):
    import pufferlib_b200 as pb
    g = gate_values(dtype)[None]
    zero, one = torch.zeros_like(g), torch.ones_like(g)
    want = smaller(g)
    for gates, x, state in ((g, one, zero.float()), (-g, zero, one.float())):
        _, new = pb.gated_recurrence_step(gates, x, state)
        within(new, want, 9 * U * want + TINY, "gate")


@pytest.mark.parametrize("steps", [1, 2, 8, 9, 40, 700, 3000])
@pytest.mark.parametrize("channels", [4096, 515, 7])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_smaller_gate_in_a_sequence(steps, channels, dtype):
    """All inputs but the last are 0 and so is the state: the last output is the gate that takes the input, as is the
    gradient of that input.  A state of 1 behind gates that hold it, and one that does not: the gate that keeps it."""
    import pufferlib_b200 as pb
    values = gate_values(dtype)
    pick = torch.arange(channels, device="cuda") * (4096 // channels)
    gates = torch.full((2, steps, channels), 200.0, device="cuda", dtype=dtype)
    gates[0, -1] = values[pick]
    gates[1, -1] = -values[pick]
    x = torch.zeros_like(gates)
    x[0, -1] = 1.0
    state = torch.zeros(2, channels, device="cuda")
    state[1] = 1.0
    x.requires_grad_(True), state.requires_grad_(True)
    _, final = pb.gated_recurrence(gates, x, state=state)
    want = smaller(values[pick])
    for row in range(2):
        within(final[row], want, 9 * U * want + TINY, f"final state {row}")
    dx, ds = torch.autograd.grad(final, [x, state], torch.ones_like(final))
    within(ds[1], want, 9 * U * want + TINY, "gradient of the state")
    if dtype == F32:
        within(dx[0, -1], want, 9 * U * want + TINY, "gradient of the input")


def test_infinite_and_nan_gates():
    import math

    import pufferlib_b200 as pb
    g = torch.tensor([math.inf, -math.inf, math.nan, 1e30, -1e30, 88.0, -88.0, 0.0, -0.0], device="cuda")
    for steps in (1, 5, 40):
        gates = g.expand(1, steps, 9).contiguous()
        x, state = torch.full_like(gates, 3.0), torch.full((1, 9), 5.0, device="cuda")
        out, final = pb.gated_recurrence(gates, x, state=state)
        assert final[0, [0, 3, 5]].eq(5.0).all() and final[0, [1, 4, 6]].eq(3.0).all() and final[0, 2].isnan()
        assert final[0, 7] == final[0, 8] == 3.0 + 2.0 * 0.5 ** steps or steps > 20
    _, new = pb.gated_recurrence_step(g[None], x[:, 0], state)
    assert new[0, [0, 3, 5]].eq(5.0).all() and new[0, [1, 4, 6]].eq(3.0).all() and new[0, 2].isnan() and new[0, 7] == 4.0
