"""GPU: the gated recurrence where the state outlives its tile: gates that hold, over every way the steps are divided.

With gates around 0 a state has faded below rounding after a tile of sixteen steps, so a join that lost or misplaced the
product of the gates would not show.  Here the gates keep the state over hundreds of steps."""
import math

import pytest
import torch

import policy_reference as ref
from policy_reference import within
from test_policy_ops_gpu import BF16, F16, F32, check_recurrence, gen, randn

pytestmark = pytest.mark.gpu

# (shape, dtype): lane blocks of 32 x 4 bytes, and what takes them.  Clusters of n CTAs where n x lane blocks is between
# 190 and 296 and there are 256 n steps; ranges of steps where lanes are fewer; warps of a CTA where they are more.
DIVISIONS = [((3, 1200, 1024), F32),      # 96: clusters of two
             ((3, 1200, 2048), BF16),     # 96: clusters of two
             ((3, 1500, 1024), BF16),     # 48: clusters of four
             ((3, 1500, 1024), F16),      # 48: clusters of four
             ((1, 2500, 1600), F32),      # 50: clusters of four
             ((1, 1037, 2368), F32),      # 74: clusters of four, a last tile of 13 steps
             ((1, 2500, 1600), BF16),     # 25: ranges
             ((2, 1100, 96), F32),        # 6: ranges
             ((1, 1300, 33), BF16),       # odd width, no TMA: ranges
             ((2, 1300, 7), F32),         # few channels, rows share warps: ranges
             ((40, 300, 512), BF16),      # 320: warps of a CTA
             ((40, 300, 515), BF16)]      # odd width: warps of a CTA


def held(shape, dtype, shift, seed):
    g = gen(seed)
    gates = (randn(g, *shape) * 0.5 + shift).to(dtype)
    x = randn(g, *shape).to(dtype)
    return gates, x, 4.0 * randn(g, shape[0], shape[2])


@pytest.mark.parametrize("shape,dtype", DIVISIONS)
@pytest.mark.parametrize("shift", [6.0, 9.0])
def test_a_state_that_lasts(shape, dtype, shift):
    gates, x, state = held(shape, dtype, shift, seed=shape[2])
    out, final, grads = check_recurrence(gates, x, None, state)
    # what the test is about: the first state still counts at the end, and the last gradient at the beginning
    kept = torch.sigmoid(gates.double()).prod(1)
    assert (kept * state.double()).abs().mean() > 1e-3
    assert grads[2].abs().mean() > 1e-3


@pytest.mark.parametrize("shape,dtype", DIVISIONS)
def test_a_reset_in_the_middle_of_a_state_that_lasts(shape, dtype):
    """One reset a row, at another step in each, among steps that hold."""
    gates, x, state = held(shape, dtype, 8.0, seed=shape[1])
    resets = torch.zeros(shape[:2], device="cuda")
    for b in range(shape[0]):
        resets[b, (shape[1] // 3 + 77 * b) % shape[1]] = 1.0
    check_recurrence(gates, x, resets, state)


@pytest.mark.parametrize("shape,dtype", DIVISIONS)
def test_what_a_reset_cuts_off_among_steps_that_hold(shape, dtype):
    """NaN and infinities up to a reset: nothing of them behind it, and nothing before them changes."""
    import pufferlib_b200 as pb
    gates, x, state = held(shape, dtype, 8.0, seed=3)
    B, T, C = shape
    for at in (T // 4, T // 2 + 5, T - 20):
        resets = torch.zeros(B, T, device="cuda")
        resets[:, at + 9] = 1.0
        spoiled = x.clone()
        spoiled[:, at] = math.nan
        spoiled[:, at + 3, ::2] = math.inf
        want, want_final = pb.gated_recurrence(gates, x, resets=resets, state=state)
        got, got_final = pb.gated_recurrence(gates, spoiled, resets=resets, state=state)
        assert torch.equal(got[:, :at], want[:, :at]) and got[:, at:at + 9].isnan().all()
        assert torch.equal(got[:, at + 9:], want[:, at + 9:]) and torch.equal(got_final, want_final)


@pytest.mark.parametrize("shape,dtype", DIVISIONS)
def test_the_same_bits_each_time(shape, dtype):
    gates, x, state = held(shape, dtype, 7.0, seed=5)
    import pufferlib_b200 as pb
    leaves = [v.requires_grad_(True) for v in (gates, x, state)]

    def run():
        out, final = pb.gated_recurrence(*leaves[:2], state=leaves[2])
        return (out.detach(), final.detach()) + torch.autograd.grad(out.float().sum() + final.sum(), leaves)
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))
