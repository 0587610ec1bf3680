"""GPU: a wait for a tile that runs out is reported, and the kernel ends with none of its copies in flight."""
import pytest
import torch

from test_policy_ops_gpu import BF16, F32, gen, randn

pytestmark = pytest.mark.gpu

# one warp a tile, warps of a CTA, ranges of steps, clusters
SHAPES = [((8192, 64, 128), BF16), ((256, 512, 128), F32), ((1, 6000, 512), BF16), ((3, 1500, 1024), F32)]


@pytest.mark.parametrize("shape,dtype", SHAPES)
def test_a_wait_that_runs_out_is_reported(shape, dtype):
    """With no time to wait every warp gives up at its first tile, which is on its way."""
    import pufferlib_b200 as pb
    from pufferlib_b200 import cabi
    g = gen(1)
    leaves = [randn(g, *shape).to(dtype).requires_grad_(True), randn(g, *shape).to(dtype).requires_grad_(True)]
    dout, dfinal = randn(g, *shape).to(dtype), randn(g, shape[0], shape[2])

    def forward():
        return pb.gated_recurrence(*leaves)

    def backward(outs):
        return torch.autograd.grad(outs, leaves, [dout, dfinal], retain_graph=True)
    outs = forward()
    want = [t.detach() for t in outs] + list(backward(outs))
    assert cabi.device_status() == 0
    try:
        cabi.set_tuning(tile_wait_us=0)
        forward()
        assert cabi.device_status() == cabi.ERR_DEVICE_WAIT
        backward(outs)
        assert cabi.device_status() == cabi.ERR_DEVICE_WAIT
        assert cabi.device_status() == 0
    finally:
        cabi.set_tuning(tile_wait_us=None)
    again = forward()
    got = [t.detach() for t in again] + list(backward(again))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert cabi.device_status() == 0


def test_a_short_limit_is_enough_for_tiles_that_come():
    import pufferlib_b200 as pb
    from pufferlib_b200 import cabi
    g = gen(2)
    gates, x = randn(g, 64, 200, 128), randn(g, 64, 200, 128)
    want = pb.gated_recurrence(gates, x)
    try:
        cabi.set_tuning(tile_wait_us=500000)
        got = pb.gated_recurrence(gates, x)
    finally:
        cabi.set_tuning(tile_wait_us=None)
    assert cabi.device_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(want, got))
