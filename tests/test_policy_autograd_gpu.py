"""GPU: the policy-update operators under activation checkpointing and ahead-of-time tracing give what they give alone."""
import math

import pytest
import torch

import pufferlib_b200 as pb
from test_policy_ops_gpu import gen, randn

pytestmark = pytest.mark.gpu


def segment(obs, w_gate, w_in, head, tokens, terminals, old, adv):
    h, _ = pb.gated_recurrence(obs @ w_gate, obs @ w_in, resets=terminals)
    logprobs, entropy = pb.action_logprobs(h @ head, tokens)
    loss, ratio, stats = pb.policy_loss(logprobs, old, adv, entropy=entropy, ent_coef=0.01)
    return loss


def inputs(S, H, seed, D=12, C=40, A=9):
    g = gen(seed)
    weights = [randn(g, D, C) / D ** 0.5, randn(g, D, C) / D ** 0.5, randn(g, C, A) / C ** 0.5]
    data = [randn(g, S, H, D)]
    rest = [torch.randint(0, A, (S, H), device="cuda", generator=g), (torch.rand(S, H, device="cuda", generator=g) < 0.05).float(),
            -torch.rand(S, H, device="cuda", generator=g) - math.log(A) + 0.5, randn(g, S, H)]
    return data, [w.requires_grad_(True) for w in weights], rest


@pytest.mark.parametrize("S,H", [(24, 30), (3, 300)])
def test_checkpointed_regions_give_the_same_gradients(S, H):
    from torch.utils.checkpoint import checkpoint
    (obs,), weights, rest = inputs(S, H, seed=1)
    want = torch.autograd.grad(segment(obs, *weights, *rest), weights)
    got = torch.autograd.grad(checkpoint(segment, obs, *weights, *rest, use_reentrant=False), weights)
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    def layer(o, a, b):
        return pb.gated_recurrence(o @ a, o @ b, resets=rest[1])[0]

    def logits(h, w):
        return pb.action_logprobs(h @ w, rest[0])
    h = checkpoint(layer, obs, *weights[:2], use_reentrant=False)
    lp, ent = checkpoint(logits, h, weights[2], use_reentrant=False)
    loss = checkpoint(lambda a, b: pb.policy_loss(a, rest[2], rest[3], entropy=b, ent_coef=0.01)[0], lp, ent, use_reentrant=False)
    got = torch.autograd.grad(loss, weights)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dynamic", [None, True])
def test_traced_programs_give_the_same_values(dynamic):
    torch._dynamo.reset()
    compiled = torch.compile(segment, backend="aot_eager", dynamic=dynamic, fullgraph=True)
    for S, H in ((24, 30), (16, 30), (5, 17), (40, 200)):
        (obs,), weights, rest = inputs(S, H, seed=S)
        want_loss, got_loss = segment(obs, *weights, *rest), compiled(obs, *weights, *rest)
        assert torch.equal(want_loss, got_loss)
        want, got = torch.autograd.grad(want_loss, weights), torch.autograd.grad(got_loss, weights)
        for a, b in zip(want, got):      # the products around the operators may be laid out anew: 100 roundings of fp32
            assert (a - b).norm() <= 100 * 2.0 ** -24 * a.norm()
    torch._dynamo.reset()


def test_refusals_on_the_device():
    """Forward mode and second derivatives with real tensors."""
    from torch.autograd import forward_ad
    z, tokens = torch.randn(4, 9, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        pb.action_logprobs(forward_ad.make_dual(z, z), tokens)
    lp = torch.randn(4, 6, device="cuda", requires_grad=True)
    loss, _, _ = pb.policy_loss(lp, torch.zeros(4, 6, device="cuda"), torch.ones(4, 6, device="cuda"))
    (d,) = torch.autograd.grad(loss, lp, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad((d * d).sum() + (lp * lp).sum(), lp)
