"""GPU: log-probabilities of confident rows over vocabularies too long for one read, to a few steps of fp32.

Rows with two actions that are not illegal: a rival and, far behind it in the row, the chosen one d above.  Then
s = 1 + e, e = exp(-d), and nothing else is added, so that few roundings are left (U = 2^-24, half a step at 1):
  e          4 U from ex2.approx, 3 U d from its argument
  1          4 U from ex2.approx of the remainder of max * log2(e) twice: in the term and in the factor that takes it out
  s          2 U: one sum, one product
so s is off by 10 U + e (4 + 3 d) U at most, log s by as much and 2 U log s, and the log-probability by one more rounding
of each.  The entropy log s - u / s has e d (ex2's 4, the argument's 3 d, and 8 more) U on top.

That is with the sums taken relative to the row's maximum.  The kernel's reference may lie 4.4 bits below it, which on
paper is 3 U more for the argument of the largest term; what is met here is 3 U in all."""
import math

import pytest
import torch

from policy_reference import U, within
from test_policy_ops_gpu import BF16, F16, F32

pytestmark = pytest.mark.gpu


def confident(rows, vocab, distance, dtype, base):
    """Chosen `distance` entries behind its rival, in another place of the row each; both values exact in `dtype`."""
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    logits = torch.full((rows, vocab), -math.inf, device="cuda")
    at = torch.randint(0, vocab - distance, (rows,), device="cuda", generator=g)
    d = (torch.randint(1, 8 * 16, (rows,), device="cuda", generator=g) / 16.0 + 1.0)
    r = torch.arange(rows, device="cuda")
    logits[r, at] = base
    logits[r, at + distance] = base + d
    out = logits.to(dtype)
    assert torch.equal(out.float(), logits)
    return out, at, at + distance, d.double()


# distances of a whole number of rounds of the threads' vectors, so that one thread meets both, for a warp a row, a CTA a
# row, and clusters of up to eight
@pytest.mark.parametrize("rows,vocab,distance", [(3000, 1600, 1024), (3000, 4096, 2048), (700, 9001, 4096), (700, 50001, 32768),
                                                 (40, 70001, 32768), (3, 131072, 65536), (3000, 515, 300)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_confident_rows(rows, vocab, distance, dtype):
    import pufferlib_b200 as pb
    for base in (0.0, -4.0):
        logits, rival, chosen, d = confident(rows, vocab, distance, dtype, base)
        e = (-d).exp()
        s_err = U * (10 + e * (4 + 3 * d))
        for actions, lp in ((chosen, -torch.log1p(e)), (rival, -d - torch.log1p(e))):
            got, entropy = pb.action_logprobs(logits, actions)
            within(got, lp, s_err + 2 * U * torch.log1p(e) + 4 * U * (lp.abs() + (lp + torch.log1p(e)).abs()), "logprobs")
            H = torch.log1p(e) + e * d / (1 + e)
            within(entropy, H, s_err + 4 * U * torch.log1p(e) + U * e * d * (24 + 3 * d) + 2 * U * H, "entropy")


@pytest.mark.parametrize("rows,vocab", [(3000, 1500), (700, 9001), (40, 131072), (3, 131072)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_chain_of_ever_larger_logits(rows, vocab, dtype):
    """Each stretch of a row lies above the one before it: the reference of the sums is replaced again and again."""
    import policy_reference as ref
    import pufferlib_b200 as pb
    g = torch.Generator(device="cuda").manual_seed(vocab)
    ramp = torch.linspace(0, 60, vocab, device="cuda").floor() * 0.75
    logits = (ramp + torch.rand(rows, vocab, device="cuda", generator=g)).to(dtype)
    actions = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    lp, H = pb.action_logprobs(logits, actions)
    # a thread's own chain of sums, sixteen or eight terms at a time, and a dozen joins
    want = ref.logprobs(logits, actions, 1.0, chain=vocab / 64)
    within(lp, *want["logprobs"], "logprobs")
    within(H, *want["entropy"], "entropy")


@pytest.mark.parametrize("rows,vocab", [(4000, 4000), (600, 9001), (300, 131072), (8, 131072), (2, 200003)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_no_logit_is_left_out(rows, vocab, dtype):
    """Equal logits: log s = log V to a few roundings, so that a sum short of one vector of eight would show."""
    import pufferlib_b200 as pb
    logits = torch.full((rows, vocab), 1.5, device="cuda", dtype=dtype)
    actions = torch.arange(rows, device="cuda") * 7 % vocab
    lp, H = pb.action_logprobs(logits, actions)
    # terms 2^r with r the remainder of the maximum: 8 U; sums of equal numbers by halves and in short chains
    bound = U * (8 + 40) + 2 * U * math.log(vocab)
    assert bound < 0.5 * 8 / vocab or vocab > 131072
    want = torch.full((rows,), math.log(vocab), dtype=torch.float64)
    within(lp, -want, torch.full_like(want, bound), "logprobs")
    within(H, want, torch.full_like(want, bound), "entropy")
