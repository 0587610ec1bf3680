"""CPU: the gradients of the policy-update operators as autograd's other modes take them, on tensors without data."""
import pytest
import torch
from torch.autograd import forward_ad

M = "meta"


def meta(*shape, dtype=torch.float32, grad=False):
    return torch.empty(*shape, device=M, dtype=dtype, requires_grad=grad)


def actions(*shape):
    return meta(*shape, dtype=torch.int64)


# an operator as a function of one tensor at a time, and that tensor's shape
ONE_INPUT = {
    "logits": ((4, 8), lambda pb, t: pb.action_logprobs(t, actions(4))[0]),
    "logits without entropy": ((4, 8), lambda pb, t: pb.action_logprobs(t, actions(4), entropy=False)[0]),
    "logprobs": ((4, 6), lambda pb, t: pb.policy_loss(t, meta(4, 6), meta(4, 6))[0]),
    "old_logprobs": ((4, 6), lambda pb, t: pb.policy_loss(meta(4, 6), t, meta(4, 6))[0]),
    "advantages": ((4, 6), lambda pb, t: pb.policy_loss(meta(4, 6), meta(4, 6), t)[0]),
    "ref_logprobs": ((4, 6), lambda pb, t: pb.policy_loss(meta(4, 6), meta(4, 6), meta(4, 6), ref_logprobs=t, kl_coef=0.1)[0]),
    "entropy": ((4, 6), lambda pb, t: pb.policy_loss(meta(4, 6), meta(4, 6), meta(4, 6), entropy=t, ent_coef=0.1)[0]),
    "gates": ((2, 7, 8), lambda pb, t: pb.gated_recurrence(t, meta(2, 7, 8))[0]),
    "inputs": ((2, 7, 8), lambda pb, t: pb.gated_recurrence(meta(2, 7, 8), t)[0]),
    "state": ((2, 8), lambda pb, t: pb.gated_recurrence(meta(2, 7, 8), meta(2, 7, 8), state=t)[0]),
    "step gates": ((2, 8), lambda pb, t: pb.gated_recurrence_step(t, meta(2, 8), meta(2, 8))[0]),
    "step inputs": ((2, 8), lambda pb, t: pb.gated_recurrence_step(meta(2, 8), t, meta(2, 8))[0]),
    "step state": ((2, 8), lambda pb, t: pb.gated_recurrence_step(meta(2, 8), meta(2, 8), t, new_state=meta(2, 8))[0]),
    "step new_state": ((2, 8), lambda pb, t: pb.gated_recurrence_step(meta(2, 8), meta(2, 8), meta(2, 8), new_state=t)[0]),
}


@pytest.mark.parametrize("which", ONE_INPUT)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(which, grad):
    """A tangent would be lost on the way: there is no forward-mode derivative."""
    import pufferlib_b200 as pb
    shape, call = ONE_INPUT[which]
    if grad and which in ("old_logprobs", "advantages", "ref_logprobs") or grad and which.startswith("step"):
        pytest.skip("requires_grad is refused for itself")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(meta(*shape, grad=grad), meta(*shape))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(pb, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            call(pb, dual)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: call(pb, t), (meta(*shape),), (meta(*shape),))
    call(pb, meta(*shape))                       # outside of it nothing is refused


def test_forward_mode_over_reverse_is_refused():
    """A tangent on the incoming gradient of a backward pass."""
    import pufferlib_b200 as pb
    z, gates = meta(4, 8, grad=True), meta(2, 7, 8, grad=True)
    x = meta(4, 6, grad=True)
    for make in (lambda: (pb.action_logprobs(z, actions(4))[0], z), lambda: (pb.action_logprobs(z, actions(4))[1], z),
                 lambda: (pb.policy_loss(x, meta(4, 6), meta(4, 6))[0], x),
                 lambda: (pb.gated_recurrence(gates, meta(2, 7, 8))[0], gates),
                 lambda: (pb.gated_recurrence(gates, meta(2, 7, 8))[1], gates)):
        out, leaf = make()
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.empty_like(out), torch.empty_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaf, dual, retain_graph=True)
        torch.autograd.grad(out, leaf, torch.empty_like(out))


def second_cases(pb):
    """(output, its differentiable leaves) per operator and output."""
    z, lp, ent = meta(4, 8, grad=True), meta(4, 6, grad=True), meta(4, 6, grad=True)
    gates, x, s = meta(2, 7, 8, grad=True), meta(2, 7, 8, grad=True), meta(2, 8, grad=True)
    yield pb.action_logprobs(z, actions(4))[0], [z]
    yield pb.action_logprobs(z, actions(4))[1], [z]
    for reduction in ("token", "sequence"):
        yield pb.policy_loss(lp, meta(4, 6), meta(4, 6), reduction=reduction)[0], [lp]
        yield pb.policy_loss(lp, meta(4, 6), meta(4, 6), entropy=ent, ent_coef=0.1, reduction=reduction)[0], [lp, ent]
    yield pb.gated_recurrence(gates, x, state=s)[0], [gates, x, s]
    yield pb.gated_recurrence(gates, x, state=s)[1], [gates, x, s]


def test_second_derivatives_are_refused_for_every_leaf():
    """A gradient taken with create_graph depends on all leaves: going back through it raises, whichever is asked for
    and whatever else the result depends on."""
    import pufferlib_b200 as pb
    for out, leaves in second_cases(pb):
        grads = torch.autograd.grad(out.sum(), leaves, create_graph=True)
        assert all(g.requires_grad for g in grads)
        for g in grads:
            for leaf in leaves:
                with pytest.raises(RuntimeError, match="derivative"):
                    torch.autograd.grad((g * g).sum() + (leaf * leaf).sum(), leaf, retain_graph=True, allow_unused=True)
        # also where the second derivative goes through the incoming gradient alone
        weight = torch.ones_like(out).requires_grad_(True)
        for out, leaves in second_cases(pb):
            if out.shape != weight.shape:
                continue
            g = torch.autograd.grad(out, leaves[0], weight, create_graph=True)[0]
            with pytest.raises(RuntimeError, match="derivative"):
                torch.autograd.grad(g.sum(), weight)


def test_first_derivatives_with_create_graph():
    """create_graph itself is not refused: a trainer may ask for it for the sake of another term."""
    import pufferlib_b200 as pb
    for out, leaves in second_cases(pb):
        (out.sum() + sum((v * v).sum() for v in leaves)).backward(create_graph=True)
        for v in leaves:
            assert v.grad.shape == v.shape
            v.grad = None
    for out, leaves in second_cases(pb):
        assert not any(g.requires_grad for g in torch.autograd.grad(out.sum(), leaves))


REGIONS = {
    "head and log-probabilities": ((4, 5), lambda pb, t, w: pb.action_logprobs(t @ w, actions(4))[0]),
    "log-probabilities without entropy": ((4, 5), lambda pb, t, w: pb.action_logprobs(t @ w, actions(4), entropy=False)[0]),
    "loss": ((4, 5), lambda pb, t, w: pb.policy_loss(t @ w, meta(4, 8), meta(4), entropy=t @ w, ent_coef=0.1, reduction="sequence",
                                                     mask=meta(4, 8, dtype=torch.bool))[0]),
    "recurrence": ((2, 7, 5), lambda pb, t, w: pb.gated_recurrence(t @ w, t @ w, resets=meta(2, 7), state=(t @ w)[:, 0].contiguous())[0]),
    "recurrence, final state": ((2, 7, 5), lambda pb, t, w: pb.gated_recurrence(t @ w, t @ w)[1]),
}


@pytest.mark.parametrize("which", REGIONS)
@pytest.mark.parametrize("reentrant", [False, True])
def test_activation_checkpointing(which, reentrant):
    """The operator at the end of a region whose activations are computed again in the backward pass."""
    import pufferlib_b200 as pb
    from torch.utils.checkpoint import checkpoint
    shape, region = REGIONS[which]
    t, w = meta(*shape, grad=True), meta(5, 8, grad=True)
    out = checkpoint(lambda a, b: region(pb, a, b), t, w, use_reentrant=reentrant)
    out.sum().backward()
    assert t.grad.shape == t.shape and w.grad.shape == w.shape
    # two regions in a row, and twice through the same graph
    t.grad = w.grad = None
    twice = sum(checkpoint(lambda a, b: region(pb, a, b), t, w, use_reentrant=reentrant).sum() for _ in range(2))
    if not reentrant:
        twice.backward(retain_graph=True)
    twice.backward()
    assert t.grad.shape == t.shape


def test_unpack_hooks_run_under_autograd():
    """Whatever a saved-tensor hook computes is recorded as under torch's own nodes."""
    import pufferlib_b200 as pb
    for which, (shape, region) in REGIONS.items():
        t, w, seen = meta(*shape, grad=True), meta(5, 8, grad=True), []

        def unpack(v):
            with torch.enable_grad():
                seen.append((torch.ones(2, requires_grad=True) * 2).requires_grad)
            return v
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, unpack):
            out = region(pb, t, w)
        out.sum().backward()
        assert len(seen) >= 3 and all(seen), which
