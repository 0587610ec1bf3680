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


def traced(pb):
    """name -> (function of one tensor whose first sizes change, the shapes it is called with)"""
    def logprobs(z):
        lp, h = pb.action_logprobs(z, torch.zeros(z.shape[:-1], dtype=torch.int64, device=M))
        return lp.sum() + h.sum()

    def logprobs_of_a_slice(z):
        lp, h = pb.action_logprobs(z[:, :-1], torch.zeros(z.shape[:-1], dtype=torch.int64, device=M)[:, 1:], entropy=False)
        assert h is None
        return lp.sum()

    def loss(lp):
        out, ratio, stats = pb.policy_loss(lp, torch.empty_like(lp), torch.empty_like(lp), entropy=lp * 2, ent_coef=0.1,
                                           mask=torch.ones_like(lp, dtype=torch.bool), reduction="sequence")
        return out + (ratio.sum() + stats.sum()).detach()

    def recurrence(g):
        out, final = pb.gated_recurrence(g, g * 2, resets=torch.zeros(g.shape[:2], device=M),
                                         state=torch.zeros(g.shape[0], g.shape[2], device=M))
        return out.sum() + final.sum()

    def halves(g):
        gates, x = g.chunk(2, -1)
        return pb.gated_recurrence(gates, x)[0].sum()

    def step(g):
        with torch.no_grad():
            out, new = pb.gated_recurrence_step(g, g, torch.zeros_like(g), resets=torch.zeros(g.shape[0], device=M))
        return out.sum() + new.sum()
    return {"logprobs": (logprobs, [(4, 8), (6, 8), (9, 500)]), "logprobs 3d": (logprobs, [(4, 5, 8), (6, 3, 8), (2, 7, 700)]),
            "logprobs of a slice": (logprobs_of_a_slice, [(4, 5, 8), (6, 3, 8), (2, 7, 700)]),
            "loss": (loss, [(4, 6), (5, 6), (9, 17)]), "recurrence": (recurrence, [(2, 7, 8), (3, 9, 8), (5, 33, 20)]),
            "halves": (halves, [(2, 7, 8), (3, 9, 8), (5, 33, 20)]), "step": (step, [(4, 8), (6, 8), (9, 20)])}


NAMES = ["logprobs", "logprobs 3d", "logprobs of a slice", "loss", "recurrence", "halves", "step"]


@pytest.mark.parametrize("which", NAMES)
@pytest.mark.parametrize("dynamic", [None, True, False])
def test_compiled_with_changing_shapes(which, dynamic):
    """Traced ahead of time, forward and backward, with sizes as symbols from the second size on or from the first."""
    import pufferlib_b200 as pb
    f, shapes = traced(pb)[which]
    torch._dynamo.reset()
    compiled = torch.compile(f, backend="aot_eager", dynamic=dynamic, fullgraph=True)
    for shape in shapes:
        leaf = meta(*shape, grad=True)
        out = compiled(leaf)
        assert out.shape == ()
        if which != "step":
            assert torch.autograd.grad(out, leaf)[0].shape == shape
    torch._dynamo.reset()


@pytest.mark.parametrize("which", NAMES)
def test_traced_with_symbols(which):
    """One trace holds for other sizes: nothing in it is a number that was a size."""
    import pufferlib_b200 as pb
    from torch.fx.experimental.proxy_tensor import make_fx
    f, shapes = traced(pb)[which]

    def both(leaf):
        if which == "step":
            return f(leaf)
        leaf = leaf.detach().requires_grad_(True)
        return torch.autograd.grad(f(leaf), leaf)[0]
    graph = make_fx(both, tracing_mode="symbolic")(meta(*shapes[0]))
    other = tuple(n + 3 for n in shapes[0][:-1]) + shapes[0][-1:]
    assert graph(meta(*other)).shape == both(meta(*other)).shape


def test_without_entropy_every_path_returns_none():
    """The operator itself, with and without a graph, on tensors without data: as on the GPU."""
    import pufferlib_b200  # noqa: F401
    import pufferlib_b200 as pb
    pb.action_logprobs(meta(4, 8), actions(4))
    op = torch.ops.pufferlib.puff_action_logprobs
    assert op(meta(4, 8), actions(4), 1.0, False)[1] is None
    assert op(meta(4, 8, grad=True), actions(4), 1.0, False)[1] is None


def test_shapes_are_still_refused_while_tracing():
    import pufferlib_b200 as pb
    from torch.fx.experimental.proxy_tensor import make_fx
    for f, shape in ((lambda z: pb.action_logprobs(z, actions(5))[0], (4, 8)),
                     (lambda z: pb.policy_loss(z, meta(4, 5), meta(4, 6))[0], (4, 6)),
                     (lambda z: pb.gated_recurrence(z, meta(2, 7, 9))[0], (2, 7, 8)),
                     (lambda z: pb.gated_recurrence_step(z, z, meta(2, 9))[0], (2, 8))):
        with pytest.raises(RuntimeError, match="shape"):
            make_fx(f, tracing_mode="symbolic")(meta(*shape))


@pytest.mark.parametrize("vocab", [1, 18, 384, 385, 5000])
def test_row_statistics_are_kept_only_for_rows_that_need_them(vocab):
    """The backward pass of small rows works the statistics out again: nothing is saved for it."""
    import pufferlib_b200 as pb
    pb.action_logprobs(meta(2, 3), actions(2))
    _, _, stats = torch.ops.pufferlib.puff_action_logprobs_forward(meta(7, vocab), actions(7), 1.0, True, True)
    assert stats.shape == ((0, 2) if vocab <= 384 else (7, 2))
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.numel()) or t, lambda t: t):
        pb.action_logprobs(meta(7, vocab, grad=True), actions(7), entropy=False)
    assert sum(saved) == 7 * vocab + 7 + (14 if vocab > 384 else 0)
