"""CPU: what the policy-update operators refuse, their shapes, and the host-side checks of their C entry points."""
import ctypes

import pytest
import torch

M = "meta"


def meta(*shape, dtype=torch.float32, grad=False):
    return torch.empty(*shape, device=M, dtype=dtype, requires_grad=grad)


def test_shapes_and_autograd_without_a_gpu():
    import pufferlib_b200 as pb
    z = meta(3, 5, 11, dtype=torch.bfloat16, grad=True)
    lp, H = pb.action_logprobs(z, meta(3, 5, dtype=torch.int64))
    assert lp.shape == H.shape == (3, 5) and lp.dtype == H.dtype == torch.float32
    (d,) = torch.autograd.grad(lp.sum() + H.sum(), z)
    assert d.shape == z.shape and d.dtype == torch.bfloat16
    lp, H = pb.action_logprobs(z.detach(), meta(3, 5, dtype=torch.int64), entropy=False)
    assert H is None and not lp.requires_grad
    lp, ent = meta(4, 6, grad=True), meta(4, 6, grad=True)
    loss, ratio, stats = pb.policy_loss(lp, meta(4, 6), meta(4), entropy=ent, ent_coef=0.1, mask=meta(4, 6, dtype=torch.bool), reduction="sequence")
    assert loss.shape == () and ratio.shape == (4, 6) and stats.shape == (6,) and not ratio.requires_grad
    assert [g.shape for g in torch.autograd.grad(loss, [lp, ent])] == [(4, 6)] * 2
    gates, s = meta(2, 7, 8, grad=True), meta(2, 8, grad=True)
    out, final = pb.gated_recurrence(gates, meta(2, 7, 8), resets=meta(2, 7), state=s)
    assert out.shape == (2, 7, 8) and final.shape == (2, 8)
    assert [g.shape for g in torch.autograd.grad(final.sum(), [gates, s])] == [(2, 7, 8), (2, 8)]
    o, n = pb.gated_recurrence_step(meta(2, 8, dtype=torch.float16), meta(2, 8, dtype=torch.float16), meta(2, 8))
    assert o.shape == n.shape == (2, 8) and o.dtype == torch.float16


@pytest.mark.parametrize("logits,actions,kw", [
    (lambda: meta(4, 8, dtype=torch.float64), lambda: meta(4, dtype=torch.int64), {}),
    (lambda: meta(4, 8), lambda: meta(4, dtype=torch.int32), {}),
    (lambda: meta(4, 8), lambda: meta(5, dtype=torch.int64), {}),
    (lambda: meta(4, 8), lambda: meta(4, 8, dtype=torch.int64), {}),
    (lambda: meta(8, 4).t(), lambda: meta(4, dtype=torch.int64), {}),
    (lambda: meta(4, 0), lambda: meta(4, dtype=torch.int64), {}),
    (lambda: meta(4, 8), lambda: meta(4, dtype=torch.int64), {"temperature": 0.0}),
    (lambda: meta(4, 8), lambda: meta(4, dtype=torch.int64), {"temperature": -1.0}),
    (lambda: meta(4, 8), lambda: meta(4, dtype=torch.int64), {"temperature": float("nan")}),
    (lambda: meta(9, 9, 9, 9)[::2, ::2, ::2], lambda: meta(5, 5, 5, dtype=torch.int64), {}),
    (lambda: meta(4, 6, 8).transpose(0, 1)[:, :3], lambda: meta(3, 6, dtype=torch.int64), {}),
    (lambda: meta(()), lambda: meta((), dtype=torch.int64), {}),
])
def test_logprobs_refusals(logits, actions, kw):
    import pufferlib_b200 as pb
    with pytest.raises(RuntimeError):
        pb.action_logprobs(logits(), actions(), **kw)


@pytest.mark.parametrize("change", [
    dict(logprobs=meta(24)), dict(logprobs=meta(4, 6, dtype=torch.bfloat16)), dict(old_logprobs=meta(4, 5)),
    dict(old_logprobs=meta(6, 4).t()), dict(advantages=meta(6)), dict(advantages=meta(1, 6)), dict(advantages=meta(4, 6, 1)),
    dict(mask=meta(4, 6)), dict(mask=meta(4, dtype=torch.bool)), dict(mask=meta(6, 4, dtype=torch.bool).t()),
    dict(ref_logprobs=meta(4)), dict(entropy=meta(4, 6, dtype=torch.float64)), dict(clip_low=-0.1), dict(clip_high=float("nan")),
    dict(reduction="mean"), dict(denominator=0.0), dict(denominator=-3.0), dict(kl_coef=0.1), dict(ent_coef=0.1),
    dict(old_logprobs=meta(4, 6, grad=True)), dict(advantages=meta(4, 6, grad=True)), dict(ref_logprobs=meta(4, 6, grad=True)),
])
def test_policy_loss_refusals(change):
    import pufferlib_b200 as pb
    args = dict(logprobs=meta(4, 6), old_logprobs=meta(4, 6), advantages=meta(4, 6)) | change
    with pytest.raises((RuntimeError, ValueError)):
        pb.policy_loss(**args)


@pytest.mark.parametrize("change", [
    dict(gates=meta(2, 7)), dict(gates=meta(2, 7, 9)), dict(inputs=meta(2, 7, 8, dtype=torch.float16)),
    dict(gates=meta(2, 7, 8, dtype=torch.float64), inputs=meta(2, 7, 8, dtype=torch.float64)),
    dict(gates=meta(2, 8, 7).transpose(1, 2)), dict(resets=meta(2, 8)), dict(resets=meta(7, 2).t()),
    dict(resets=meta(2, 7, dtype=torch.int64)), dict(state=meta(2, 7)), dict(state=meta(2, 8, dtype=torch.bfloat16)),
    dict(state=meta(8, 2).t()),
])
def test_recurrence_refusals(change):
    import pufferlib_b200 as pb
    args = dict(gates=meta(2, 7, 8), inputs=meta(2, 7, 8)) | change
    with pytest.raises(RuntimeError):
        pb.gated_recurrence(**args)


def test_step_refusals():
    import pufferlib_b200 as pb
    ok = dict(gates=meta(4, 8), inputs=meta(4, 8), state=meta(4, 8))
    for change in (dict(gates=meta(4, 1, 8)), dict(state=meta(4, 7)), dict(state=meta(8, 4).t()), dict(resets=meta(4, 1)),
                   dict(new_state=meta(4, 8, dtype=torch.float16)), dict(gates=meta(4, 8, grad=True)), dict(state=meta(4, 8, grad=True))):
        with pytest.raises(RuntimeError):
            pb.gated_recurrence_step(**(ok | change))


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU failure mode")
def test_no_cpu_fallback():
    import pufferlib_b200 as pb
    with pytest.raises((RuntimeError, NotImplementedError)):
        pb.action_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises((RuntimeError, NotImplementedError)):
        pb.policy_loss(torch.zeros(2, 3), torch.zeros(2, 3), torch.zeros(2, 3))
    with pytest.raises((RuntimeError, NotImplementedError)):
        pb.gated_recurrence(torch.zeros(2, 3, 4), torch.zeros(2, 3, 4))


class Host:
    """A host buffer whose address stands in for a device pointer: everything below is refused before a launch."""

    def __init__(self, size=1 << 14):
        self.buffer = (ctypes.c_char * size)()
        self.base = (ctypes.addressof(self.buffer) + 255) & ~255

    def __getitem__(self, offset):
        return self.base + offset


def test_logprobs_entry_point_checks():
    from pufferlib_b200 import cabi
    lib, h = cabi.load(), Host()
    ok = dict(logits=h[0], dtype=cabi.DTYPE_F32, actions=h[1024], outer=1, inner=4, vocab=8, los=0, lis=8, aos=0, ais=1, t=1.0,
              lp=h[2048], ent=h[2304], stats=h[2560])

    def call(**kw):
        a = ok | kw
        return lib.puff_policy_sm100_logprobs(a["logits"], a["dtype"], a["actions"], a["outer"], a["inner"], a["vocab"], a["los"],
                                              a["lis"], a["aos"], a["ais"], a["t"], a["lp"], a["ent"], a["stats"], None)
    assert call(dtype=7) == cabi.ERR_DTYPE
    assert call(inner=-1) == call(vocab=0) == call(lis=-8) == cabi.ERR_SHAPE
    assert call(t=0.0) == call(t=-1.0) == call(t=float("nan")) == call(t=float("inf")) == call(t=1e-39) == cabi.ERR_VALUE
    assert call(outer=1 << 30, inner=1 << 30) == cabi.ERR_SIZE
    assert call(logits=None) == call(actions=None) == call(lp=None) == cabi.ERR_NULL
    assert call(logits=h[2]) == call(actions=h[1028]) == call(lp=h[2050]) == call(stats=h[2564]) == cabi.ERR_ALIGN
    assert call(lp=h[64]) == call(lp=h[1024]) == call(ent=h[2048]) == call(stats=h[2304]) == cabi.ERR_ALIAS
    assert call(outer=0) == call(inner=0, logits=None) == cabi.OK

    def back(**kw):
        a = ok | dict(dlp=h[3072], dent=h[3328], out=h[4096]) | kw
        return lib.puff_policy_sm100_logprobs_backward(a["logits"], a["dtype"], a["actions"], a["outer"], a["inner"], a["vocab"],
                                                       a["los"], a["lis"], a["aos"], a["ais"], a["t"], a["stats"], a["ent"], a["dlp"],
                                                       a["dent"], a["out"], None)
    assert back(stats=None) == back(dlp=None) == back(out=None) == back(ent=None) == cabi.ERR_NULL
    assert back(out=h[0]) == back(out=h[1000]) == back(out=h[3072]) == back(out=h[2560]) == cabi.ERR_ALIAS
    assert back(out=h[4097]) == cabi.ERR_ALIGN and back(inner=0) == cabi.OK


def test_loss_entry_point_checks():
    from pufferlib_b200 import cabi
    lib, h = cabi.load(), Host(1 << 20)
    need = lib.puff_policy_sm100_loss_scratch_bytes(4, 8)
    ok = dict(lp=h[0], old=h[256], adv=h[512], per_row=0, ref=h[768], ent=h[1024], mask=h[1280], low=0.2, high=0.2, kl=0.1, ec=0.1,
              red=0, den=0.0, rows=4, steps=8, loss=h[1536], ratio=h[1792], stats=h[2048], slope=h[2304], scale=h[2560], weight=h[2816],
              scratch=h[4096], size=need)

    def call(**kw):
        return lib.puff_policy_sm100_loss(*(ok | kw).values(), None)
    assert call(rows=-1) == cabi.ERR_SHAPE and call(rows=1 << 30, steps=1 << 30) == cabi.ERR_SIZE
    assert call(low=-0.1) == call(high=float("nan")) == call(red=2) == call(den=-1.0) == call(den=float("inf")) == cabi.ERR_VALUE
    assert call(lp=None) == call(loss=None) == call(ratio=None) == call(weight=None) == call(red=1, scale=None) == cabi.ERR_NULL
    assert call(scratch=None) == call(size=need - 1) == call(scratch=h[4100]) == cabi.ERR_WORKSPACE
    assert call(lp=h[2]) == call(slope=h[2305]) == cabi.ERR_ALIGN
    assert call(ratio=h[0]) == call(slope=h[1792]) == call(loss=h[1284]) == call(scratch=h[2048]) == cabi.ERR_ALIAS
    back = dict(slope=h[0], scale=h[256], weight=h[512], dloss=h[768], mask=h[1024], ec=0.1, rows=4, steps=8, dlp=h[1280], dent=h[1536])
    run = lambda **kw: lib.puff_policy_sm100_loss_backward(*(back | kw).values(), None)  # noqa: E731
    assert run(slope=None) == run(dloss=None) == cabi.ERR_NULL and run(dlp=None, dent=None) == run(steps=0) == cabi.OK
    assert run(dlp=h[0]) == run(dent=h[1280]) == cabi.ERR_ALIAS and run(dlp=h[1281]) == cabi.ERR_ALIGN and run(rows=-4) == cabi.ERR_SHAPE


def test_recurrence_entry_point_checks():
    from pufferlib_b200 import cabi
    lib, h = cabi.load(), Host(1 << 21)
    assert lib.puff_policy_sm100_recurrence_saved_floats(2, 3, 0) == 0 and lib.puff_policy_sm100_recurrence_saved_floats(2, 3, 4) >= 8
    ok = dict(gates=h[0], inputs=h[512], dtype=0, resets=h[1024], rb=4, state=h[1280], B=2, T=5, C=4, gb=20, gs=4, ib=20, is_=4,
              out=h[2048], final=h[3072], saved=h[4096], scratch=None, size=0)
    run = lambda **kw: lib.puff_policy_sm100_recurrence(*(ok | kw).values(), None)  # noqa: E731
    assert run(dtype=3) == run(rb=2) == cabi.ERR_DTYPE
    assert run(B=-1) == run(gs=-4) == cabi.ERR_SHAPE and run(B=1 << 30, C=1 << 30) == run(T=1 << 40) == cabi.ERR_SIZE
    assert run(gates=None) == run(final=None) == run(out=None) == cabi.ERR_NULL
    assert run(gates=h[2]) == run(state=h[1281]) == run(final=h[3073]) == cabi.ERR_ALIGN
    assert run(out=h[0]) == run(out=h[600]) == run(final=h[1280]) == run(saved=h[2048]) == run(final=h[1024]) == cabi.ERR_ALIAS
    assert run(B=0) == run(C=0) == cabi.OK
    # one long row is cut into ranges whose joins need a workspace
    big = dict(T=4000, gb=0, gs=0, ib=0, is_=0, resets=None, saved=None, out=h[1 << 20], final=h[4096])
    need = lib.puff_policy_sm100_recurrence_scratch_bytes(2, 4000, 4)
    assert need >= 16 and lib.puff_policy_sm100_recurrence_scratch_bytes(1 << 14, 64, 512) == 0
    assert run(**big) == run(**big, scratch=h[8192], size=need - 1) == run(**big, scratch=h[8196], size=need) == cabi.ERR_WORKSPACE
    assert run(**big, scratch=h[4096], size=need) == run(**big, scratch=h[1 << 20], size=need) == cabi.ERR_ALIAS
    b = dict(gates=h[0], inputs=h[512], dtype=0, resets=h[1024], rb=4, saved=h[1280], B=2, T=5, C=4, gb=20, gs=4, ib=20, is_=4,
             dout=h[4096], dfinal=h[5120], dg=h[6144], dx=h[7168], ds=h[8192], scratch=None, size=0)
    back = lambda **kw: lib.puff_policy_sm100_recurrence_backward(*(b | kw).values(), None)  # noqa: E731
    assert back(saved=None) == back(dg=None) == cabi.ERR_NULL and back(dg=h[4096]) == back(dx=h[6144]) == back(ds=h[1280]) == cabi.ERR_ALIAS
    s = dict(gates=h[0], inputs=h[512], dtype=0, resets=h[1024], rb=4, state=h[1280], B=2, C=4, gs=4, is_=4, out=h[2048], new=h[3072])
    step = lambda **kw: lib.puff_policy_sm100_recurrence_step(*(s | kw).values(), None)  # noqa: E731
    assert step(state=None) == step(out=None) == cabi.ERR_NULL and step(new=h[1284]) == step(out=h[1280]) == step(new=h[0]) == cabi.ERR_ALIAS
    assert step(B=0) == cabi.OK and step(dtype=-1) == cabi.ERR_DTYPE


def test_error_texts():
    from pufferlib_b200 import cabi
    for code in (cabi.ERR_DTYPE, cabi.ERR_VALUE):
        assert cabi.strerror(code) != "unknown error code"
