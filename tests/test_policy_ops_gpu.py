"""GPU: log-probabilities, clipped policy loss and gated recurrence against their formulas in 64 bits."""
import math

import pytest
import torch

import policy_reference as ref
from policy_reference import within

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


# ---- log-probabilities -------------------------------------------------------------------------------------------

def check_logprobs(logits, actions, temperature=1.0, entropy=True, seed=0):
    import pufferlib_b200 as pb
    g = gen(seed + 1000)
    leaf = logits.detach().requires_grad_(True)
    lp, H = pb.action_logprobs(leaf, actions, temperature=temperature, entropy=entropy)
    dlp, dH = randn(g, *actions.shape), randn(g, *actions.shape)
    outs, grads = ([lp, H], [dlp, dH]) if entropy else ([lp], [dlp])
    (dlogits,) = torch.autograd.grad(outs, leaf, grads)
    want = ref.logprobs(logits, actions, temperature, dlp, dH if entropy else None)
    assert lp.dtype == F32 and dlogits.dtype == logits.dtype and dlogits.is_contiguous()
    within(lp, *want["logprobs"], "logprobs")
    if entropy:
        within(H, *want["entropy"], "entropy")
    within(dlogits, *want["dlogits"], "dlogits")
    with torch.no_grad():                       # without a graph: the same values
        lp2, H2 = pb.action_logprobs(logits, actions, temperature=temperature, entropy=entropy)
    assert torch.equal(lp2, lp.detach()) and (H2 is None if not entropy else torch.equal(H2, H.detach()))
    return lp, H, dlogits


VOCABS = [1, 2, 3, 4, 5, 7, 8, 15, 18, 31, 32, 33, 64, 65, 127, 128, 200, 255, 256, 257, 384, 385, 500, 512, 513, 1000, 1024,
          1025, 2047, 2048, 2049, 4097, 10007, 33000, 70001]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_logprobs_sizes(vocab, dtype):
    for rows, seed in ((1, 0), (2, 1), (67, 2)):
        g = gen(seed + vocab)
        logits = (randn(g, rows, vocab) * 2.5).to(dtype)
        actions = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
        check_logprobs(logits, actions, seed=seed)


@pytest.mark.parametrize("rows,vocab,dtype", [(1, 200003, BF16), (3, 131072, F16), (40, 100001, F32), (700, 9001, BF16),
                                              (20000, 18, F32), (20001, 6, BF16), (5000, 333, F16), (149, 50001, BF16)])
def test_logprobs_rows_and_vocabularies(rows, vocab, dtype):
    g = gen(7)
    logits = (randn(g, rows, vocab) * 3.0).to(dtype)
    actions = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    check_logprobs(logits, actions, temperature=0.7)
    check_logprobs(logits, actions, entropy=False)


@pytest.mark.parametrize("vocab,pitch", [(18, 18), (18, 21), (18, 24), (333, 333), (333, 340), (5001, 5001), (5001, 5003), (5001, 5008)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprobs_strided_rows_and_padding(vocab, pitch, dtype):
    """logits[:, :-1, :vocab] of a wider tensor, actions[:, 1:]: read in place, at any alignment of a row."""
    g = gen(vocab)
    full = (randn(g, 5, 9, pitch) * 2.0).to(dtype)
    logits = full[:, :-1, :vocab]
    tokens = torch.randint(0, vocab, (5, 9), device="cuda", generator=g)
    tokens[torch.rand(5, 9, device="cuda", generator=g) < 0.25] = -1
    full[:, -1] = math.nan                       # not part of the rows
    full[:, :, vocab:] = math.nan
    check_logprobs(logits, tokens[:, 1:])
    check_logprobs(logits.transpose(0, 1), tokens[:, 1:].t())
    check_logprobs(logits, tokens[:, 1:].contiguous())
    check_logprobs(full[2, 3, 1:vocab], tokens[0, 0].clamp(0, vocab - 2))     # one row, zero-dimensional action
    # padding is zeros whatever its logits hold
    poisoned = full.clone()
    poisoned[:, :-1][tokens[:, 1:] < 0] = math.nan
    check = check_logprobs(poisoned[:, :-1, :vocab], tokens[:, 1:])
    assert not check[2].isnan().any()


@pytest.mark.parametrize("vocab", [1, 18, 300, 6000, 40000])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_logprobs_illegal_actions(vocab, dtype):
    """Masks of -inf and of the type's lowest value, rows with one legal action, rows with none, NaN and +inf."""
    import pufferlib_b200 as pb
    g = gen(3)
    rows = 12
    logits = (randn(g, rows, vocab) * 2.0).to(dtype)
    legal = torch.rand(rows, vocab, device="cuda", generator=g) < 0.5
    actions = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    legal[torch.arange(rows), actions] = True
    logits[~legal] = -math.inf
    low = torch.finfo(dtype).min
    logits[0] = -math.inf                                   # nothing legal
    logits[1] = -math.inf
    logits[1, actions[1]] = 0.5                             # one legal action
    logits[2] = torch.where(legal[2], logits[2], low)       # the lowest value as a mask
    logits[3] = low                                         # all of it: the uniform distribution
    if vocab > 1:
        logits[4, actions[4]] = -math.inf                   # the chosen action itself is illegal
    logits[5] = torch.where(legal[5], torch.full_like(logits[5], low), logits[5])   # lowest and -inf only
    lp, H, d = check_logprobs(logits, actions)
    assert lp[0] == -math.inf and H[0] == 0 and not d[0].any()
    assert lp[1] == 0 and H[1] == 0
    if vocab > 1:
        assert lp[4] == -math.inf or not (logits[4] > -math.inf).any()
    # NaN and +inf spoil their own row and no other
    spoiled = logits.clone()
    spoiled[7, vocab // 2] = math.nan
    spoiled[8, vocab // 3] = math.inf
    leaf = spoiled.requires_grad_(True)
    lp2, H2 = pb.action_logprobs(leaf, actions)
    (d2,) = torch.autograd.grad([lp2, H2], leaf, [torch.ones_like(lp2), torch.ones_like(H2)])
    for r in (7, 8):
        assert lp2[r].isnan() and H2[r].isnan() and d2[r].isnan().all()
    others = [r for r in range(rows) if r not in (7, 8)]
    assert torch.equal(lp2[others], lp[others]) and torch.equal(H2[others], H[others]) and not d2[others].isnan().any()


@pytest.mark.parametrize("vocab", [18, 40000])
def test_logprobs_large_values_and_offsets(vocab):
    g = gen(5)
    actions = torch.randint(0, vocab, (6,), device="cuda", generator=g)
    for scale, shift in ((50.0, 0.0), (1.0, 30000.0), (1e30, 0.0), (0.0, -7.0)):
        check_logprobs(randn(g, 6, vocab) * scale + shift, actions)
    check_logprobs(randn(g, 6, vocab), actions, temperature=1e-3)
    check_logprobs(randn(g, 6, vocab), actions, temperature=50.0)


def test_logprobs_bad_actions_are_flagged():
    import pufferlib_b200 as pb
    for vocab in (18, 40000):
        logits = torch.zeros(4, vocab, device="cuda", requires_grad=True)
        pb.bad_action()
        lp, H = pb.action_logprobs(logits, torch.tensor([0, vocab, -5, vocab - 1], device="cuda"))
        (d,) = torch.autograd.grad(lp.sum() + H.sum(), logits)
        assert lp[1] == 0 and H[1] == 0 and not d[1].any() and lp[2] == 0 and lp[3] != 0
        assert pb.bad_action() and not pb.bad_action()


def test_logprobs_gradient_against_differences():
    import pufferlib_b200 as pb
    g = gen(11)
    for vocab in (18, 3001):
        logits = randn(g, 9, vocab).requires_grad_(True)
        actions = torch.randint(0, vocab, (9,), device="cuda", generator=g)
        w, v, direction = randn(g, 9), randn(g, 9), randn(g, 9, vocab).double()
        lp, H = pb.action_logprobs(logits, actions, temperature=0.8)
        (d,) = torch.autograd.grad((w * lp + v * H).sum(), logits)

        def f(z):
            logp = torch.log_softmax(z / float(torch.tensor(0.8)), -1)
            return (w.double() * logp.gather(-1, actions[:, None])[:, 0] - v.double() * (logp.exp() * logp).sum(-1)).sum()
        step = 1e-5
        slope = (f(logits.detach().double() + step * direction) - f(logits.detach().double() - step * direction)) / (2 * step)
        terms = d.double() * direction
        # differences: third derivative times step^2, and 2^-52 |f| / step
        assert abs(terms.sum() - slope) <= 1e-6 * terms.abs().sum() + 1e-7 * (1 + slope.abs())


def test_logprobs_empty():
    import pufferlib_b200 as pb
    lp, H = pb.action_logprobs(torch.empty(0, 7, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"))
    assert lp.shape == (0,) and H.shape == (0,)
    z = torch.empty(3, 0, 7, device="cuda", requires_grad=True)
    lp, H = pb.action_logprobs(z, torch.empty(3, 0, dtype=torch.int64, device="cuda"))
    assert torch.autograd.grad(lp.sum(), z)[0].shape == (3, 0, 7)


def test_logprobs_beyond_32_bit_offsets():
    """More than 2^31 elements (4.4 GB): the last rows are checked."""
    import pufferlib_b200 as pb
    vocab, rows = 140001, 15500
    logits = torch.zeros(rows, vocab, device="cuda", dtype=BF16)
    g = gen(2)
    actions = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    logits[-3:] = randn(g, 3, vocab).to(BF16)
    leaf = logits.requires_grad_(True)
    lp, H = pb.action_logprobs(leaf, actions)
    dlp, dH = randn(g, rows), randn(g, rows)
    (d,) = torch.autograd.grad([lp, H], leaf, [dlp, dH])
    want = ref.logprobs(logits.detach()[-3:], actions[-3:], 1.0, dlp[-3:], dH[-3:])
    within(lp[-3:], *want["logprobs"], "logprobs")
    within(d[-3:], *want["dlogits"], "dlogits")
    assert (lp[:-3] + math.log(vocab)).abs().max() < 1e-3


# ---- policy loss -------------------------------------------------------------------------------------------------

def loss_inputs(rows, steps, seed, per_row=False, masked=False):
    g = gen(seed)
    lp = -(randn(g, rows, steps) - 1.0).abs()
    old = lp + 0.2 * randn(g, rows, steps)
    rf = lp + 0.4 * randn(g, rows, steps)
    adv = randn(g, rows) if per_row else randn(g, rows, steps)
    ent = torch.rand(rows, steps, device="cuda", generator=g)
    mask = None
    if masked:
        mask = torch.rand(rows, steps, device="cuda", generator=g) < 0.6
        if rows > 2:
            mask[1] = False                     # a row with nothing left
            mask[2] = True
    return lp, old, adv, rf, ent, mask


def check_loss(lp, old, adv, rf, ent, mask, seed=0, **kw):
    import pufferlib_b200 as pb
    lp, ent = lp.detach().requires_grad_(True), None if ent is None else ent.detach().requires_grad_(True)
    loss, ratio, stats = pb.policy_loss(lp, old, adv, ref_logprobs=rf, entropy=ent, mask=mask, **kw)
    leaves = [lp] + ([] if ent is None else [ent])
    grads = torch.autograd.grad(loss, leaves)
    args = dict(clip_low=0.2, clip_high=0.2) | kw
    want = ref.policy_loss(lp.detach(), old, adv, ref=rf, entropy=None if ent is None else ent.detach(), mask=mask, **args)
    within(loss, *want["loss"], "loss")
    within(ratio, *want["ratio"], "ratio")
    within(stats, *want["stats"], "stats")
    within(grads[0], *want["dlogprobs"], "dlogprobs")
    if ent is not None:
        within(grads[1], *want["dentropy"], "dentropy")
    return loss, ratio, stats, grads


SHAPES = [(1, 1), (1, 2), (2, 1), (3, 5), (1, 33), (5, 32), (7, 64), (64, 7), (33, 127), (300, 3), (1000, 1), (1, 4096),
          (2, 5001), (129, 1025), (1024, 64), (10007, 4), (517, 256)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("per_row", [False, True])
def test_policy_loss_shapes(shape, reduction, masked, per_row):
    lp, old, adv, rf, ent, mask = loss_inputs(*shape, seed=shape[0] + shape[1], per_row=per_row, masked=masked)
    check_loss(lp, old, adv, rf, ent, mask, reduction=reduction, kl_coef=0.1, ent_coef=0.02, clip_high=0.3)
    check_loss(lp, old, adv, None, None, mask, reduction=reduction)
    check_loss(lp, old, adv[:, None] if per_row else adv, rf, None, mask, reduction=reduction, kl_coef=0.1, denominator=77.0)


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss_masked_values_are_not_read(reduction):
    lp, old, adv, rf, ent, mask = loss_inputs(37, 50, seed=4, masked=True)
    kw = dict(reduction=reduction, kl_coef=0.1, ent_coef=0.02)
    a = check_loss(lp, old, adv, rf, ent, mask, **kw)
    for poison in (math.nan, math.inf, -math.inf, -3.4e38):
        t = [torch.where(mask, v, poison) for v in (lp, old, adv, rf, ent)]
        b = check_loss(*t, mask, **kw)
        for x, y in zip(a[:3] + tuple(a[3]), b[:3] + tuple(b[3])):
            assert torch.equal(x, y)
    nothing = check_loss(*[torch.full_like(v, math.nan) for v in (lp, old, adv, rf, ent)], torch.zeros_like(mask), **kw)
    assert nothing[0] == 0 and not nothing[2].any() and not nothing[3][0].any() and not nothing[3][1].any()
    assert (nothing[1] == 1).all()


def test_policy_loss_borders_and_extremes():
    """Ratios at the clip borders are decided in 64 bits; advantages of 0; clips of 0 and of more than 1; tiny and large ratios."""
    n = 4001
    steps = torch.arange(n, device="cuda", dtype=torch.float64) - n // 2
    old = torch.full((1, n), -0.7, device="cuda")
    for border in (math.log(1.2), math.log(0.8)):
        lp = (old.double() + border).float() + (steps * 2.0 ** -24).float()[None]
        for sign in (1.0, -1.0, 0.0):
            adv = torch.full((1, n), sign, device="cuda")
            check_loss(lp, old, adv, None, None, None)
    g = gen(9)
    lp, old = randn(g, 3, 400) * 30, randn(g, 3, 400) * 30
    adv = randn(g, 3, 400)
    for low, high in ((0.0, 0.0), (1.0, 5.0), (2.0, 1e9), (0.2, 0.2)):
        check_loss(lp.clamp(-60, 20), old.clamp(-60, 20), adv, None, None, None, clip_low=low, clip_high=high)
    small = randn(g, 3, 400) * 1e-4                       # the KL term without cancellation
    check_loss(small, torch.zeros_like(small), adv, torch.zeros_like(small), None, None, kl_coef=1.0)
    # an action that the new policy cannot take any more
    lp = torch.tensor([[-math.inf, -0.5]], device="cuda")
    check_loss(lp, torch.tensor([[-1.0, -1.0]], device="cuda"), torch.ones(1, 2, device="cuda"), None, None, None)


def test_policy_loss_empty():
    import pufferlib_b200 as pb
    for shape in ((0, 5), (5, 0), (0, 0)):
        z = torch.empty(*shape, device="cuda", requires_grad=True)
        loss, ratio, stats = pb.policy_loss(z, z.detach(), z.detach())
        assert loss == 0 and ratio.shape == shape and not stats.any()
        assert torch.autograd.grad(loss, z)[0].shape == shape


def test_policy_loss_gradient_against_differences():
    import pufferlib_b200 as pb
    lp, old, adv, rf, ent, mask = loss_inputs(9, 20, seed=21, masked=True)
    # away from the clip borders, where the loss has no slope
    ratio = (lp - old).exp()
    mask &= ((ratio - 1.2).abs() > 1e-3) & ((ratio - 0.8).abs() > 1e-3)
    lp, ent = lp.requires_grad_(True), ent.requires_grad_(True)
    for reduction in ("token", "sequence"):
        loss, _, _ = pb.policy_loss(lp, old, adv, ref_logprobs=rf, kl_coef=0.3, entropy=ent, ent_coef=0.1, mask=mask, reduction=reduction)
        grads = torch.autograd.grad(loss * 3.0, [lp, ent])
        g = gen(1)
        v = [randn(g, 9, 20).double(), randn(g, 9, 20).double()]

        def f(s):
            out = ref.policy_loss(lp.detach().double() + s * v[0], old, adv, 0.2, 0.2, rf, 0.3, ent.detach().double() + s * v[1], 0.1, mask, reduction)
            return 3.0 * out["loss"][0]
        slope = (f(1e-5) - f(-1e-5)) / 2e-5
        terms = sum((a.double() * b).abs().sum() for a, b in zip(grads, v))
        assert abs(sum((a.double() * b).sum() for a, b in zip(grads, v)) - slope) <= 1e-6 * terms + 1e-8


def test_policy_loss_same_bits_each_time():
    import pufferlib_b200 as pb
    for shape, masked in (((3000, 70), True), ((70, 3000), False)):
        lp, old, adv, rf, ent, mask = loss_inputs(*shape, seed=1, masked=masked)
        for reduction in ("token", "sequence"):
            first = pb.policy_loss(lp, old, adv, ref_logprobs=rf, mask=mask, reduction=reduction)
            for _ in range(3):
                again = pb.policy_loss(lp, old, adv, ref_logprobs=rf, mask=mask, reduction=reduction)
                assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---- gated recurrence --------------------------------------------------------------------------------------------

def rec_inputs(B, T, C, dtype, seed, resets=0.05, state=True, joint=False):
    g = gen(seed)
    if joint:
        gates, x = (randn(g, B, T, 2 * C) * 1.5).to(dtype).split(C, -1)
    else:
        gates, x = (randn(g, B, T, C) * 1.5 + 0.5).to(dtype), randn(g, B, T, C).to(dtype)
    r = (torch.rand(B, T, device="cuda", generator=g) < resets).float() if resets else None
    s = randn(g, B, C) if state else None
    return gates, x, r, s


def check_recurrence(gates, x, resets, state, seed=0, use=(True, True)):
    import pufferlib_b200 as pb
    g = gen(seed + 500)
    gates, x = gates.detach().requires_grad_(True), x.detach().requires_grad_(True)
    state = None if state is None else state.detach().requires_grad_(True)
    out, final = pb.gated_recurrence(gates, x, resets=resets, state=state)
    dout, dfinal = randn(g, *out.shape).to(out.dtype), randn(g, *final.shape)
    leaves = [gates, x] + ([] if state is None else [state])
    outs = [v for v, u in ((out, use[0]), (final, use[1])) if u]
    grads = torch.autograd.grad(outs, leaves, [v for v, u in ((dout, use[0]), (dfinal, use[1])) if u])
    want = ref.recurrence(gates.detach(), x.detach(), resets, None if state is None else state.detach(),
                          dout if use[0] else None, dfinal if use[1] else None)
    assert out.dtype == x.dtype and final.dtype == F32 and out.is_contiguous() and all(v.is_contiguous() for v in grads)
    within(out, *want["outputs"], "outputs")
    within(final, *want["final"], "final")
    within(grads[0], *want["dgates"], "dgates")
    within(grads[1], *want["dinputs"], "dinputs")
    if state is not None:
        within(grads[2], *want["dstate"], "dstate")
    with torch.no_grad():
        out2, final2 = pb.gated_recurrence(gates, x, resets=resets, state=state)
    assert torch.equal(out2, out.detach()) and torch.equal(final2, final.detach())
    return out, final, grads


@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 2, 3), (2, 15, 8), (3, 16, 16), (2, 17, 33), (1, 31, 64), (4, 32, 130), (2, 33, 31),
                                   (1, 100, 256), (5, 64, 65), (2, 127, 128), (1, 128, 7), (1, 129, 500), (3, 257, 96),
                                   (1, 1000, 32), (1, 2049, 40), (2, 513, 1030), (200, 20, 24), (2, 5003, 2),
                                   # rows of a multiple of 16 bytes: tiles at every edge of steps, channels and rounds
                                   (3, 1, 64), (2, 5, 32), (5, 16, 40), (3, 48, 72), (2, 130, 200), (1, 777, 1024),
                                   (1, 4097, 64), (3, 2100, 96), (700, 33, 64), (70000, 2, 32),
                                   # a few steps: four channels a thread, or one
                                   (5, 7, 33), (4, 8, 36), (9, 8, 130), (2, 9, 36), (3000, 4, 515), (40, 3, 256),
                                   # few lanes over many steps: clusters of two and four, and ranges
                                   (3, 1500, 1024), (6, 1100, 1000), (2, 2100, 640), (1, 2500, 1600)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_recurrence_shapes(shape, dtype):
    check_recurrence(*rec_inputs(*shape, dtype, seed=sum(shape)))
    if shape[1] <= 1000:       # (the reference walks step by step)
        check_recurrence(*rec_inputs(*shape, dtype, seed=sum(shape), resets=0.0, state=False), use=(True, False))


@pytest.mark.parametrize("shape", [(3, 40, 64), (2, 300, 33), (64, 16, 128), (1, 3000, 512), (40, 200, 300),
                                   (300, 6, 36), (50, 8, 31), (2, 1, 1000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_recurrence_strides(shape, dtype):
    """Halves of one projection, time-major tensors, odd offsets: read in place."""
    B, T, C = shape
    check_recurrence(*rec_inputs(B, T, C, dtype, seed=1, joint=True))
    gates, x, r, s = rec_inputs(T, B, C, dtype, seed=2)
    r = r.t().contiguous()
    check_recurrence(gates.transpose(0, 1), x.transpose(0, 1), r, torch.zeros(B, C, device="cuda"))
    gates, x, r, s = rec_inputs(B, T, C + 3, dtype, seed=3)
    check_recurrence(gates[..., 1:1 + C], x[..., 3:], r.bool(), s[:, :C].contiguous(), use=(False, True))
    gates, x, r, s = rec_inputs(B, 1, C, dtype, seed=4)
    check_recurrence(gates.expand(B, T, C), x.expand(B, T, C), None, s)        # the same step again and again


def test_recurrence_resets_cut_everything_off():
    import pufferlib_b200 as pb
    for T in (40, 700):
        gates, x, _, s = rec_inputs(2, T, 64, F32, seed=8, resets=0)
        r = torch.zeros(2, T, device="cuda")
        r[0, 17] = 1.0
        r[1, 0] = 1.0
        x2, s2 = x.clone(), s.clone()
        x2[0, 5] = math.nan
        x2[0, 9] = math.inf
        s2[1] = math.nan
        out, final = pb.gated_recurrence(gates, x, resets=r, state=s)
        out2, final2 = pb.gated_recurrence(gates, x2, resets=r, state=s2)
        assert torch.equal(out[0, 17:], out2[0, 17:]) and torch.equal(out[1], out2[1]) and torch.equal(final, final2)
        assert out2[0, 9:17].isnan().all() and torch.equal(out[0, :5], out2[0, :5])
        # a gradient does not cross a reset
        leaf = x.detach().requires_grad_(True)
        o, f = pb.gated_recurrence(gates, leaf, resets=r, state=s)
        (d,) = torch.autograd.grad(f.sum(), leaf)
        assert not d[0, :17].any() and d[0, 17:].abs().sum() > 0
    # every step a reset; a fraction counts as one
    gates, x, _, s = rec_inputs(3, 50, 20, F32, seed=9, resets=0)
    check_recurrence(gates, x, torch.full((3, 50), 0.5, device="cuda"), s)


def test_recurrence_extreme_gates():
    gates, x, r, s = rec_inputs(2, 400, 64, F32, seed=10)
    for shift in (-30.0, -200.0, 12.0, 30.0, 200.0):
        check_recurrence(gates + shift, x, r, s)
    gates[0, :, 5] = math.inf                  # hold the state
    gates[0, :, 6] = -math.inf                 # take the input
    out, final, _ = check_recurrence(gates, x, None, s)
    assert (out[0, :, 5] == s[0, 5]).all() and torch.equal(out[0, :, 6], x[0, :, 6])


def test_recurrence_lengths_zero():
    import pufferlib_b200 as pb
    for B, T, C in ((0, 4, 5), (3, 0, 5), (3, 4, 0)):
        gates = torch.zeros(B, T, C, device="cuda", requires_grad=True)
        s = torch.randn(B, C, device="cuda", requires_grad=True)
        out, final = pb.gated_recurrence(gates, gates * 1.0, state=s)
        assert out.shape == (B, T, C) and (T > 0 or torch.equal(final, s))
        g = torch.autograd.grad(final.sum(), [gates, s], allow_unused=True)
        assert g[1].shape == (B, C) and (T > 0 or (g[1] == 1).all())
    out, final = pb.gated_recurrence(torch.zeros(2, 0, 3, device="cuda"), torch.zeros(2, 0, 3, device="cuda"))
    assert not final.any()


def test_recurrence_gradient_against_differences():
    import pufferlib_b200 as pb
    gates, x, r, s = rec_inputs(2, 45, 20, F32, seed=12)
    leaves = [v.requires_grad_(True) for v in (gates, x, s)]
    g = gen(13)
    wo, wf = randn(g, 2, 45, 20), randn(g, 2, 20)
    v = [randn(g, *t.shape).double() for t in leaves]
    out, final = pb.gated_recurrence(gates, x, resets=r, state=s)
    grads = torch.autograd.grad((out * wo).sum() + (final * wf).sum(), leaves)

    def f(e):
        q = ref.recurrence(gates.detach().double() + e * v[0], x.detach().double() + e * v[1], r, s.detach().double() + e * v[2])
        return (q["outputs"][0] * wo.double()).sum() + (q["final"][0] * wf.double()).sum()
    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    terms = sum((a.double() * b).abs().sum() for a, b in zip(grads, v))
    assert abs(sum((a.double() * b).sum() for a, b in zip(grads, v)) - slope) <= 1e-6 * terms


@pytest.mark.parametrize("B,C", [(1, 1), (3, 7), (64, 128), (1000, 33), (4096, 512), (1, 5000)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_recurrence_step(B, C, dtype):
    import pufferlib_b200 as pb
    g = gen(B + C)
    joint = randn(g, B, 2 * C + 1).to(dtype)
    for gates, x in ((joint[:, :C], joint[:, C:2 * C]), (joint[:, 1:C + 1].contiguous(), joint[:, C + 1:].contiguous())):
        state = randn(g, B, C)
        for resets in (None, (torch.rand(B, device="cuda", generator=g) < 0.3).float(), torch.rand(B, device="cuda", generator=g) < 0.3):
            want = ref.recurrence(gates[:, None], x[:, None], None if resets is None else resets[:, None], state)
            out, new = pb.gated_recurrence_step(gates, x, state, resets=resets)
            within(out[:, None], *want["outputs"], "outputs")
            within(new, *want["final"], "state")
            mine = state.clone()                         # in place: the same bits
            out2, same = pb.gated_recurrence_step(gates, x, mine, resets=resets, new_state=mine)
            assert same is mine and torch.equal(mine, new) and torch.equal(out2, out)


def test_steps_and_sequence_agree():
    """Acting step by step and reading the whole segment give one trajectory."""
    import pufferlib_b200 as pb
    gates, x, r, s = rec_inputs(5, 70, 96, F32, seed=15)
    out, final = pb.gated_recurrence(gates, x, resets=r, state=s)
    want = ref.recurrence(gates, x, r, s)
    state = s.clone()
    for t in range(70):
        o, state = pb.gated_recurrence_step(gates[:, t], x[:, t], state, resets=r[:, t].contiguous(), new_state=state)
        value, bound = want["outputs"]
        within(o, value[:, t], bound[:, t], f"step {t}")
    within(state, final.double(), 2 * want["final"][1], "final")


def test_recurrence_beyond_32_bit_offsets():
    """More than 2^31 elements: the last rows are checked."""
    import pufferlib_b200 as pb
    B, T, C = 1030, 2048, 1024
    gates = torch.zeros(B, T, C, device="cuda", dtype=BF16)
    x = torch.zeros(B, T, C, device="cuda", dtype=BF16)
    g = gen(16)
    gates[-1], x[-1] = randn(g, T, C).to(BF16), randn(g, T, C).to(BF16)
    gates.requires_grad_(True), x.requires_grad_(True)
    out, final = pb.gated_recurrence(gates, x)
    dfinal = randn(g, B, C)
    dg, dx = torch.autograd.grad(final, [gates, x], dfinal)
    want = ref.recurrence(gates.detach()[-1:], x.detach()[-1:], None, None, None, dfinal[-1:])
    within(out[-1:], *want["outputs"], "outputs")
    within(dg[-1:], *want["dgates"], "dgates")
    within(dx[-1:], *want["dinputs"], "dinputs")
    assert not out[:-1].any()


# ---- together, streams, graphs -----------------------------------------------------------------------------------

def update(pb, weights, obs, terminals, rewards, values, tokens, old, importance):
    """One policy update the way a trainer writes it: recurrent layer, head, log-probabilities, advantages, loss."""
    w_gate, w_in, head = weights
    h, _ = pb.gated_recurrence(obs @ w_gate, obs @ w_in, resets=terminals)
    logprobs, entropy = pb.action_logprobs(h @ head, tokens)
    advantages = torch.zeros_like(values)
    pb.compute_puff_advantage(values, rewards, terminals, importance, advantages, 0.99, 0.95, 1.0, 1.0)
    loss, ratio, stats = pb.policy_loss(logprobs, old, advantages, entropy=entropy, ent_coef=0.01)
    return loss, ratio, stats, advantages


def update_inputs(S, H, D, C, A, seed):
    g = gen(seed)
    weights = [randn(g, D, C) / D ** 0.5, randn(g, D, C) / D ** 0.5, randn(g, C, A) / C ** 0.5]
    obs = randn(g, S, H, D)
    terminals = (torch.rand(S, H, device="cuda", generator=g) < 0.05).float()
    rewards, values = randn(g, S, H), randn(g, S, H)
    tokens = torch.randint(0, A, (S, H), device="cuda", generator=g)
    old = -torch.rand(S, H, device="cuda", generator=g) - math.log(A) + 0.5
    return [w.requires_grad_(True) for w in weights], (obs, terminals, rewards, values, tokens, old, torch.ones(S, H, device="cuda"))


def test_the_whole_update_against_64_bits():
    import pufferlib_b200 as pb
    weights, data = update_inputs(24, 30, 12, 40, 9, seed=17)
    loss, ratio, _, advantages = update(pb, weights, *data)
    grads = torch.autograd.grad(loss, weights)
    obs, terminals, _, _, tokens, old, _ = data
    wide = [w.detach().double().requires_grad_(True) for w in weights]
    f, x = torch.sigmoid(obs.double() @ wide[0]), obs.double() @ wide[1]
    h, hs = torch.zeros(24, 40, device="cuda", dtype=torch.float64), []
    for t in range(30):
        h = f[:, t] * (1 - terminals[:, t, None]) * h + (1 - f[:, t]) * x[:, t]
        hs.append(h)
    logp = torch.log_softmax(torch.stack(hs, 1) @ wide[2], -1)
    lp = logp.gather(-1, tokens[..., None])[..., 0]
    r = (lp - old.double()).exp()
    A = advantages.double()
    want = torch.maximum(-A * r, -A * r.clamp(0.8, 1.2)).mean() + 0.01 * (logp.exp() * logp).sum(-1).mean()
    want_grads = torch.autograd.grad(want, wide)
    # fp32 products over 12 and 40 terms in front of and behind operators good to a few 2^-24: 100 roundings in all
    assert abs(loss.double() - want) <= 100 * ref.U * (A.abs() * r).mean()
    for a, b in zip(grads, want_grads):
        assert (a.double() - b).norm() <= 300 * ref.U * b.norm() + 1e-9
    within(ratio, r.detach(), 200 * ref.U * r.detach(), "ratio")


def test_the_whole_update_captured_and_replayed():
    """Captured once, replayed on other inputs; two graphs with a pool each.  An eager graph of the same weights lives on
    meanwhile: autograd ties a leaf's node to the stream it was made on, so the capture takes leaves of its own over
    the same memory."""
    import pufferlib_b200 as pb
    weights, data = update_inputs(32, 48, 16, 64, 40, seed=18)
    _, other = update_inputs(32, 48, 16, 64, 40, seed=19)

    def run(d):
        leaves = [w.detach().requires_grad_(True) for w in weights]
        loss, ratio, stats, _ = update(pb, leaves, *d)
        return (loss.detach(), ratio, stats) + torch.autograd.grad(loss, leaves)
    eager_loss = update(pb, weights, *data)[0]           # its graph stays alive over the capture
    want, want_other = run(data), run(other)
    buffers = [t.clone() for t in data]
    graphs, results = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(buffers)
    torch.cuda.current_stream().wait_stream(side)
    for graph in graphs:
        with torch.cuda.graph(graph):
            results.append(run(buffers))
    for inputs, expected in ((data, want), (other, want_other), (data, want)):
        for b, t in zip(buffers, inputs):
            b.copy_(t)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in results:
            for a, b in zip(got, expected):
                assert torch.equal(a, b)
    torch.autograd.grad(eager_loss, weights)


def test_operators_on_side_streams():
    import pufferlib_b200 as pb
    weights, data = update_inputs(32, 48, 16, 64, 40, seed=20)
    want = update(pb, weights, *data)[0].detach()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(5):
                got.append(update(pb, weights, *data)[0].detach())
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got)


def test_no_wait_has_given_up():
    """The bounded waits of the kernels above all ended with their data."""
    from pufferlib_b200 import cabi
    check_recurrence(*rec_inputs(3, 300, 64, BF16, seed=30))
    assert cabi.device_status() == 0


def test_second_derivatives_are_refused():
    import pufferlib_b200 as pb
    z = torch.randn(4, 9, device="cuda", requires_grad=True)
    lp, H = pb.action_logprobs(z, torch.zeros(4, dtype=torch.int64, device="cuda"))
    (d,) = torch.autograd.grad(lp.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_launches_are_this_librarys():
    from pufferlib_b200 import cabi
    import pufferlib_b200 as pb
    before = cabi.launch_count()
    z = torch.randn(4, 9, device="cuda", requires_grad=True)
    lp, H = pb.action_logprobs(z, torch.zeros(4, dtype=torch.int64, device="cuda"))
    torch.autograd.grad(lp.sum(), z)
    assert cabi.launch_count() >= before + 2
