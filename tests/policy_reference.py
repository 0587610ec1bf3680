"""The policy-update operators in 64 bits, from their formulas, with bounds on what fp32 evaluation may add.

Every bound counts roundings: u = 2^-24 is half a step of fp32 relative to the value, `half_step(dtype)` half a step of
the output's type.  ex2.approx is good to 2^-22 = 4 u, expf and logf to 2 u.
"""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(value, dtype):
    """Half a step of `dtype` at `value`: relative, and for subnormal results absolute."""
    return half_step(dtype) * value.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, want, bound, what=""):
    got, want = got.double().cpu(), want.double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= bound))
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {i}: got {got[i].item()!r} "
                             f"want {want[i].item()!r} bound {bound[i].item():.3g}")


# ---- log-probabilities -------------------------------------------------------------------------------------------

def logprobs(logits, actions, temperature, dlogprobs=None, dentropy=None, chain=None):
    """dict of (value, bound) for logprobs, entropy and, where gradients are given, dlogits."""
    T = float(torch.tensor(temperature, dtype=torch.float32))
    V = logits.shape[-1]
    z = logits.double() / T
    m = z.amax(-1, keepdim=True)
    empty = (m == -math.inf)[..., 0]
    d = z - torch.where(m == -math.inf, 0.0, m)
    e = d.exp()
    s = e.sum(-1, keepdim=True)
    logp = d - s.log()
    p = e / s
    weighted = torch.where(e > 0, p * d, 0.0)
    H = (s.log()[..., 0] - weighted.sum(-1))
    pad = (actions < 0) | (actions >= V)
    taken = actions.clamp(0, V - 1)[..., None]
    lp = logp.gather(-1, taken)[..., 0]
    zero = pad | empty
    # a sum of positive terms in a chain of adds: one u each; every e: 4 u from ex2 and three roundings of its argument
    adds = (V / 8 if chain is None else chain) + 40
    s_err = U * (adds + 4) + 3 * U * weighted.abs().sum(-1)
    lp_err = s_err + 4 * U * (d.gather(-1, taken)[..., 0].abs() + s.log()[..., 0].abs()) + 2 * U
    lp_err = lp_err.nan_to_num(0.0, 0.0, 0.0)
    second = torch.where(e > 0, p * d * d, 0.0).sum(-1)
    H_err = s_err + 4 * U * s.log()[..., 0].abs() + (adds + 8) * U * weighted.abs().sum(-1) + 3 * U * second + 2 * U
    out = {"logprobs": (torch.where(pad, 0.0, torch.where(empty, -math.inf, lp)), lp_err),
           "entropy": (torch.where(zero, 0.0, H), H_err)}
    if dlogprobs is not None:
        up = dlogprobs.double()[..., None]
        g = -up * p
        size = up.abs() * p
        logp_err = lp_err_all = (s_err[..., None] + 4 * U * (d.abs() + s.log().abs()) + 2 * U).nan_to_num(0.0, 0.0, 0.0)
        rel = logp_err + 5 * U + 2 * U * torch.where(p > 0, logp.abs(), 0.0)
        err = size * rel
        if dentropy is not None:
            dh = dentropy.double()[..., None]
            inner = torch.where(p > 0, logp, 0.0) + H[..., None]
            g = g - dh * torch.where(p > 0, p * inner, 0.0)
            err = err + dh.abs() * p * (inner.abs() * (rel + 4 * U) + lp_err_all + H_err[..., None] + 2 * U * (torch.where(p > 0, logp.abs(), 0.0) + H[..., None].abs()))
        g = g.scatter_add(-1, taken, up)
        err = err + 2 * U * (g.abs() + size)
        g, err = g / T, err / T + 3 * U * g.abs() / T
        keep = ~zero[..., None]
        g = torch.where(keep, g, 0.0)
        # p below the smallest normal, 2^-126, comes out as 0: the gradient then misses up to 2^-126 (|dlp| + |dh| |log p + H|)
        # / T, with |log p| up to 104 (where p is below the smallest subnormal too)
        flushed = up.abs() + (0.0 if dentropy is None else dentropy.double()[..., None].abs() * (104 + H[..., None].abs()))
        err = err + 2.0 ** -126 * flushed / T
        err = torch.where(keep, err, 0.0) * (1 + half_step(logits.dtype)) + rounding(g, logits.dtype) + 2.0 ** -120
        out["dlogits"] = (g, err)
    return out


# ---- policy loss -------------------------------------------------------------------------------------------------

def policy_loss(logprobs, old, advantages, clip_low, clip_high, ref=None, kl_coef=0.0, entropy=None, ent_coef=0.0,
                mask=None, reduction="token", denominator=None):
    """dict of (value, bound): loss, ratio, stats, and the gradients dlogprobs, dentropy for dloss = 1."""
    lp, old = logprobs.double(), old.double()
    adv = (advantages.double() if advantages.dim() == 2 else advantages.double()[:, None]).expand_as(lp)
    keep = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask
    d = torch.where(keep, lp - old, 0.0)
    ratio = d.exp()
    low, high = 1.0 - clip_low, 1.0 + clip_high
    above, below = ratio > high, ratio < low
    cut = (above & (adv > 0)) | (below & (adv < 0))
    held = torch.where(above, high, torch.where(below, low, ratio))
    policy = torch.where(cut, -adv * held, -adv * ratio)
    slope = torch.where(cut, 0.0, -adv * ratio)
    slope_err = slope.abs() * 6 * U
    kl = torch.zeros_like(lp)
    if ref is not None:
        q = torch.where(keep, ref.double() - lp, 0.0)
        # the cancelled value, from the series where e^q - 1 - q has lost it
        kl = torch.where(q.abs() < 1e-3, q * q * (0.5 + q / 6 + q * q / 24), torch.expm1(q) - q)
        slope = slope - kl_coef * torch.expm1(q)
        slope_err = slope_err + kl_coef * (torch.expm1(q).abs() + q.exp()) * 6 * U + 2 * U * slope.abs()
    zero = torch.zeros_like(lp)
    ent = zero if entropy is None else entropy.double()
    pick = lambda v: torch.where(keep, v, zero)  # noqa: E731
    n = keep.sum().double()
    length = keep.sum(1, keepdim=True).double()
    if reduction == "token":
        w = keep / (n.clamp(min=1) if denominator is None else denominator)
    else:
        w = keep / (length.clamp(min=1) * ((length > 0).sum().clamp(min=1) if denominator is None else denominator))
    mean = lambda v: (pick(v) * w).sum()  # noqa: E731
    tokens = lambda v: pick(v).sum() / n.clamp(min=1)  # noqa: E731
    excess = torch.where(d.abs() < 1e-3, d * d * (0.5 + d / 6 + d * d / 24), torch.expm1(d) - d)
    clipped = (above | below).double()
    values = [mean(policy), mean(kl), mean(ent), tokens(-d), tokens(excess), tokens(clipped)]
    # sums are 64-bit; every token term has at most 8 roundings, k3 beyond |q| = 1 up to 8 u of e^q
    bounds = [mean(policy.abs()) * 8 * U, mean(kl + kl * 0 if ref is None else kl.abs() + pick(torch.where(q.abs() >= 1, q.exp() + 1, zero))) * 8 * U,
              mean(ent.abs()) * 2 * U, tokens(d.abs()) * 4 * U,
              tokens(excess.abs() + torch.where(d.abs() >= 1, ratio + 1, zero)) * 8 * U, tokens(clipped) * 2 * U]
    loss = values[0] + kl_coef * values[1] - ent_coef * values[2]
    out = {"loss": (loss, bounds[0] + kl_coef * (bounds[1] + 2 * U * values[1].abs()) + abs(ent_coef) * (bounds[2] + 2 * U * values[2].abs()) + 2 * U * loss.abs()),
           "ratio": (torch.where(keep, ratio, 1.0), ratio * 4 * U),
           "stats": (torch.stack(values), torch.stack(bounds) + 2 * U * torch.stack(values).abs())}
    g = pick(slope) * w
    out["dlogprobs"] = (g, pick(slope_err) * w + 6 * U * g.abs() + 2.0 ** -140)
    h = -ent_coef * w
    out["dentropy"] = (h, 6 * U * h.abs() + 2.0 ** -140)
    return out


# ---- gated recurrence --------------------------------------------------------------------------------------------

def recurrence(gates, inputs, resets=None, state=None, doutputs=None, dfinal=None):
    """dict of (value, bound) for outputs, final and, with doutputs/dfinal, dgates, dinputs, dstate."""
    x, g = inputs.double(), gates.double()
    B, T, C = x.shape
    f, n = torch.sigmoid(g), torch.sigmoid(-g)
    cut = torch.zeros(B, T, dtype=torch.bool, device=x.device) if resets is None else resets != 0
    a = torch.where(cut[..., None], 0.0, f)
    # relative error of the smaller gate: ex2 4 u, its argument 3 roundings of |g|, a quotient and a sum 4 u
    # (beyond |g| = 104 the smaller gate is below the smallest subnormal: its relative error counts no more)
    gate = U * (3 * g.abs().clamp(max=110) + 10)
    h = torch.zeros(B, C, dtype=torch.float64, device=x.device) if state is None else state.double()
    E = torch.zeros_like(h)
    hs, Es, before, Eb = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    for t in range(T):
        c = cut[:, t, None]
        prev, Ep = torch.where(c, 0.0, h), torch.where(c, 0.0, E)
        before[:, t], Eb[:, t] = prev, Ep
        h = torch.where(c, 0.0, f[:, t] * prev) + n[:, t] * x[:, t]
        # 4 roundings of each term; products of gains joined over a span carry one more per step, counted here too
        E = a[:, t] * Ep + gate[:, t] * n[:, t] * f[:, t].clamp(min=0.5) * 2 * (prev.abs() + x[:, t].abs()) \
            + 6 * U * (f[:, t] * prev.abs() + n[:, t] * x[:, t].abs()) + 2.0 ** -126
        hs[:, t], Es[:, t] = h, E
    out = {"outputs": (hs, Es + rounding(hs, inputs.dtype)), "final": (h, E + 2 * U * h.abs())}
    if doutputs is None and dfinal is None:
        return out
    lam = torch.zeros_like(h) if dfinal is None else dfinal.double()
    EL = torch.zeros_like(h)
    dg, dx, Eg, Ex = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    for t in range(T - 1, -1, -1):
        if doutputs is not None:
            lam = lam + doutputs[:, t].double()
            EL = EL + 2 * U * (lam.abs() + doutputs[:, t].double().abs())
        dx[:, t] = lam * n[:, t]
        Ex[:, t] = EL * n[:, t] + dx[:, t].abs() * (gate[:, t] + 2 * U)
        diff = before[:, t] - x[:, t]
        dg[:, t] = lam * f[:, t] * n[:, t] * diff
        Eg[:, t] = (EL * n[:, t] * diff.abs() + lam.abs() * n[:, t] * (Eb[:, t] + 2 * U * (before[:, t].abs() + x[:, t].abs()))) * f[:, t] \
            + dg[:, t].abs() * (2 * gate[:, t] + 6 * U)
        EL = a[:, t] * EL + a[:, t] * lam.abs() * (2 * gate[:, t] * n[:, t] + gate[:, t] * (f[:, t] < 0.5) + 6 * U) + 2.0 ** -126
        lam = a[:, t] * lam
    out["dgates"] = (dg, Eg * (1 + 2 ** -8) + rounding(dg, gates.dtype) + 2.0 ** -120)
    out["dinputs"] = (dx, Ex * (1 + 2 ** -8) + rounding(dx, inputs.dtype) + 2.0 ** -120)
    out["dstate"] = (lam, EL + 2 * U * lam.abs())
    return out
