"""Timed cases of the policy-update operators: log-probabilities, clipped policy loss, gated recurrence.

`run` makes one pass through an operator.  With `own` false it evaluates the operator's formula with elementary torch
operations in 32 bits (64 where sums are long or a value is next to a clip border) and rounds once at the end; with
`own` true it makes the call that a trainer makes of this package.

    log-probabilities   z = logits / temperature;  lp = z[action] - logsumexp(z);  H = -sum p log p;
                        dlogits = (dlp (onehot - p) - dH p (log p + H)) / temperature; an action < 0 is padding
    policy loss         r = exp(lp - old);  L = mean(max(-A r, -A clip(r))) + kl_coef mean(e^d - 1 - d), d = ref - lp,
                        - ent_coef mean(H); means over the unmasked tokens, or over sequences of their token means
    gated recurrence    f = sigmoid(gates);  h_t = f_t [not reset_t] h_{t-1} + (1 - f_t) x_t
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def _logprobs(name, rows, vocab, dtype, grad=True, entropy=True, pad=0.0, illegal=0.0, temperature=1.0, split=0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "grad": grad,
            "entropy": entropy, "pad": pad, "illegal": illegal, "temperature": temperature, "split": split}


def _loss(name, rows, steps, grad=True, masked=False, reduction="token", kl=0.0, ent=0.0, per_row=False):
    return {"name": name, "op": "loss", "rows": rows, "steps": steps, "grad": grad, "masked": masked,
            "reduction": reduction, "kl": kl, "ent": ent, "per_row": per_row}


def _recurrence(name, batch, steps, channels, dtype, grad=True, resets=0.01, state=True, joint=False):
    return {"name": name, "op": "recurrence", "batch": batch, "steps": steps, "channels": channels, "dtype": dtype,
            "grad": grad, "resets": resets, "state": state, "joint": joint}


def _step(name, batch, channels, dtype):
    return {"name": name, "op": "step", "batch": batch, "channels": channels, "dtype": dtype, "resets": 0.01}


def listed():
    return [
        # action heads of a minibatch of 8192 segments of 64 steps, a few of the 18 actions illegal, training
        _logprobs("actions 524288x18", 8192 * 64, 18, "fp32", illegal=0.2),
        # the log-probability of one sampled token for each of eight sequences that are being generated
        _logprobs("sampled 8x131072", 8, 131072, "bf16", grad=False, entropy=False, temperature=0.7),
        # a training microbatch of tokens over a large vocabulary
        _logprobs("tokens 4096x131072", 4096, 131072, "bf16"),
        # padded sequences, predictions taken from all positions but the last, an odd vocabulary
        _logprobs("tokens odd 2040x50001", 2040, 50001, "fp16", pad=0.15, split=8),
        # the smallest buffer of the advantage benchmark: launches count
        _loss("loss 1024x64", 1024, 64, ent=0.01),
        # the loss read without training on it (early stopping by its KL, logging)
        _loss("loss read 8192x64", 8192, 64, grad=False, kl=0.05),
        # ragged responses with one advantage each, mean over sequences, a reference policy
        _loss("loss ragged 10007x127", 10007, 127, masked=True, reduction="sequence", kl=0.05, per_row=True),
        # the largest buffer of the advantage benchmark
        _loss("loss 131072x256", 131072, 256, masked=True, kl=0.02, ent=0.01),
        # one environment step of a rollout, or one generated token for each sequence
        _step("step 4096x512", 4096, 512, "bf16"),
        # training on 8192 segments of 64 steps, both inputs halves of one projection
        _recurrence("recurrence 8192x64x128", 8192, 64, 128, "bf16", joint=True),
        # training on few long segments
        _recurrence("recurrence 256x4096x128", 256, 4096, 128, "fp32", resets=0.001),
        # reading one long sequence in before generating, an odd width
        _recurrence("recurrence read 1x50001x515", 1, 50001, 515, "bf16", grad=False, resets=0.0, state=False),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["logprobs", "loss", "recurrence", "recurrence", "logprobs", "loss", "step"])
    if kind == "logprobs":
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        vocab = _spread(rng, 2, 160000)
        rows = _spread(rng, 1, max(1, min(600000, (1 << 30) // (vocab * SIZE[dtype]))))
        grad, split = rng.random() < 0.7, rng.choice([0, 0, 4]) if rows >= 16 else 0
        rows -= rows % split if split else 0
        return _logprobs(None, rows, vocab, dtype, grad=grad, entropy=rng.random() < 0.7,
                         pad=rng.choice([0.0, 0.1]), illegal=0.2 if vocab < 512 and rng.random() < 0.5 else 0.0,
                         temperature=rng.choice([1.0, 0.7, 1.3]), split=split)
    if kind == "loss":
        steps = _spread(rng, 1, 4096)
        rows = _spread(rng, 1, max(1, (1 << 25) // steps))
        return _loss(None, rows, steps, grad=rng.random() < 0.8, masked=rng.random() < 0.7,
                     reduction=rng.choice(["token", "sequence"]), kl=rng.choice([0.0, 0.05]),
                     ent=rng.choice([0.0, 0.01]), per_row=rng.random() < 0.4)
    if kind == "step":
        return _step(None, _spread(rng, 1, 16384), _spread(rng, 1, 2048), rng.choice(["fp32", "bf16", "fp16"]))
    dtype, steps, channels = rng.choice(["fp32", "bf16", "fp16"]), _spread(rng, 1, 65536), _spread(rng, 8, 2048)
    batch = _spread(rng, 1, max(1, min(16384, (1 << 27) // (steps * channels))))
    return _recurrence(None, batch, steps, channels, dtype, grad=rng.random() < 0.7, resets=rng.choice([0.0, 0.01]),
                       state=rng.random() < 0.7, joint=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------------------------

def _lead(case):
    """Leading sizes of the logits: [rows], or [split, rows / split] taken from one position more per sequence."""
    return [case["rows"]] if not case["split"] else [case["split"], case["rows"] // case["split"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    s = {"case": case}
    if case["op"] == "logprobs":
        lead, vocab = _lead(case), case["vocab"]
        full = lead if len(lead) == 1 else [lead[0], lead[1] + 1]
        logits = randn(*full, vocab).mul_(2.5)
        if case["illegal"]:
            legal = rand(*full, vocab) >= case["illegal"]
            legal[..., 0] = True
            logits.masked_fill_(~legal, -math.inf)
        logits = logits.to(TYPES[case["dtype"]])
        if len(lead) == 2:
            logits = logits[:, :-1]
        # actions drawn from the softmax itself: the largest of logits + Gumbel noise
        noise = rand(*lead, vocab).clamp_(min=1e-20).log_().neg_().log_().neg_()
        actions = noise.add_(logits).argmax(-1)
        del noise
        if case["pad"]:
            actions = torch.where(rand(*lead) < case["pad"], torch.full_like(actions, -1), actions)
        s |= {"logits": logits.detach().requires_grad_(case["grad"]), "actions": actions}
        if case["grad"]:
            s |= {"dlogprobs": randn(*lead), "dentropy": randn(*lead) * 0.1}
    elif case["op"] == "loss":
        shape = (case["rows"], case["steps"])
        logprobs = randn(*shape).sub_(1.0).abs_().neg_()
        s["old"] = logprobs + 0.15 * randn(*shape)
        s["ref"] = logprobs + 0.3 * randn(*shape) if case["kl"] else None
        s["advantages"] = randn(case["rows"], 1) if case["per_row"] else randn(*shape)
        s["entropy"] = rand(*shape).mul_(2.0).requires_grad_(case["grad"]) if case["ent"] else None
        s["mask"] = None
        if case["masked"]:
            length = (rand(case["rows"], 1) * (case["steps"] + 1)).long()
            s["mask"] = torch.arange(case["steps"], device="cuda")[None] < length
            logprobs.masked_fill_(~s["mask"], 0.0)
        s["logprobs"] = logprobs.requires_grad_(case["grad"])
    else:
        lead = (case["batch"],) if case["op"] == "step" else (case["batch"], case["steps"])
        C, t = case["channels"], TYPES[case["dtype"]]
        if case.get("joint"):
            gates, inputs = randn(*lead, 2 * C).to(t).split(C, -1)
        else:
            gates, inputs = randn(*lead, C).to(t), randn(*lead, C).to(t)
        s["resets"] = (rand(*lead) < case["resets"]).float() if case["resets"] else None
        s["state"] = randn(case["batch"], C) if case["op"] == "step" or case["state"] else None
        s["gates"], s["inputs"] = gates.add(1.0) if not case.get("joint") else gates, inputs
        if case.get("grad"):
            s["gates"] = s["gates"].detach().requires_grad_(True)
            s["inputs"] = inputs.detach().requires_grad_(True)
            if s["state"] is not None:
                s["state"].requires_grad_(True)
            s["doutputs"], s["dfinal"] = randn(*lead, C).to(t), randn(case["batch"], C)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------

def _plain_logprobs(s):
    case, logits, actions = s["case"], s["logits"].detach(), s["actions"]
    d = logits.float() / case["temperature"]
    d = d - d.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    valid = actions >= 0
    taken = actions.clamp(min=0)[..., None]
    out = {"logprobs": torch.where(valid, (d.gather(-1, taken) - total.log())[..., 0], 0.0)}
    H = total.log() - torch.where(e > 0, d * e, 0.0).sum(-1, keepdim=True) / total
    if case["entropy"]:
        out["entropy"] = torch.where(valid, H[..., 0], 0.0)
    if case["grad"]:
        p, dlp = e / total, s["dlogprobs"][..., None]
        dz = -dlp * p
        if case["entropy"]:
            dz = dz - s["dentropy"][..., None] * torch.where(p > 0, p * (d - total.log() + H), 0.0)
        dz = dz.scatter_add(-1, taken, dlp) / case["temperature"]
        out["dlogits"] = torch.where(valid[..., None], dz, 0.0).to(logits.dtype)
    return out


#: clip range, as a trainer sets it: symmetric, or with a higher upper end
CLIP = (0.2, 0.28)


def _plain_loss(s):
    case, mask = s["case"], s["mask"]
    lp, old, adv = s["logprobs"].detach(), s["old"], s["advantages"].expand_as(s["old"])
    keep = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask
    logratio = torch.where(keep, lp - old, 0.0)
    ratio = logratio.exp()
    exact_ratio = (lp.double() - old.double()).exp()      # which side of a border a ratio is on
    above, below = exact_ratio > 1 + CLIP[1], exact_ratio < 1 - CLIP[0]
    held = torch.where(above, 1 + CLIP[1], torch.where(below, 1 - CLIP[0], ratio))
    pg = torch.maximum(-adv * ratio, -adv * held)
    cut = (above & (adv > 0)) | (below & (adv < 0))
    slope = torch.where(cut, 0.0, -adv * ratio)
    count = keep.sum()
    if case["reduction"] == "token":
        weight = keep / count.clamp(min=1).double()
    else:
        length = keep.sum(1, keepdim=True)
        weight = keep / (length.clamp(min=1).double() * (length > 0).sum().clamp(min=1))
    mean = lambda v: torch.where(keep, v, 0.0).double().mul(weight).sum()  # noqa: E731
    tokens = lambda v: torch.where(keep, v, 0.0).double().sum() / count.clamp(min=1)  # noqa: E731
    zero = torch.zeros((), device=lp.device, dtype=torch.float64)
    kl = entropy = zero
    if case["kl"]:
        d = torch.where(keep, s["ref"] - lp, 0.0).double()      # e^d - 1 - d cancels for small d
        kl = mean(torch.expm1(d) - d)
        slope = slope - case["kl"] * torch.expm1(d).float()
    if case["ent"]:
        entropy = mean(s["entropy"].detach())
    policy = mean(pg)
    lr = logratio.double()
    out = {"loss": (policy + case["kl"] * kl - case["ent"] * entropy).float(), "ratio": ratio,
           "stats": torch.stack([policy, kl, entropy, tokens(-lr), tokens(torch.expm1(lr) - lr),
                                 tokens((above | below).double())]).float()}
    if case["grad"]:
        out["dlogprobs"] = torch.where(keep, slope * weight, 0.0).float()
        if case["ent"]:
            out["dentropy"] = (-case["ent"] * weight).float()
    return out


def _plain_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, by doubling: each pass joins spans of twice the length."""
    span = 1
    while span < b.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _plain_recurrence(s):
    case, gates, x = s["case"], s["gates"].detach().float(), s["inputs"].detach().float()
    B, T, C = gates.shape
    f = 1 / (1 + (-gates).exp())
    g = 1 / (1 + gates.exp())
    a = f if s["resets"] is None else torch.where(s["resets"][..., None] != 0, 0.0, f)
    h0 = torch.zeros(B, C, device=x.device) if s["state"] is None else s["state"].detach()
    b = g * x
    h = _plain_scan(a, torch.cat([b[:, :1] + a[:, :1] * h0[:, None], b[:, 1:]], 1))
    out = {"outputs": h.to(s["inputs"].dtype), "final": h[:, -1].clone()}
    if case["grad"]:
        before = torch.cat([h0[:, None], h[:, :-1]], 1)
        dh = s["doutputs"].float()
        dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dfinal"][:, None]], 1)
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        lam = _plain_scan(after.flip(1), dh.flip(1)).flip(1)
        kept = before if s["resets"] is None else torch.where(s["resets"][..., None] != 0, 0.0, before)
        out["dgates"] = (lam * f * g * (kept - x)).to(s["gates"].dtype)
        out["dinputs"] = (lam * g).to(s["inputs"].dtype)
        if s["state"] is not None:
            out["dstate"] = a[:, 0] * lam[:, 0]
    return out


def _plain_step(s):
    gates, x, h = s["gates"].float(), s["inputs"].float(), s["state"]
    if s["resets"] is not None:
        h = torch.where(s["resets"][:, None] != 0, 0.0, h)
    h = h / (1 + (-gates).exp()) + x / (1 + gates.exp())
    return {"outputs": h.to(s["inputs"].dtype), "state": h}


# ---- the package's calls -----------------------------------------------------------------------------------------

def _own(s):
    import pufferlib_b200 as pb
    case = s["case"]
    if case["op"] == "logprobs":
        logprobs, entropy = pb.action_logprobs(s["logits"], s["actions"], temperature=case["temperature"],
                                               entropy=case["entropy"])
        out = {"logprobs": logprobs} | ({"entropy": entropy} if case["entropy"] else {})
        if case["grad"]:
            outs, douts = ([logprobs, entropy], [s["dlogprobs"], s["dentropy"]]) if case["entropy"] else \
                ([logprobs], [s["dlogprobs"]])
            out["dlogits"] = torch.autograd.grad(outs, s["logits"], douts)[0]
        return out
    if case["op"] == "loss":
        loss, ratio, stats = pb.policy_loss(s["logprobs"], s["old"], s["advantages"], clip_low=CLIP[0],
                                            clip_high=CLIP[1], ref_logprobs=s["ref"], kl_coef=case["kl"],
                                            entropy=s["entropy"], ent_coef=case["ent"], mask=s["mask"],
                                            reduction=case["reduction"])
        out = {"loss": loss, "ratio": ratio, "stats": stats}
        if case["grad"]:
            grads = torch.autograd.grad(loss, [s["logprobs"]] + ([s["entropy"]] if case["ent"] else []))
            out |= dict(zip(("dlogprobs", "dentropy"), grads))
        return out
    if case["op"] == "step":
        outputs, state = pb.gated_recurrence_step(s["gates"], s["inputs"], s["state"], resets=s["resets"])
        return {"outputs": outputs, "state": state}
    outputs, final = pb.gated_recurrence(s["gates"], s["inputs"], resets=s["resets"], state=s["state"])
    out = {"outputs": outputs, "final": final}
    if case["grad"]:
        leaves = [s["gates"], s["inputs"]] + ([] if s["state"] is None else [s["state"]])
        grads = torch.autograd.grad([outputs, final], leaves, [s["doutputs"], s["dfinal"]])
        out |= dict(zip(("dgates", "dinputs", "dstate"), grads))
    return out


def run(state):
    if own:
        out = _own(state)
        return {k: v.detach() for k, v in out.items()}
    return {"logprobs": _plain_logprobs, "loss": _plain_loss, "recurrence": _plain_recurrence,
            "step": _plain_step}[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    if case["op"] == "logprobs":
        rows, n = case["rows"], case["rows"] * case["vocab"]
        size, live = SIZE[case["dtype"]], 1 - case["pad"]
        outs = 4 + (4 if case["entropy"] else 0)
        moved = n * size * live + rows * (8 + outs)
        flops = n * live * (7 if case["entropy"] else 4)
        if case["grad"]:
            moved += n * size + rows * outs
            flops += n * live * (7 if case["entropy"] else 4)
        return {"bytes": moved, "flops": flops}
    if case["op"] == "loss":
        rows, n = case["rows"], case["rows"] * case["steps"]
        reads = 8 + (0 if case["per_row"] else 4) + (4 if case["kl"] else 0) + (4 if case["ent"] else 0) + \
            (1 if case["masked"] else 0)
        writes = 4 + ((4 + (4 if case["ent"] else 0)) if case["grad"] else 0)
        return {"bytes": n * (reads + writes) + (4 * rows if case["per_row"] else 0) + 28, "flops": n * 25}
    size, C = SIZE[case["dtype"]], case["channels"]
    lanes = case["batch"] * C
    n = lanes * case.get("steps", 1)
    moved = 3 * size * n + 4 * lanes + (4 * n // C if case["resets"] else 0)
    if case["op"] == "step":
        return {"bytes": moved + 4 * lanes, "flops": 8 * n}
    moved += 4 * lanes if case["state"] else 0
    flops = 8 * n
    if case["grad"]:
        moved += 3 * size * n + 4 * lanes + (4 * lanes if case["state"] else 0)
        flops += 14 * n
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def _exact_logprobs(s):
    case, z, a = s["case"], s["logits"].detach().double() / s["case"]["temperature"], s["actions"]
    logp = z - torch.logsumexp(z, -1, keepdim=True)
    del z
    pad = a < 0
    onehot_at = a.masked_fill(pad, 0).unsqueeze(-1)
    out = {"logprobs": logp.gather(-1, onehot_at).squeeze(-1).masked_fill(pad, 0)}
    p = logp.exp()
    plogp = torch.special.xlogy(p, p)
    H = -plogp.sum(-1)
    if case["entropy"]:
        out["entropy"] = H.masked_fill(pad, 0)
    if case["grad"]:
        up = s["dlogprobs"].double()
        grad = p * -up.unsqueeze(-1)
        grad.scatter_add_(-1, onehot_at, up.unsqueeze(-1))
        if case["entropy"]:
            # d/dz of -sum p log p is -p (log p + H)
            grad -= s["dentropy"].double().unsqueeze(-1) * (plogp + p * H.unsqueeze(-1))
        out["dlogits"] = grad.div_(case["temperature"]).masked_fill_(pad.unsqueeze(-1), 0)
    return out


def _exact_loss(s):
    case = s["case"]
    B, T = s["old"].shape
    lp = s["logprobs"].detach().double().requires_grad_(True)
    leaves = [lp]
    valid = s["mask"] if s["mask"] is not None else lp.new_ones(B, T).bool()
    lr = (lp - s["old"].double()).masked_fill(~valid, 0)
    ratio = lr.exp()
    adv = s["advantages"].double()
    low, high = 1 - CLIP[0], 1 + CLIP[1]
    term = -torch.min(adv * ratio, adv * ratio.clamp(low, high))
    n = valid.sum()
    if case["reduction"] == "token":
        average = lambda v: v.masked_fill(~valid, 0).sum() / max(1, int(n))  # noqa: E731
    else:
        some = valid.any(1)

        def average(v):
            per = v.masked_fill(~valid, 0).sum(1) / valid.sum(1).clamp(min=1)
            return per.sum() / max(1, int(some.sum()))
    policy = average(term)
    kl = entropy = torch.zeros_like(policy)
    if case["kl"]:
        x = (s["ref"].double() - lp).masked_fill(~valid, 0)
        kl = average(x.expm1() - x)
    if case["ent"]:
        ent = s["entropy"].detach().double().requires_grad_(True)
        leaves.append(ent)
        entropy = average(ent)
    loss = policy + case["kl"] * kl - case["ent"] * entropy
    out = {"loss": loss.detach(), "ratio": ratio.detach()}
    with torch.no_grad():
        plain = lambda v: v.masked_fill(~valid, 0).sum() / n.clamp(min=1)  # noqa: E731
        outside = (ratio > high) | (ratio < low)
        out["stats"] = torch.stack([policy, kl, entropy, plain(-lr), plain(lr.expm1() - lr), plain(outside.double())])
    if case["grad"]:
        grads = torch.autograd.grad(loss, leaves)
        out |= dict(zip(("dlogprobs", "dentropy"), grads))
    return out


def _exact_recurrence(s):
    case, x = s["case"], s["inputs"].detach().double()
    f = torch.sigmoid(s["gates"].detach().double())
    if case["op"] == "step":
        h = s["state"].double()
        if s["resets"] is not None:
            h = h * (s["resets"] == 0).double().unsqueeze(-1)
        h = f * h + (1 - f) * x
        return {"outputs": h, "state": h}
    B, T, C = x.shape
    keep = None if s["resets"] is None else (s["resets"] == 0).double()
    h = x.new_zeros(B, C) if s["state"] is None else s["state"].detach().double()
    hs, kept = torch.empty_like(x), torch.empty_like(x) if case["grad"] else None
    gain, new = f, (1 - f) * x
    if keep is not None:
        gain = f * keep.unsqueeze(-1)
    for t in range(T):
        if kept is not None:
            kept[:, t] = h if keep is None else h * keep[:, t, None]
        h = torch.addcmul(new[:, t], gain[:, t], h)
        hs[:, t] = h
    out = {"outputs": hs, "final": h}
    if case["grad"]:
        dh, lam = s["doutputs"].double(), s["dfinal"].double()
        lams = torch.empty_like(x)
        for t in range(T - 1, -1, -1):
            lam = dh[:, t] + lam
            lams[:, t] = lam
            lam = gain[:, t] * lam
        out["dgates"] = lams * f * torch.sigmoid(-s["gates"].detach().double()) * (kept - x)
        out["dinputs"] = lams * (1 - f)
        if s["state"] is not None:
            out["dstate"] = lam
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "loss": _exact_loss}.get(case["op"], _exact_recurrence)(s)
