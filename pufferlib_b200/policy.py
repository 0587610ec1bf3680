"""The policy update on top of the advantages: log-probabilities, clipped loss, gated recurrence.

What the reference's trainer computes with torch between the policy's outputs
and `loss.backward()` (pufferl.py:385-422; sample_logits of
pufferlib/pytorch.py), as differentiable operators over the experience buffers'
`[segments, horizon]` layout.  Like the advantage ops they run on an sm_100 GPU
only, on the current stream of the tensors' device, and raise when the extension
is missing.  Reverse-mode gradients only: second derivatives and forward mode
raise.  Activation checkpointing and ahead-of-time tracing (torch.compile, sizes
that change included) take them as any other operator.
"""
import contextlib

import torch

from .advantage import _ops as _load_ops

_loaded = None


def _ops():
    """torch.ops.pufferlib, looked up once: these calls are made for every generated token."""
    global _loaded
    if _loaded is None:
        _loaded = _load_ops()
    return _loaded


def action_logprobs(logits, actions, temperature=1.0, entropy=True):
    """(logprobs, entropy) of `actions` under softmax(logits / temperature).

    `logits` is [..., vocab] in float32, float16 or bfloat16, `actions` int64 [...]; both results are float32 [...]
    (entropy is None when `entropy` is false).  Slices of a larger tensor are read in place as long as a row's logits
    are adjacent and its rows lie in at most two strided runs (`logits[:, :-1]`).  A logit of -inf is an action that
    cannot be taken; a row with no other has log-probability -inf, entropy 0 and no gradient.  An action below 0 marks
    padding: zeros, no gradient, whatever the logits hold.  An action beyond the vocabulary gives zeros too and raises
    the flag that `bad_action()` reads."""
    logprobs, ent = _ops().puff_action_logprobs(logits, actions, temperature, entropy)
    return logprobs, ent if entropy else None


def bad_action(device=None):
    """Whether `action_logprobs` on `device` (default: the current one) has met an action beyond the vocabulary since
    the last call for it.  Synchronises that device; an error of CUDA raises."""
    from . import cabi
    with contextlib.nullcontext() if device is None else torch.cuda.device(device):
        code = cabi.load().puff_policy_sm100_bad_action()
    if code < 0:
        cabi.check(code, "puff_policy_sm100_bad_action")
    return code != 0


def policy_loss(logprobs, old_logprobs, advantages, clip_low=0.2, clip_high=0.2, ref_logprobs=None, kl_coef=0.0,
                entropy=None, ent_coef=0.0, mask=None, reduction="token", denominator=None):
    """(loss, ratio, stats) of the clipped policy loss of pufferl.py:390-411 over [rows, steps] tokens:

        loss = mean(max(-A r, -A clip(r, 1 - clip_low, 1 + clip_high)))
               + kl_coef mean(e^q - 1 - q) - ent_coef mean(entropy)

    with r = exp(logprobs - old_logprobs) and q = ref_logprobs - logprobs.  All tensors are contiguous float32
    [rows, steps]; `advantages` may be [rows] or [rows, 1], one for all tokens of a row; `mask` is bool, False where a
    token is not part of the loss (whatever stands there is not read into any result).  `reduction` "token" takes the
    mean over all unmasked tokens, "sequence" over the rows that have one of the row's own mean.  `denominator`
    replaces the number of tokens (or rows) of that mean: pass the count over all micro-batches or ranks of one update.

    Gradients flow to `logprobs` and `entropy`.  `ratio` is r, 1 where masked, for the trainer's importance buffer
    (pufferl.py:394).  `stats` holds the means of policy term, KL and entropy as they enter the loss, and over the
    unmasked tokens old_approx_kl, approx_kl and clipfrac (pufferl.py:396-398)."""
    if denominator is not None and not denominator > 0:
        raise ValueError("denominator must be positive")
    if kl_coef != 0.0 and ref_logprobs is None:
        raise ValueError("kl_coef needs ref_logprobs")
    if ent_coef != 0.0 and entropy is None:
        raise ValueError("ent_coef needs entropy")
    return _ops().puff_policy_loss(logprobs, old_logprobs, advantages, clip_low, clip_high, ref_logprobs, kl_coef,
                                   entropy, ent_coef, mask, reduction, 0.0 if denominator is None else denominator)


def gated_recurrence(gates, inputs, resets=None, state=None):
    """(outputs, final_state) of h_t = f_t h_{t-1} + (1 - f_t) inputs_t, f = sigmoid(gates), over [batch, steps, channels].

    `gates` and `inputs` share a type (float32, float16, bfloat16) and may be strided as long as channels are adjacent
    (the halves of one projection).  `resets` [batch, steps], float32 (the `terminals` buffer) or bool: where it is not
    0 the state from before is cut off.  `state` is float32 [batch, channels] (zeros when omitted), `final_state`
    likewise; `outputs` has the inputs' type.  Gradients flow to gates, inputs and state."""
    return _ops().puff_gated_recurrence(gates, inputs, resets, state)


def gated_recurrence_step(gates, inputs, state, resets=None, new_state=None):
    """(outputs, new_state) of one step for every row: gates, inputs [batch, channels], state float32, resets [batch].

    `new_state` receives the state; pass `state` itself to update it in place.  For acting: no gradient."""
    if new_state is None:
        new_state = torch.empty_like(state)
    return _ops().puff_gated_recurrence_step(gates, inputs, state, resets, new_state), new_state
