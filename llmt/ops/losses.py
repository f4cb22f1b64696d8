"""Losses of post-training: token log-probabilities, a clipped policy loss with a KL term, and a
preference loss over pairs of sequences, on logits (B, T, V) or on log-probabilities (B, T).

A token counts where its mask is set (every token without a mask) and its target is an id of the
vocabulary; the logits of the others are not read and get a zero gradient. Without a token that
counts a policy loss is 0 and a sequence's gain is 0.

  logprob_rows           log-probabilities of the targets
  policy_loss_rows       loss, log-probabilities and the gradient of the logits in one call: logits of
  preference_loss_rows   rows up to 64 KB are read once (twice for the pairs, whose slopes need both
                         sums); of longer rows what lies before the last 64 KB a second time, in part from L2
  policy_loss            the same behind autograd; the gradient goes to the logits
  preference_loss
  policy_loss_tokens     the losses on log-probabilities that a fused head gives
  preference_loss_tokens (llmt.models.native.NativeLlama.token_logprobs), behind autograd

old_logp, ref_logp and advantages are constants of the loss (fp32; a tensor that requires a
gradient is refused), and a loss can be differentiated once. Everything else about a loss is an
argument of the call, and the kernels' scratch is allocated per call, so calls on several streams
or in several graphs share nothing. To capture a backward pass into a CUDA graph, drop the results of
eager calls on the same leaves first: autograd adds a leaf's gradient on the stream of the oldest
graph that still holds it, which a capture on another stream does not allow.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from llmt.ops import native as N

REDUCTIONS = {"token": 0, "sequence": 1, "sum": 2}
KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}


class PolicyRows(NamedTuple):
    loss: torch.Tensor
    logp: torch.Tensor
    dlogits: Optional[torch.Tensor]


class PreferenceRows(NamedTuple):
    loss: torch.Tensor
    logp: torch.Tensor
    rewards: torch.Tensor
    dlogits: Optional[torch.Tensor]


class PolicyLoss(NamedTuple):
    loss: torch.Tensor
    logp: torch.Tensor


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor
    logp: torch.Tensor
    rewards: torch.Tensor


def _choice(table, key, what):
    if key not in table:
        raise ValueError(f"{what} must be one of {', '.join(table)}, not {key!r}")
    return table[key]


def _clip(clip):
    lo, hi = (clip, clip) if isinstance(clip, (int, float)) else clip
    return float(lo), float(hi)


def logprob_rows(logits, targets, mask=None):
    """(B, T) fp32 log-probabilities of the targets under logits (B, T, V) bf16 / fp16 / fp32; 0 where
    a token does not count. No gradient: see policy_loss, preference_loss and token_logprobs."""
    return N.ext().logprob_rows(logits, targets, mask)[0]


def _policy_rows(logits, targets, old_logp, advantages, ref_logp, mask, clip, kl_coef, reduction, grad, out=None, keep=False):
    lo, hi = _clip(clip)
    C = N.ext()
    if reduction == "sequence" or (reduction == "token" and targets.numel() > C.tokens_counted_in_rows):
        N.LAUNCHES.count += 1  # the kernel that counts the tokens
    return C.policy_rows(logits, targets, old_logp, advantages, ref_logp, mask, lo, hi, float(kl_coef),
                         _choice(REDUCTIONS, reduction, "reduction"), bool(grad), out, keep)


def policy_loss_rows(logits, targets, old_logp, advantages, ref_logp=None, mask=None, clip=(0.2, 0.2), kl_coef=0.0,
                     reduction="token", grad=True, out=None):
    """Clipped policy loss of logits (B, T, V) with the gradient of the logits.

    Per token, with r = exp(logp - old_logp) and d = ref_logp - logp,
        -min(r A, clip(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef (e^d - 1 - d)
    averaged over the tokens that count ("token"), over sequences of their own averages
    ("sequence", sequences without such tokens left out), or summed ("sum").
    old_logp None takes the current log-probabilities (the first step on a batch); advantages are
    (B, T) or broadcast to it, (B, 1) for one per sequence; one of zero takes no part whatever the
    ratio, a NaN makes the loss and its own row of the gradient NaN. `out` takes the gradient; it may be the
    logits themselves. Returns PolicyRows(loss, logp, dlogits)."""
    loss, logp, d, _, _ = _policy_rows(logits, targets, old_logp, advantages, ref_logp, mask, clip, kl_coef, reduction,
                                       grad, out)
    return PolicyRows(loss, logp, d if grad else None)


def preference_loss_rows(logits, targets, ref_logp=None, mask=None, beta=0.1, kind="sigmoid", label_smoothing=0.0,
                         average=False, grad=True, out=None):
    """Preference loss of logits (2 P, T, V), the P chosen sequences first and then the rejected ones
    in the same order, with the gradient of the logits.

    A sequence's gain is the sum of logp - ref_logp over its tokens that count (with `average`
    their mean; without ref_logp of logp alone), D the gain of the chosen less that of the rejected:
        sigmoid: -(1 - s) log sigma(beta D) - s log sigma(-beta D), s = label_smoothing
        hinge:   max(0, 1 - beta D)
        ipo:     (D - 1 / (2 beta))^2
    averaged over pairs. Returns PreferenceRows(loss, logp, rewards = beta * gains (2 P), dlogits)."""
    N.LAUNCHES.count += 1 if grad else 0  # the gradient's rows
    loss, logp, rewards, d, _, _ = N.ext().preference_rows(
        logits, targets, ref_logp, mask, float(beta), float(label_smoothing), _choice(KINDS, kind, "kind"), bool(average),
        bool(grad), out)
    return PreferenceRows(loss, logp, rewards, d if grad else None)


class _PolicyRowsFn(torch.autograd.Function):
    """The forward writes the gradient for an incoming gradient of 1 while it has the logits; the
    backward computes it again from the logits where it is another one (decided on the device), so
    it is rounded once either way."""

    @staticmethod
    def forward(ctx, logits, targets, old_logp, advantages, ref_logp, mask, clip, kl_coef, reduction):
        want = ctx.needs_input_grad[0]
        loss, logp, d, coef, stats = _policy_rows(logits, targets, old_logp, advantages, ref_logp, mask, clip, kl_coef,
                                                  reduction, want, keep=want)
        if want:
            ctx.save_for_backward(logits, targets, mask, coef, stats)
            ctx.ready = d
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        logits, targets, mask, coef, stats = ctx.saved_tensors
        ready, ctx.ready = ctx.ready, None  # handed out once; a second backward makes its own
        d = N.ext().grad_rows(logits, targets, mask, coef, stats, g.float().contiguous(), ready, ready is not None)
        return (d,) + (None,) * 8


class _PreferenceRowsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ref_logp, mask, beta, kind, label_smoothing, average):
        loss, logp, rewards, _, coef, stats = N.ext().preference_rows(
            logits, targets, ref_logp, mask, float(beta), float(label_smoothing), _choice(KINDS, kind, "kind"),
            bool(average), False, None, True)
        ctx.save_for_backward(logits, targets, mask, coef, stats)
        ctx.mark_non_differentiable(logp, rewards)
        return loss, logp, rewards

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _lp, _rw):
        logits, targets, mask, coef, stats = ctx.saved_tensors
        d = N.ext().grad_rows(logits, targets, mask, coef, stats, g.float().contiguous(), None, False)
        return (d,) + (None,) * 7


def policy_loss(logits, targets, old_logp, advantages, ref_logp=None, mask=None, clip=(0.2, 0.2), kl_coef=0.0,
                reduction="token"):
    """policy_loss_rows behind autograd: PolicyLoss(loss, logp); loss.backward() reaches the logits."""
    if not torch.is_grad_enabled():
        logits = logits.detach()  # a Function is told of the logits' flag alone: it would write their gradient
    return PolicyLoss(*_PolicyRowsFn.apply(logits, targets, old_logp, advantages, ref_logp, mask, clip, kl_coef, reduction))


def preference_loss(logits, targets, ref_logp=None, mask=None, beta=0.1, kind="sigmoid", label_smoothing=0.0,
                    average=False):
    """preference_loss_rows behind autograd: PreferenceLoss(loss, logp, rewards)."""
    return PreferenceLoss(*_PreferenceRowsFn.apply(logits, targets, ref_logp, mask, beta, kind, label_smoothing, average))


class _PolicyTokensFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, targets, vocab, old_logp, advantages, ref_logp, mask, clip, kl_coef, reduction):
        lo, hi = _clip(clip)
        loss, coef = N.ext().policy_tokens(logp.detach().contiguous(), targets, int(vocab), old_logp, advantages, ref_logp, mask,
                                           lo, hi, float(kl_coef), _choice(REDUCTIONS, reduction, "reduction"))
        ctx.save_for_backward(coef)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (coef,) = ctx.saved_tensors
        return (coef * g,) + (None,) * 9


class _PreferenceTokensFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, targets, vocab, ref_logp, mask, beta, kind, label_smoothing, average):
        loss, coef, rewards = N.ext().preference_tokens(
            logp.detach().contiguous(), targets, int(vocab), ref_logp, mask, float(beta), float(label_smoothing),
            _choice(KINDS, kind, "kind"), bool(average))
        ctx.save_for_backward(coef)
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        (coef,) = ctx.saved_tensors
        return (coef * g,) + (None,) * 8


def policy_loss_tokens(logp, targets, vocab, old_logp, advantages, ref_logp=None, mask=None, clip=(0.2, 0.2),
                       kl_coef=0.0, reduction="token"):
    """policy_loss_rows on log-probabilities (B, T) fp32 of the targets (ids of a vocabulary of
    `vocab`): the loss; its gradient goes to logp."""
    return _PolicyTokensFn.apply(logp, targets, vocab, old_logp, advantages, ref_logp, mask, clip, kl_coef, reduction)


def preference_loss_tokens(logp, targets, vocab, ref_logp=None, mask=None, beta=0.1, kind="sigmoid",
                           label_smoothing=0.0, average=False):
    """preference_loss_rows on log-probabilities (2 P, T) fp32: PreferenceLoss(loss, logp, rewards)."""
    loss, rewards = _PreferenceTokensFn.apply(logp, targets, vocab, ref_logp, mask, beta, kind, label_smoothing, average)
    return PreferenceLoss(loss, logp, rewards)
