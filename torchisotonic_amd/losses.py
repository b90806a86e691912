"""Losses of language-model training over the log-probabilities of tokens: preference losses over
pairs of sequences, and the clipped policy loss with a divergence term, each with its gradient.

Sequences come as rows of one length ([sequences, tokens]) or, as ``isotonic_ragged`` takes its rows,
packed end to end with ``offsets`` (or ``lengths``); a boolean ``mask`` leaves tokens out (prompts,
pads), whatever their values. ``token_logprobs`` gives the log-probabilities.

- ``preference_loss``: with s the sum (or mean) over a sequence's tokens of its log-probabilities less
  the reference model's, and h = s_chosen - s_rejected for each pair, the pairs' mean of a loss of h.
  The margins beta * h are scores of "the chosen one is better", which ``IsotonicCalibrator`` turns
  into probabilities.
- ``policy_loss``: with r = exp(logps - old_logps) and A a token's advantage, the tokens' mean of
  -min(r A, clip(r) A), plus kl_coef (exp(d) - 1 - d), d = reference_logps - logps, an estimate of the
  divergence from the reference. Advantages of a group of samples may be their soft ranks.

The tokens' sums, the losses and the gradients run in HIP kernels (``ti_preference``, ``ti_policy``);
sums are float64 in a fixed order, but that a policy loss's first adds the terms of four float32 tokens
in float32. Nothing waits for the GPU: offsets on the GPU that are not what they
have to be make the loss and the gradient of every unmasked token NaN instead of raising (of single
losses, the pairs' whose own they are: no other can then be relied on). The reference has no counterpart.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import Tensor

from torchisotonic_amd import _ext
from torchisotonic_amd.ragged import _offsets_tensor

_KINDS = {"logistic": 0, "hinge": 1, "squared": 2}
_PAIRS = {"none": 0, "mean": 1, "sum": 2}
_TOKENS = {"token_mean": 1, "sum": 2, "sequence_mean": 3}


class PreferenceLoss(NamedTuple):
    """``loss``: the reduced loss (or one a pair). ``chosen_rewards``, ``rejected_rewards``: beta times
    each pair's log ratios, without gradient."""

    loss: Tensor
    chosen_rewards: Tensor
    rejected_rewards: Tensor


class PolicyLoss(NamedTuple):
    """``loss``: the reduced loss. ``kl``, ``clip_fraction``: the tokens' mean divergence estimate from
    the reference (0 without one) and the share of tokens whose clipped term counts, without gradient."""

    loss: Tensor
    kl: Tensor
    clip_fraction: Tensor


def _tokens(logps: Tensor) -> Tensor:
    """The token log-probabilities as the kernels take them: contiguous float32 or float64."""
    if not isinstance(logps, Tensor):
        raise TypeError(f"logps must be a torch.Tensor, got {type(logps).__name__}")
    if logps.ndim not in (1, 2):
        raise ValueError(f"logps must be 1-D or [sequences, tokens], got shape {tuple(logps.shape)}")
    if not logps.is_floating_point():
        raise TypeError(f"logps must be a float tensor, got {logps.dtype}")
    _ext._on_gpu(logps, "logps")
    if logps.dtype not in (torch.float32, torch.float64):
        logps = logps.to(torch.float32)
    return logps.contiguous()


def _constant(name: str, t: Tensor, like: Tensor, shapes: tuple = ()) -> Tensor:
    """An input that no gradient goes to, in the dtype and on the device of ``like``."""
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.shape != like.shape and t.shape not in shapes:
        raise ValueError(f"{name} of shape {tuple(t.shape)} does not fit logps of shape {tuple(like.shape)}")
    if t.requires_grad:
        if torch.is_grad_enabled():
            raise ValueError(f"{name} gets no gradient: detach it")
        t = t.detach()
    if t.dtype != like.dtype or t.device != like.device:
        t = t.to(device=like.device, dtype=like.dtype)
    return t.contiguous()


def _mask(mask: Tensor | None, like: Tensor) -> Tensor | None:
    if mask is None:
        return None
    if not isinstance(mask, Tensor) or mask.dtype != torch.bool or mask.shape != like.shape:
        raise ValueError("mask must be a bool tensor shaped like logps")
    return (mask if mask.device == like.device else mask.to(device=like.device)).contiguous()


def _sequences(logps: Tensor, offsets, lengths) -> Tensor | None:
    """The offsets of packed sequences on the GPU, or None: rows of one length, or (1-D) one sequence.
    Offsets that are on the host are checked here."""
    if offsets is None and lengths is None:
        return None
    if logps.ndim != 1:
        raise ValueError("offsets / lengths go with 1-D logps (sequences packed end to end)")
    src = offsets if offsets is not None else lengths
    if not isinstance(src, Tensor) or src.device.type == "cpu":
        host = _offsets_tensor(offsets, lengths, torch.device("cpu"))
        if bool((host.diff() < 0).any()):
            raise ValueError("offsets must not decrease" if offsets is not None else "lengths must be non-negative")
        if int(host[0]) != 0 or int(host[-1]) != logps.numel():
            raise ValueError(f"offsets must run from 0 to logps.numel() = {logps.numel()}")
        offsets, lengths = host, None
    off = _offsets_tensor(offsets, lengths, logps.device)
    if off.numel() == 1 and logps.numel() > 0:
        raise ValueError(f"offsets must run from 0 to logps.numel() = {logps.numel()}")
    return off


def preference_loss(
    logps: Tensor,
    reference_logps: Tensor | None = None,
    *,
    offsets: Tensor | None = None,
    lengths: Tensor | None = None,
    mask: Tensor | None = None,
    beta: float = 0.1,
    loss: str = "logistic",
    label_smoothing: float = 0.0,
    average: bool = False,
    reduction: str = "mean",
) -> PreferenceLoss:
    """A preference loss over pairs of sequences: the first half of the sequences are the chosen ones,
    the second half the rejected ones, in the same order. ``logps`` are their tokens' log-probabilities
    under the trained model ([2 pairs, tokens], or 1-D with ``offsets`` or ``lengths``) and
    ``reference_logps`` those under the reference model (None: zeros); tokens whose ``mask`` is False
    are left out. With s a sequence's sum of ``logps - reference_logps`` (``average``: its mean; 0
    without tokens) and h = s_chosen - s_rejected, the loss of a pair is

    - "logistic": -(1 - label_smoothing) log sigmoid(beta h) - label_smoothing log sigmoid(-beta h),
    - "hinge": max(0, 1 - beta h),
    - "squared": (h - 1 / (2 beta))^2,

    (``label_smoothing``, the share of pairs taken to be labelled the wrong way round, counts in the
    first only) and ``reduction`` the pairs' "mean" (0 where there are none), "sum" or "none". The gradient goes to
    ``logps``. float16 and bfloat16 are computed in float32."""
    x = _tokens(logps)
    ref = None if reference_logps is None else _constant("reference_logps", reference_logps, x)
    m = _mask(mask, x)
    if loss not in _KINDS:
        raise ValueError(f"loss must be one of {', '.join(_KINDS)}, got {loss!r}")
    if reduction not in _PAIRS:
        raise ValueError(f"reduction must be one of {', '.join(_PAIRS)}, got {reduction!r}")
    if not (beta > 0 and math.isfinite(beta)):
        raise ValueError("beta must be positive and finite")
    if not 0 <= label_smoothing < 1:
        raise ValueError("label_smoothing must be in [0, 1)")
    off = _sequences(x, offsets, lengths)
    if off is None and x.ndim != 2:
        raise ValueError("1-D logps need offsets or lengths")
    count = x.shape[0] if off is None else off.numel() - 1
    if count % 2:
        raise ValueError(f"the sequences must be pairs, got {count}")
    out = _ext.ops().preference_loss(x, ref, off, m, _KINDS[loss], float(beta), float(label_smoothing), bool(average),
                                     _PAIRS[reduction])
    return PreferenceLoss(*out)


def policy_loss(
    logps: Tensor,
    old_logps: Tensor,
    advantages: Tensor,
    *,
    reference_logps: Tensor | None = None,
    offsets: Tensor | None = None,
    lengths: Tensor | None = None,
    mask: Tensor | None = None,
    clip: float = 0.2,
    clip_high: float | None = None,
    kl_coef: float = 0.0,
    reduction: str = "token_mean",
) -> PolicyLoss:
    """The clipped policy loss of sampled tokens: ``logps`` under the trained model, ``old_logps`` under
    the one that sampled them ([sequences, tokens], or 1-D, with ``offsets`` or ``lengths`` where
    sequences matter); ``advantages`` one a token (shaped like ``logps``; a 1-D shape that fits both is
    taken so) or one a sequence; tokens whose ``mask`` is False are left out. With
    r = exp(logps - old_logps), a token's loss is

        -min(r A, clip(r, 1 - clip, 1 + clip_high) A)   (clip_high: ``clip`` where not given)

    plus, given ``reference_logps``, kl_coef (exp(d) - 1 - d) with d = reference_logps - logps.
    ``reduction``: "token_mean" over all tokens, "sequence_mean" (the mean over all sequences of each
    one's mean over its tokens) or "sum"; of no tokens, 0. float16 and bfloat16 are computed in float32.

    The gradient goes to ``logps``. Where one may be asked for, it is computed with the loss and held (a
    value a token, not seen by saved-tensor hooks) until the backward, which multiplies it by the upstream
    gradient in one more read and write, or leaves it where that is one: ``loss / k`` costs that pass, a
    coefficient that is in ``advantages`` and ``kl_coef`` already does not."""
    x = _tokens(logps)
    old = _constant("old_logps", old_logps, x)
    ref = None if reference_logps is None else _constant("reference_logps", reference_logps, x)
    m = _mask(mask, x)
    if reduction not in _TOKENS:
        raise ValueError(f"reduction must be one of {', '.join(_TOKENS)}, got {reduction!r}")
    high = clip if clip_high is None else clip_high
    if not (0 <= clip <= 1 and 0 <= high < math.inf):
        raise ValueError("clip must be in [0, 1] and clip_high finite and not negative")
    if not math.isfinite(kl_coef):
        raise ValueError("kl_coef must be finite")
    if kl_coef != 0 and ref is None:
        raise ValueError("kl_coef needs reference_logps")
    off = _sequences(x, offsets, lengths)
    sequences = off is not None or x.ndim == 2
    count = off.numel() - 1 if off is not None else x.shape[0]
    if reduction == "sequence_mean" and not sequences:
        raise ValueError("sequence_mean of 1-D logps needs offsets or lengths")
    adv = _constant("advantages", advantages, x, ((count,),) if sequences else ())
    out = _ext.ops().policy_loss(x, old, adv, ref, off, m, float(clip), float(high), float(kl_coef), _TOKENS[reduction])
    return PolicyLoss(*out)
