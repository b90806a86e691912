"""Log-probabilities of given tokens under a language model's logits: the scores that the losses
of ``torchisotonic_amd.losses`` compare, that a calibrator maps to probabilities, and that a
serving loop returns beside its tokens.

For a row z of logits, its target t and a temperature T,

    logp    = z_t / T - log sum_j exp(z_j / T)
    entropy = -sum_j p_j log p_j,                    p = softmax(z / T)
    dlogp/dz_j    = ((j == t) - p_j) / T
    dentropy/dz_j = -p_j (log p_j + entropy) / T

computed in one pass over the logits and differentiated in one more (``ti_logprobs``,
``ti_logprobs_bwd``), with no softmax, one-hot or float copy of the logits in memory. The reference
has no language-model operators; its users bring scores.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from torchisotonic_amd import _ext

_FLOATS = (torch.float32, torch.float64, torch.bfloat16, torch.float16)


def token_logprobs(
    logits: Tensor,
    targets: Tensor,
    *,
    temperature: float = 1.0,
    ignore_index: int = -100,
    entropy: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    """The log-probability of each target token: ``log_softmax(logits / temperature)`` at
    ``targets``, for logits [..., vocab] (float32, float64, bfloat16 or float16, on the GPU) and
    integer targets [...]; with ``entropy`` the rows' entropies (in nats) as well. Results are
    float32 (float64 for float64 logits) and differentiable in the logits (once, in reverse mode), whose
    gradient has their dtype.

    A row whose target is ``ignore_index`` (a prompt's or a pad's) gives 0 with a gradient of 0,
    and its logits are not read, whatever they hold. To score a text against itself shifted by one,
    shift the targets and ignore the last place, rather than slicing the logits: the gradient of a
    slice costs another copy. A target outside [0, vocab) otherwise gives NaN (nothing waits for the
    GPU to check it), and so does a row with a NaN, with +inf, or with -inf only. A logit of -inf
    among others is a token of probability 0. Rows may be strided; rows that are not contiguous
    themselves are copied."""
    for name, t in (("logits", logits), ("targets", targets)):
        if not isinstance(t, Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., vocab], got shape {tuple(logits.shape)}")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits must be float32, float64, bfloat16 or float16, got {logits.dtype}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets must have logits' leading shape {tuple(logits.shape[:-1])}, got {tuple(targets.shape)}")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise TypeError(f"targets must be integers, got {targets.dtype}")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError("temperature must be positive and finite")
    _ext._on_gpu(logits, "logits")
    if targets.dtype != torch.int64 or targets.device != logits.device:
        targets = targets.to(device=logits.device, dtype=torch.int64)
    logp, h = _ext.ops().token_logprobs(logits, targets.contiguous(), float(temperature), int(ignore_index), entropy)
    return (logp, h) if entropy else logp
