"""Log-probabilities of given tokens and the paired preference loss, straight
from logits of any float dtype (csrc/preference.cu): one pass over the rows
that count forward, one backward, no 32-bit copy of the logits.

As in causal language models, position ``l`` is scored on ``labels[:, l + 1]``
(the shift happens inside), and labels equal to ``ignore_index`` (prompts,
padding) do not count; their rows are not read.
"""
from typing import NamedTuple

import torch

from rocm_qlora import _native as nat

_FORMS = {"sigmoid": 0, "ipo": 1}


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """[batch, length] float32: at each label's place its log-probability
    under the position before it, 0 where the label does not count (and at
    the first place).  A label outside the vocabulary gives NaN.
    Differentiable in ``logits``."""
    try:
        return nat.loaded_ops().label_logprobs(logits, labels, int(ignore_index))
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None


class PreferenceOutput(NamedTuple):
    """``loss`` (differentiable), and without gradients: ``logps`` [batch] sums
    of the log-probabilities that count, ``chosen_rewards`` and
    ``rejected_rewards`` [batch / 2]: beta * (log-probability - reference's)."""
    loss: torch.Tensor
    logps: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logps: torch.Tensor, beta: float = 0.1,
                    label_smoothing: float = 0.0, form: str = "sigmoid",
                    ignore_index: int = -100) -> PreferenceOutput:
    """The paired preference loss of a batch whose first half are the chosen
    answers and whose second half the rejected ones of the same prompts.

    ``ref_logps`` [batch, length] are the reference model's log-probabilities
    as ``token_logprobs`` gives them: per token, since the loss takes a small
    difference of two sums over the sequence.  With R the sum of
    (log p - ref) over the tokens of an answer and n their number,

        sigmoid: mean(-(1 - w) log sigma(z) - w log sigma(-z)),
                 z = beta (R_chosen - R_rejected), w = label_smoothing
        ipo:     mean((R_chosen / n - R_rejected / n - 1 / (2 beta))^2), which has no w
    """
    if form not in _FORMS:
        raise ValueError(f"form must be one of {sorted(_FORMS)}, got {form!r}")
    if not beta > 0.0:
        raise ValueError(f"beta must be positive, got {beta}")
    if not 0.0 <= label_smoothing <= 0.5:
        raise ValueError(f"label_smoothing must be between 0 and 0.5, got {label_smoothing}")
    try:
        return PreferenceOutput(*nat.loaded_ops().preference_loss(
            logits, labels, ref_logps, int(ignore_index), _FORMS[form], float(beta), float(label_smoothing)))
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None
