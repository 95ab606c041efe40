"""The loss against a teacher's top logits, with its gradient."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ._ext import ext


@dataclass
class Teacher:
    """A teacher's top entries for the tokens of a micro-batch, and how they enter the loss."""

    ids: torch.Tensor  # int32 [..., K], -1: an unused place
    logits: torch.Tensor  # [..., K]
    temperature: float = 1.0
    alpha: float = 1.0  # weight of the teacher's part; the hard labels have 1 - alpha


def distill_topk(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                 targets: torch.Tensor | None = None, cap: float = 15.0, temperature: float = 1.0, alpha: float = 1.0,
                 scale: float | None = None, need_grad: bool = True,
                 grad: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """``(loss, rows, grad)`` of ``rows = alpha t^2 KL(teacher || student) + (1 - alpha) CE`` and
    ``loss = scale * sum(rows)`` (``scale`` defaults to ``1 / M``); ``grad`` is the gradient of ``loss`` with respect to
    the scores before the softcap.

    ``logits`` ``[M, V]`` (fp32, bf16, fp16; rows of up to 1 MB) are the student's, softcapped at ``cap`` (0: no
    softcap).
    ``teacher_ids`` (int32 ``[M, K]``, ``K`` up to 1024) and ``teacher_logits`` (fp32, bf16, fp16) are each row's top
    entries of the teacher; its distribution at temperature ``t`` is the softmax over them. An id of -1 is an unused
    place, and a row without entries adds nothing to the KL. Several entries with the same id add up. ``targets``
    (int32 ``[M]``, -1: ignored) are the hard labels of the cross-entropy ``-log(p + 1e-10)``, needed for
    ``alpha < 1``. Any other id outside ``[0, V)`` is skipped and reported through the device status word.

    ``grad`` may be given, also as ``logits`` itself (in place). ``need_grad=False`` returns the loss alone. Runs on
    the current stream of the logits' device, in a captured graph too (once any kernel of this package has run on
    that device); the same inputs give the same bits. Wrong arguments raise
    ``ValueError``, a ``grad`` that shares memory with another argument otherwise ``RuntimeError``."""
    if scale is None:
        scale = 1.0 / max(1, logits.shape[0])
    return ext().distill_topk(logits, teacher_ids, teacher_logits, targets, cap, temperature, alpha, scale, need_grad,
                              grad)
