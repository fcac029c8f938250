"""Distillation from a teacher's top logits, beside the label loss of xent.py.

A teacher's whole distribution over a 50k vocabulary is 100 KB a token; its
K largest logits and their indices are a few hundred bytes and carry nearly
all of its mass.  One row of `distill_loss` is

    q   = softmax(t / tau)          over the entries that the row lists
    p   = softmax(z / tau)          over the whole vocabulary
    row = alpha * tau^2 * sum_k q_k (log q_k - log p[i_k])
          + (1 - alpha) * (logsumexp(z) - z[y])

and the loss is the sum of the rows over the number of rows that list an
entry or carry a label.  Loss and gradient come out of ONE pass over the logits
(csrc/distill.hip); no (N, V) fp32 intermediate.  bf16, fp16 and fp32 logits run the kernels on the GPU, the
CPU and fp64 the reference below.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import extension
from .functional import _acc_dtype


def _ref_distill(logits, index, teacher, targets, alpha, tau):
    """Plain-torch semantics (CPU path and test oracle); autograd gives its
    gradient."""
    V = logits.shape[1]
    z = logits.to(_acc_dtype(logits.dtype))
    t = teacher.detach().to(z.dtype)
    given = (index >= 0) & (index < V) & (t != -math.inf)
    soft = given.any(dim=1)
    label = torch.zeros_like(soft)
    if targets is not None:
        label = (targets >= 0) & (targets < V)
    # a row that adds nothing has a zero gradient whatever its logits hold
    used = torch.zeros_like(soft)
    if alpha != 0.0:
        used = used | soft
    if alpha != 1.0:
        used = used | label
    z = torch.where(used[:, None], z, 0.0)
    rows = z.new_zeros(z.shape[0])
    if alpha != 0.0 and index.shape[1] > 0:
        t = torch.where(given, t / tau, -math.inf)
        q = torch.softmax(torch.where(soft[:, None], t, 0.0), dim=1)
        q = torch.where(given, q, 0.0)
        logq = torch.where(q == 0, 0.0, q.log())
        logp = torch.log_softmax(z / tau, dim=1).gather(
            1, torch.where(given, index, 0).long())
        kl = torch.where(q == 0, 0.0, q * (logq - logp)).sum(dim=1)
        rows = rows + alpha * tau * tau * kl
    if targets is not None and alpha != 1.0:
        y = torch.where(label, targets, 0)
        ce = -torch.log_softmax(z, dim=1).gather(1, y[:, None]).squeeze(1)
        rows = rows + (1.0 - alpha) * torch.where(label, ce, 0.0)
    return rows.sum() / (soft | label).sum().clamp_min(1)


def _check(logits, teacher_index, teacher_logits, targets):
    """What the kernels' path refuses in csrc/lm_ops.cpp."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be (N, V), got {tuple(logits.shape)}")
    N, V = logits.shape
    if V < 1 or not logits.dtype.is_floating_point:
        raise ValueError("logits must be floating and have a vocabulary")
    if (teacher_index.dim() != 2 or teacher_index.shape[0] != N
            or teacher_index.shape != teacher_logits.shape):
        raise ValueError(
            f"teacher_index and teacher_logits must be (N={N}, K), got "
            f"{tuple(teacher_index.shape)}, {tuple(teacher_logits.shape)}")
    if teacher_index.dtype not in (torch.int32, torch.int64):
        raise ValueError("teacher_index must be int32 or int64")
    if not teacher_logits.dtype.is_floating_point:
        raise ValueError("teacher_logits must be floating")
    if targets is not None and (targets.dtype != torch.long
                                or targets.shape != (N,)):
        raise ValueError(f"targets must be (N={N},) int64")
    for t in (teacher_index, teacher_logits, targets):
        if t is not None and t.device != logits.device:
            raise ValueError(f"all tensors must be on {logits.device}")


def distill_loss(logits: torch.Tensor, teacher_index: torch.Tensor,
                 teacher_logits: torch.Tensor,
                 targets: Optional[torch.Tensor] = None, *,
                 alpha: float = 1.0, temperature: float = 1.0,
                 weight: float = 1.0) -> torch.Tensor:
    """Mean loss (fp32 scalar; fp64 for fp64 logits) over the rows that list
    a teacher's entry or carry a label.

    logits: (N, V) of the student; its rows may have any stride.
    teacher_index, teacher_logits: (N, K), e.g. `topk` of the teacher's
    logits.  An entry whose index lies outside [0, V), or whose logit is
    -inf, is absent: rows may list fewer than K, or none.  The same index
    twice in a row counts twice.  The teacher gets no gradient.
    targets: (N,) int64 labels or None; one outside [0, V) is no label.
    alpha weighs the teacher against the labels (without labels it has to be
    1), `temperature` applies to the teacher's term alone.
    weight multiplies the loss.  Given here (1 / micro-batches, a loss scale)
    and not afterwards, it keeps the incoming gradient at 1, for which the
    forward has already written the logits' gradient; for any other the
    backward computes it anew.
    A row of padding (no entry and no label) adds nothing, is not counted
    and gets a zero gradient.
    """
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"alpha must be in [0, 1], got {alpha}")
    if not 1e-6 <= temperature <= 1e6:      # its square and inverse in fp32
        raise ValueError("temperature must be in [1e-6, 1e6], got "
                         f"{temperature}")
    if not math.isfinite(weight):
        raise ValueError(f"weight must be finite, got {weight}")
    if targets is None and alpha != 1.0:
        raise ValueError("alpha < 1 needs targets")
    if extension.use_hip_lm(logits):
        return extension.get_extension().distill_loss(
            logits, teacher_index, teacher_logits, targets, alpha,
            temperature, weight)
    _check(logits, teacher_index, teacher_logits, targets)
    loss = _ref_distill(logits, teacher_index, teacher_logits, targets,
                        float(alpha), float(temperature))
    return loss * weight
