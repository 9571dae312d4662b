"""Distillation from a teacher's top logits (csrc/distill.hip), forward and
backward: the divergence from the teacher's distribution, of which each row
keeps its ``K`` best entries, to the student's over the whole vocabulary.

    p = softmax over the teacher's entries / temperature (and its rest)
    q = softmax(logits / temperature)
    loss = temperature ** 2 * [sum_k p_k (ln p_k - ln q_k) + r (ln r - ln R)]

``teacher_rest`` is the log-sum-exp of the teacher's other logits (each
divided by the temperature): ``r`` is the share of the rest, ``R`` what the
student gives to the columns outside the row's entries.  Without it the
entries are renormalised and ``r = 0``.

GPU tensors run the native kernels, which make no copy of the logits in fp32,
sum in 32 bits or more and are bit-reproducible.  With 256 rows or more in
bf16 or fp32 the forward reads the logits once and writes their gradient in
the same pass; otherwise the backward reads them once more.  CPU tensors run
the same formula in torch.  ``utils.training.TopKDistillLoss`` is the module
form.
"""
from __future__ import annotations

import torch

from distributed_kfac_pytorch_amd.ops import _native as _nat

__all__ = ['topk_distill_loss']

MAX_ENTRIES = 1024
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_REDUCTIONS = ('none', 'sum', 'mean')
_INF = float('inf')
_LARGEST = 2.0 ** 63


def _reference(z: torch.Tensor, teacher: torch.Tensor, index: torch.Tensor,
               rest: torch.Tensor | None, tau: float, reduction: str) -> torch.Tensor:
    work = torch.float64 if z.dtype == torch.float64 else torch.float32
    there = index >= 0
    outside = (index >= z.shape[-1]).any(dim=-1)
    idx = torch.where(there & (index < z.shape[-1]), index, 0).long()
    # the type's lowest value over a temperature under 1 is a number of 64 bits
    t = (teacher.double() / tau).masked_fill(~there, -_INF)
    if rest is not None:
        t = torch.cat([t, rest.double()[..., None]], dim=-1)
    counts = there.any(dim=-1) & (t != -_INF).any(dim=-1)
    logp = torch.log_softmax(torch.where(counts[..., None], t, 0.0), dim=-1).to(work)
    p = torch.exp(logp)
    # a row that does not count may hold anything
    u = torch.where(counts[..., None], z, 0.0).to(work)
    top = u.detach().amax(dim=-1, keepdim=True)
    logq = torch.log_softmax((u - torch.where(top.isfinite(), top, 0.0)) / tau, dim=-1)
    k = index.shape[-1]
    weighs = there & (p[..., :k] != 0.0) & counts[..., None]
    diff = torch.where(weighs, logp[..., :k], 0.0) - torch.where(weighs, logq.gather(-1, idx), 0.0)
    rows = (p[..., :k].masked_fill(~weighs, 0.0) * diff).sum(dim=-1)
    if rest is not None:
        hits = torch.zeros(z.shape, dtype=torch.int32, device=z.device)
        member = hits.scatter_add_(-1, idx, there.to(torch.int32)) > 0
        some = (p[..., k] != 0.0) & counts & ~member.all(dim=-1)
        left = logq.masked_fill(member | ~some[..., None], -_INF)
        log_r = torch.logsumexp(torch.where(some[..., None], left, 0.0), dim=-1)
        empty = (p[..., k] != 0.0) & counts & member.all(dim=-1)
        rest_term = p[..., k].masked_fill(~some, 0.0) * (
            torch.where(some, logp[..., k], 0.0) - torch.where(some, log_r, 0.0))
        rows = rows + rest_term.masked_fill(empty, _INF)
    rows = rows * torch.where(outside, float('nan'), 1.0)
    rows = rows.masked_fill(~counts, 0.0) * (tau * tau)
    if reduction == 'none':
        return rows.float() if work == torch.float32 else rows
    total = rows.sum()
    return total / counts.sum().clamp(min=1) if reduction == 'mean' else total


def topk_distill_loss(
    logits: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_index: torch.Tensor,
    *,
    teacher_rest: torch.Tensor | None = None,
    temperature: float = 1.0,
    weight: float = 1.0,
    reduction: str = 'mean',
) -> torch.Tensor:
    """Divergence of the student's ``logits`` ``[..., V]`` from a teacher of
    which ``K`` entries a row are known.

    Args:
        logits: bf16, fp16 or fp32, any strides with a unit last one.  Columns
            masked with -inf or the type's lowest value have no probability;
            a row of nothing but the lowest value is uniform over its columns.
        teacher_logits: ``[..., K]``, the teacher's logits of the entries
            (not divided by the temperature), 1 <= K <= 1024; constant.
        teacher_index: int32 or int64 ``[..., K]``, their columns.  A negative
            index is no entry; a row without entries is padding: no loss, no
            gradient, not counted by the mean.  An index given twice counts
            with both its parts; one at or behind ``V`` makes its row's loss
            and gradient NaN.
        teacher_rest: ``[...]``, log-sum-exp of the teacher's other logits
            divided by the temperature; constant.
        temperature: positive, from 2^-63 to 2^63 (its square is a number of
            32 bits); the loss carries the square.
        weight: factor of the loss, finite in 32 bits.  Give a known factor (a mixing weight, one
            over the accumulation steps) here rather than multiply the result:
            in bf16 and fp32 the forward already writes the gradient, and a
            factor put on later costs another pass over it.
        reduction: ``'mean'`` over the rows that have entries, ``'sum'`` or
            ``'none'`` (``[...]``).

    Returns:
        fp32.  Gradients flow to ``logits``.
    """
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f'logits must be [..., V], got {tuple(logits.shape)}')
    lead = tuple(logits.shape[:-1])
    k = teacher_logits.shape[-1] if teacher_logits.dim() > 0 else 0
    if tuple(teacher_logits.shape) != (*lead, k) or teacher_index.shape != teacher_logits.shape:
        raise ValueError(f'teacher_logits and teacher_index must be {(*lead, "K")}, got '
                         f'{tuple(teacher_logits.shape)}, {tuple(teacher_index.shape)}')
    if not 1 <= k <= MAX_ENTRIES:
        raise ValueError(f'1 to {MAX_ENTRIES} teacher entries a row, got {k}')
    if logits.dtype not in _DTYPES and (logits.is_cuda or logits.dtype != torch.float64):
        raise TypeError(f'logits must be bf16, fp16 or fp32, got {logits.dtype}')
    if not teacher_logits.is_floating_point():
        raise TypeError(f'teacher_logits must be floating point, got {teacher_logits.dtype}')
    if teacher_index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f'teacher_index must be int32 or int64, got {teacher_index.dtype}')
    if teacher_rest is not None and (tuple(teacher_rest.shape) != lead
                                     or not teacher_rest.is_floating_point()):
        raise ValueError(f'teacher_rest must be floating point {lead}, got '
                         f'{teacher_rest.dtype} {tuple(teacher_rest.shape)}')
    for t in (teacher_logits, teacher_index, teacher_rest):
        if t is not None and t.device != logits.device:
            raise ValueError('logits and the teacher must be on one device')
    temperature = float(temperature)
    if not 1.0 / _LARGEST <= temperature <= _LARGEST:
        raise ValueError(f'temperature must be positive, from 2^-63 to 2^63, got {temperature}')
    weight = float(weight)
    if not abs(weight) <= torch.finfo(torch.float32).max:
        raise ValueError(f'weight must be finite in 32 bits, got {weight}')
    if reduction not in _REDUCTIONS:
        raise ValueError(f'reduction must be one of {_REDUCTIONS}, got {reduction!r}')
    teacher_logits = teacher_logits.detach()
    rest = None if teacher_rest is None else teacher_rest.detach()
    if not _nat.use_native(logits):
        loss = _reference(logits, teacher_logits, teacher_index, rest, temperature, reduction)
        return loss if weight == 1.0 else loss * weight
    z = logits
    if z.stride(-1) != 1 and z.shape[-1] > 1:
        z = z.contiguous()
    if z.dim() < 3:
        z = z[(None,) * (3 - z.dim())]
    elif z.dim() > 3:
        z = z.flatten(0, -3)
    return _nat.native().topk_distill_loss(  # type: ignore[union-attr]
        z, teacher_logits.float().contiguous(), teacher_index.contiguous(),
        None if rest is None else rest.float().contiguous(), temperature,
        weight, _REDUCTIONS.index(reduction), lead)
