"""Causal attention with a sliding window and a few first tokens that stay
visible (csrc/window_attn.hip): forward, backward and single tokens over a
cache.

Row ``i`` of sequence ``b`` stands at position ``p = q_start + i`` and sees
key ``j`` where ``j <= p`` and either ``p - j < window`` (the last ``window``
tokens, its own among them) or ``j < sinks``.  A row whose position lies
outside its sequence (``p < 0`` or ``p >= lengths[b]``) is padding: its output
is zero and nothing flows back through it.

GPU tensors run the native kernels (scores are never written to memory;
scores, softmax statistics and sums in 32 bits, probabilities and score
gradients rounded to the inputs' dtype for the products that follow, in fp16 at
a power of two that keeps them clear of its subnormals and its end), CPU
tensors the same formula in torch.
The backward pass sums in a fixed order: no atomics, bit-reproducible.
"""
from __future__ import annotations

import contextlib

import torch

from distributed_kfac_pytorch_amd.ops import _native as _nat

__all__ = ['window_attention']

MAX_HEAD = 128
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_SMALLEST = 2.0 ** -126  # fp32 holds numbers from here to 1 / here in full


def _reference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int,
               lengths: torch.Tensor | None, start: torch.Tensor, scale: float) -> torch.Tensor:
    tq, tk, group = q.shape[2], k.shape[2], q.shape[1] // k.shape[1]
    work = torch.float64 if q.dtype == torch.float64 else torch.float32
    p = start.long()[:, None, None] + torch.arange(tq, device=q.device)[:, None]
    j = torch.arange(tk, device=q.device)
    n = torch.full_like(p[:, :1], tk) if lengths is None else lengths.long().clamp(0, tk)[:, None, None]
    see = (j <= p) & ((p - j < window) | (j < sinks)) & (p < n) & (j < n)
    see = see[:, None]
    # keys that no row sees may hold anything, and so may rows of padding and
    # what comes back for them
    used, rows = see.any(dim=2)[..., None], see.any(dim=3)[..., None]
    kk = torch.where(used, k, 0.0).to(work).repeat_interleave(group, dim=1)
    vv = torch.where(used, v, 0.0).to(work).repeat_interleave(group, dim=1)
    # the products keep `work` under autocast, as the kernels' sums do
    with (torch.autocast(q.device.type, enabled=False)
          if torch.amp.is_autocast_available(q.device.type) else contextlib.nullcontext()):
        s = (torch.where(rows, q, 0.0).to(work) @ kk.transpose(-1, -2)) * scale
        s = s.masked_fill(~see, float('-inf'))
        m = s.detach().amax(dim=-1, keepdim=True) if tk else s.new_zeros(*s.shape[:-1], 1)
        e = torch.exp(s - m.masked_fill(m == float('-inf'), 0.0))
        total = e.sum(dim=-1, keepdim=True)
        o = torch.where(rows, (e / total.masked_fill(total == 0.0, 1.0)) @ vv, 0.0)
    b, h, t, d = o.shape
    return torch.empty_strided((b, h, t, d), (t * h * d, d, h * d, 1), dtype=q.dtype,
                               device=q.device).copy_(o)


def window_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    window: int,
    sinks: int = 0,
    lengths: torch.Tensor | None = None,
    q_start: int | torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of ``q`` ``[B, Hq, Tq, D]`` to ``k``, ``v`` ``[B, Hk, Tk, D]``.

    Args:
        q, k, v: bf16, fp16 or fp32 of one dtype, any strides (rows that
            16-byte accesses cannot read are copied first); ``Hq`` a multiple
            of ``Hk`` (heads ``h * Hq / Hk ...`` share key / value head
            ``h``), ``D`` a multiple of 8, at most 128.
        window: tokens a row sees, itself included; at least 1.
        sinks: first tokens that stay visible behind the window.
        lengths: int32 ``[B]``, tokens of each sequence (at most ``Tk``; more
            count as ``Tk``, negative ones as 0).  Keys from there on may hold
            anything.  Default: ``Tk``.
        q_start: position of row 0: one number, or int32 ``[B]``.  Default:
            the rows are a sequence's last ones, ``lengths - Tq`` -- new
            tokens behind a cache, or a full sequence.  A right-padded
            training batch passes ``lengths`` and ``q_start=0``.
        scale: factor of the scores, from 2^-126 to 2^126; default
            ``D ** -0.5``.

    Returns:
        ``[B, Hq, Tq, D]`` over memory laid out ``[B, Tq, Hq, D]``, which
        ``transpose(1, 2).flatten(2)`` reads without a copy.  Gradients flow
        to ``q``, ``k`` and ``v``.  Rows of padding and keys that no row sees
        may hold anything; infinities and NaN in what is seen may reach other
        rows of their sequence and head.
    """
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f'q must be [B, Hq, Tq, D], k and v [B, Hk, Tk, D], got '
                         f'{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}')
    b, hq, tq, d = q.shape
    if k.shape[0] != b or k.shape[3] != d or k.shape[1] == 0 or hq % k.shape[1] != 0:
        raise ValueError(f'q {tuple(q.shape)} does not fit k {tuple(k.shape)}')
    if d % 8 != 0 or not 8 <= d <= MAX_HEAD:
        raise ValueError(f'head size must be a multiple of 8, at most {MAX_HEAD}, got {d}')
    if not (q.dtype == k.dtype == v.dtype) or (
            q.dtype not in _DTYPES and (q.is_cuda or q.dtype != torch.float64)):
        raise TypeError(f'q, k, v must share bf16, fp16 or fp32, got {q.dtype}, {k.dtype}, {v.dtype}')
    if not (q.device == k.device == v.device):
        raise ValueError('q, k and v must be on one device')
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f'window must be at least 1 and sinks at least 0, got {window}, {sinks}')
    scale = d ** -0.5 if scale is None else float(scale)
    if not _SMALLEST <= scale <= 1.0 / _SMALLEST:
        raise ValueError(f'scale must be positive, a normal number of 32 bits, got {scale}')
    for name, t in (('lengths', lengths), ('q_start', q_start)):
        if isinstance(t, torch.Tensor) and (
                t.dtype != torch.int32 or tuple(t.shape) != (b,) or t.device != q.device):
            raise ValueError(f'{name} must be int32 [{b}] on the device of q, got {t.dtype} '
                             f'{tuple(t.shape)} on {t.device}')
    starts = q_start if isinstance(q_start, torch.Tensor) else None
    if _nat.use_native(q, k, v):
        return _nat.native().window_attention(  # type: ignore[union-attr]
            q, k, v, None if lengths is None else lengths.contiguous(),
            None if starts is None else starts.contiguous(), window, sinks,
            int(q_start) if starts is None and q_start is not None else 0,
            q_start is not None, scale)
    if starts is None:
        if q_start is not None:
            starts = torch.full((b,), int(q_start), device=q.device)
        elif lengths is not None:
            starts = lengths.long().clamp(0, k.shape[2]) - tq
        else:
            starts = torch.full((b,), k.shape[2] - tq, device=q.device)
    return _reference(q, k, v, window, sinks, lengths, starts, scale)
