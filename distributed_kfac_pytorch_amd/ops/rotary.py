"""Rotary positions with several axes (csrc/rotary.hip): text positions, or
(time, height, width) of image and video tokens, for q and k in one launch,
forward and backward.

``sections`` says how many pairs of a head each axis turns, in order; they
take the first ``2 * sum(sections)`` elements of the head and what lies
behind is passed through.  Pair ``i`` of axis ``a`` turns by
``positions[..., a] * base ** -e``, with ``e = i / sum(sections)`` counted
over all pairs (``ladder='shared'``) or ``i / sections[a]`` counted within
the axis (``'per_axis'``).  ``layout='interleaved'`` pairs elements
``(2 i, 2 i + 1)`` as ``models/gpt_neox.py`` does, ``'halves'`` pairs
``(i, i + sum(sections))``.

Angles are formed in 64 bits, products in 32; results are rounded once.  GPU
tensors run the native kernel, CPU tensors the same formula in torch.
"""
from __future__ import annotations

import functools
import math
from typing import Sequence

import torch

from distributed_kfac_pytorch_amd.ops import _native as _nat

__all__ = ['rotary_axes']

MAX_PAIRS = 128
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


@functools.lru_cache(maxsize=64)
def _rows(sections: tuple[int, ...], base: float, ladder: str) -> tuple[tuple[float, float], ...]:
    """(frequency in turns per position, axis) of each pair."""
    pairs = sum(sections)
    rows: list[tuple[float, float]] = []
    for a, n in enumerate(sections):
        for i in range(n):
            e = i / n if ladder == 'per_axis' else len(rows) / pairs
            rows.append((base ** -e / (2.0 * math.pi), float(a)))
    return tuple(rows)


_kept: dict[tuple[tuple[int, ...], float, str], torch.Tensor] = {}


def _table(sections: tuple[int, ...], base: float, ladder: str) -> torch.Tensor:
    """The rows as fp64 [pairs, 2] on the CPU.  Kept for the next call: an
    ordinary tensor under inference mode too, and not kept at all where the
    call's own mode makes another one of it (a fake one)."""
    key = (sections, base, ladder)
    table = _kept.get(key)
    if table is None:
        with torch.inference_mode(False):
            table = torch.tensor(_rows(*key), dtype=torch.float64, device='cpu')
        if type(table) is torch.Tensor and len(_kept) < 64:
            _kept[key] = table
    return table


def _reference(x: torch.Tensor, positions: torch.Tensor, rows: tuple[tuple[float, float], ...],
               halves: bool) -> torch.Tensor:
    n = len(rows)
    table = torch.tensor(rows, dtype=torch.float64, device=x.device)
    pos = positions if positions.dim() == 3 else positions[None]
    freq, axis = table[:, 0] * (2.0 * math.pi), table[:, 1].long()
    ang = pos.double()[..., axis] * freq
    # a 64-bit input keeps its bits; the others are turned in 32
    work = torch.float64 if x.dtype == torch.float64 else torch.float32
    c, s = ang.cos().to(work)[:, None], ang.sin().to(work)[:, None]
    y = x.to(work)
    if halves:
        x1, x2 = y[..., :n], y[..., n: 2 * n]
        out = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s, y[..., 2 * n:]], dim=-1)
    else:
        x1, x2 = y[..., 0: 2 * n: 2], y[..., 1: 2 * n: 2]
        out = torch.stack([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).flatten(-2)
        out = torch.cat([out, y[..., 2 * n:]], dim=-1)
    return out.to(x.dtype)


def rotary_axes(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    *,
    sections: Sequence[int],
    base: float = 10000.0,
    ladder: str = 'shared',
    layout: str = 'interleaved',
) -> tuple[torch.Tensor, torch.Tensor]:
    """Turn ``q`` ``[B, Hq, T, D]`` and ``k`` ``[B, Hk, T, D]`` by their
    tokens' positions.

    Args:
        q, k: bf16, fp16 or fp32, any strides; they may differ in their
            number of heads.
        positions: int32 or int64, ``[T, axes]`` or ``[B, T, axes]``; any
            values, negative ones included.
        sections: pairs of each axis, each at least 1, together at most
            ``D / 2`` (and 128).
        base: ratio of the ladder of frequencies, positive.
        ladder: ``'shared'`` or ``'per_axis'``.
        layout: ``'interleaved'`` or ``'halves'``.

    Returns:
        The turned ``(q, k)``, contiguous, in the inputs' dtype.  Gradients
        flow to ``q`` and ``k``.
    """
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f'q and k must be [B, H, T, D], got {tuple(q.shape)}, {tuple(k.shape)}')
    if (q.shape[0], *q.shape[2:]) != (k.shape[0], *k.shape[2:]):
        raise ValueError(f'q {tuple(q.shape)} and k {tuple(k.shape)} may differ in heads only')
    if q.dtype != k.dtype or (q.dtype not in _DTYPES and (q.is_cuda or q.dtype != torch.float64)):
        raise TypeError(f'q and k must share bf16, fp16 or fp32, got {q.dtype}, {k.dtype}')
    if not (q.device == k.device == positions.device):
        raise ValueError('q, k and positions must be on one device')
    sections = tuple(int(s) for s in sections)
    pairs = sum(sections)
    d = q.shape[-1]
    if not sections or min(sections) < 1 or 2 * pairs > d or pairs > MAX_PAIRS or d % 2 != 0:
        raise ValueError(f'sections {sections} do not fit a head of {d} (even, at most '
                         f'{MAX_PAIRS} pairs)')
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f'positions must be int32 or int64, got {positions.dtype}')
    b, t, axes = q.shape[0], q.shape[2], len(sections)
    if tuple(positions.shape) not in ((t, axes), (b, t, axes)):
        raise ValueError(f'positions must be {(t, axes)} or {(b, t, axes)}, got '
                         f'{tuple(positions.shape)}')
    if not (base > 0.0 and math.isfinite(base)):
        raise ValueError(f'base must be positive, got {base}')
    if ladder not in ('shared', 'per_axis') or layout not in ('interleaved', 'halves'):
        raise ValueError(f'unknown ladder {ladder!r} or layout {layout!r}')
    base = float(base)
    if _nat.use_native(q, k):
        return _nat.native().rotary_axes(  # type: ignore[union-attr]
            q, k, positions, _table(sections, base, ladder), layout == 'halves')
    rows = _rows(sections, base, ladder)
    return (_reference(q, positions, rows, layout == 'halves'),
            _reference(k, positions, rows, layout == 'halves'))
