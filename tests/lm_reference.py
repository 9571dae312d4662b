"""64-bit formulas of the decoder operators and how far a kernel that works
in 32 bits and rounds operands and results to ``dtype`` may be from them.

Every bound is a sum over the roundings of the computation, to first order:
``half`` is half a step of the stored type, ``2**-24`` that of the 32-bit
work, and sums of n terms carry n of them.
"""
from __future__ import annotations

import math

import torch


def half(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def smallest(dtype: torch.dtype) -> float:
    """Half the distance of the type's smallest values from each other."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def attention(q, k, v, *, window, sinks=0, lengths=None, q_start=None, scale=None, do=None):
    """(values, bounds) of out and, with ``do``, of dq, dk, dv."""
    dt = q.dtype
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    b, hq, tq, d = q.shape
    hk, tk = k.shape[1:3]
    g = hq // hk
    scale = d ** -0.5 if scale is None else scale
    u, tiny, w = half(dt), smallest(dt), 2.0 ** -24
    out = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    tol = [torch.zeros_like(x) for x in out]
    for i in range(b):
        n = tk if lengths is None else max(0, min(tk, int(lengths[i])))
        st = n - tq if q_start is None else int(q_start if isinstance(q_start, int) else q_start[i])
        p = torch.arange(tq) + st
        j = torch.arange(tk)
        gap = p[:, None] - j
        see = (gap >= 0) & ((gap < window) | (j < sinks)) & (p < n)[:, None] & (j < n)
        rows, keys = see.any(1), see.any(0)
        for h in range(hq):
            kh = torch.where(keys[:, None], k[i, h // g], 0.0)
            vh = torch.where(keys[:, None], v[i, h // g], 0.0)
            qh = torch.where(rows[:, None], q[i, h], 0.0)
            s = (qh @ kh.T * scale).masked_fill(~see, -math.inf)
            pr = torch.where(rows[:, None], torch.softmax(s, -1), 0.0).nan_to_num(0.0)
            o = pr @ vh
            # relative error of a probability: scores of d terms, the factor,
            # the difference to the maximum, 2^x
            size = (qh.abs() @ kh.abs().T * scale).amax(-1, keepdim=True) if tk else qh[:, :1]
            ka = w * (2 * (d + 16) * size + 16)
            acc = 2 * w * (see.sum(1, keepdim=True) + 16)
            A = pr @ vh.abs()
            few = tiny * see.sum(1, keepdim=True) * (vh.abs().max() if tk else 0.0)
            out[0][i, h] = o
            to = u * o.abs() + (u + 2 * ka + acc) * A + few + tiny
            tol[0][i, h] = torch.where(rows[:, None], to, 0.0)
            if do is None:
                continue
            gh = torch.where(rows[:, None], do.detach().cpu().double()[i, h], 0.0)
            dp, delta = gh @ vh.T, (gh * o).sum(-1, keepdim=True)
            ds = pr * (dp - delta)
            e_delta = (gh.abs() * to).sum(-1, keepdim=True)
            size_dp = gh.abs() @ vh.abs().T + (gh.abs() * o.abs()).sum(-1, keepdim=True)
            e_ds = u * ds.abs() + pr * e_delta + (4 * ka + 4 * w * (d + 16)) * pr * size_dp + tiny
            e_ds = torch.where(see, e_ds, 0.0)
            e_p = torch.where(see, (u + 4 * ka) * pr + tiny, 0.0)
            grow = 2 * w * (see.sum(0)[:, None] * g + 16)  # terms of a key's sums
            dq, dk, dv = scale * ds @ kh, scale * ds.T @ qh, pr.T @ gh
            out[1][i, h] = dq
            tol[1][i, h] = scale * (e_ds + acc * ds.abs()) @ kh.abs() + u * dq.abs() + tiny
            tol[1][i, h][~rows] = 0.0
            out[2][i, h // g] += dk
            out[3][i, h // g] += dv
            tol[2][i, h // g] += scale * (e_ds.T + grow * ds.abs().T) @ qh.abs()
            tol[3][i, h // g] += (e_p.T + grow * pr.T) @ gh.abs()
    tol[2] += u * out[2].abs() + tiny
    tol[3] += u * out[3].abs() + tiny
    if do is None:
        return out[:1], tol[:1]
    return out, tol


def rotary(x, positions, *, sections, base=10000.0, ladder='shared', layout='interleaved',
           sign=1.0):
    """(value, bound) of one operand."""
    dt = x.dtype
    y = x.detach().cpu().double()
    pos = positions.cpu().double()
    pos = pos if pos.dim() == 3 else pos[None]
    pairs = sum(sections)
    out, tol = y.clone(), torch.zeros_like(y)
    i = 0
    for a, n in enumerate(sections):
        for m in range(n):
            e = m / n if ladder == 'per_axis' else i / pairs
            ang = (sign * pos[..., a] * base ** -e)[:, None]
            f, s = (i, i + pairs) if layout == 'halves' else (2 * i, 2 * i + 1)
            x1, x2 = y[..., f], y[..., s]
            c, sn = ang.cos(), ang.sin()
            out[..., f], out[..., s] = x1 * c - x2 * sn, x2 * c + x1 * sn
            # the reduced angle keeps 24 bits of at most pi, its sine and
            # cosine a few units, two products and a sum: 16 roundings in all
            tol[..., f] = tol[..., s] = 2.0 ** -20 * (x1.abs() + x2.abs())
            i += 1
    moved = tol > 0
    return out, torch.where(moved, tol + half(dt) * out.abs() + smallest(dt), 0.0)


def distill(z, teacher, index, *, rest=None, temperature=1.0, reduction='mean', upstream=1.0):
    """(loss, bound, gradient, bound); rows by the definition, one at a time."""
    dt = z.dtype
    tau, u, w = temperature, half(z.dtype), 2.0 ** -24
    v, k = z.shape[-1], teacher.shape[-1]
    zz = z.detach().cpu().double().reshape(-1, v)
    tt, ii = teacher.cpu().double().reshape(-1, k), index.cpu().long().reshape(-1, k)
    rr = None if rest is None else rest.cpu().double().reshape(-1)
    n = zz.shape[0]
    loss, e_loss = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    grad, tol = torch.zeros_like(zz), torch.zeros_like(zz)
    counted = 0
    for a in range(n):
        has = ii[a] >= 0
        if not bool(has.any()):
            continue
        counted += 1
        idx = ii[a][has]
        x = zz[a] / tau
        logq = torch.log_softmax(x, 0)
        lt = tt[a][has] / tau
        if rr is not None:
            lt = torch.cat([lt, rr[a][None]])
        logp = torch.log_softmax(lt, 0)
        m = len(idx)
        p = logp.exp()
        size = x.abs().max() + lt[lt > -math.inf].abs().max()
        e = w * (8 * size + 2 * math.ceil(v / 256) + 64)  # of a log-probability
        terms = p[:m] * (logp[:m] - logq[idx])
        terms = terms[p[:m] > 0]
        mag = (p[:m] * (logp[:m].abs() + logq[idx].abs()))[p[:m] > 0].sum()
        loss[a] = terms.sum()
        q = logq.exp()
        inside = torch.zeros(v, dtype=torch.bool)
        inside[idx] = True
        gr, mass = q.clone(), q.clone()
        if rr is not None and p[m] > 0:
            log_r = torch.logsumexp(logq[~inside], 0) if bool((~inside).any()) else torch.tensor(-math.inf)
            loss[a] += p[m] * (logp[m] - log_r)
            mag = mag + p[m] * (logp[m].abs() + log_r.abs())
            ratio = p[m] / log_r.exp()
            gr[~inside] = q[~inside] * (1 - ratio)
            mass[~inside] = q[~inside] * (1 + ratio)
        gr.scatter_add_(0, idx, -p[:m])
        mass.scatter_add_(0, idx, p[:m])
        e_loss[a] = 4 * e * (1 + mag)
        grad[a], tol[a] = tau * gr, tau * 4 * e * mass
    loss, e_loss = loss * tau ** 2, e_loss * tau ** 2
    f = 1.0 / max(counted, 1) if reduction == 'mean' else 1.0
    up = torch.as_tensor(upstream).cpu().double().reshape(-1, 1)
    grad, tol = grad * f * up, tol * f * up.abs()
    tol = torch.where(grad != 0.0, tol + u * grad.abs() + smallest(dt), tol)
    if reduction != 'none':
        loss, e_loss = loss.sum() * f, e_loss.sum() * f + 2.0 ** -24 * loss.sum().abs() * f
    else:
        loss, e_loss = loss.reshape(z.shape[:-1]), e_loss.reshape(z.shape[:-1])
    return loss, e_loss, grad.reshape(z.shape), tol.reshape(z.shape)


def check(name: str, got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor) -> None:
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f'{name}: not finite'
    over = (got - want).abs() - tol
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0.0, f'{name}: {worst:.3g} over its bound at {int(over.argmax())} of {over.numel()}'
