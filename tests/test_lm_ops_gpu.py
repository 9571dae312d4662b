"""Decoder operators on the GPU against 64 bits, at the sizes, masks, strides
and uses where a kernel can go wrong."""
from __future__ import annotations

import pytest
import torch
import torch.utils.checkpoint

from distributed_kfac_pytorch_amd.ops.attention import window_attention
from distributed_kfac_pytorch_amd.ops.distill import topk_distill_loss
from distributed_kfac_pytorch_amd.ops.rotary import rotary_axes
from tests import lm_reference as ref
from tests.test_lm_ops import lowest_case

pytestmark = pytest.mark.gpu

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def rand(dev, *shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


# ------------------------------------------------------------- attention
ATTN = [
    # b, hq, hk, tq, tk, d, window, sinks, lengths, start
    (1, 1, 1, 1, 1, 8, 1, 0, None, None),
    (2, 2, 2, 33, 33, 16, 5, 0, None, None),
    (1, 2, 1, 64, 64, 64, 64, 0, None, None),
    (1, 2, 1, 65, 65, 64, 7, 2, None, None),
    (2, 3, 1, 129, 129, 32, 40, 5, None, None),
    (1, 4, 2, 200, 200, 40, 1, 1, None, None),
    (1, 2, 2, 257, 257, 96, 64, 33, None, None),
    (1, 5, 1, 130, 130, 104, 50, 0, None, None),
    (1, 2, 1, 191, 191, 128, 500, 3, None, None),
    (3, 4, 2, 100, 100, 24, 17, 3, [100, 1, 64], 0),
    (3, 2, 1, 70, 70, 64, 9, 1, [70, 0, 33], 0),
    (2, 2, 1, 40, 150, 72, 30, 4, None, None),       # a chunk behind a cache
    (2, 2, 1, 40, 150, 72, 30, 4, [150, 20], None),  # fewer tokens than rows
    (2, 2, 1, 40, 50, 16, 30, 4, None, -20),
    (2, 2, 1, 40, 50, 16, 30, 4, None, [30, -1000000000]),
    (1, 2, 1, 20, 0, 16, 4, 1, None, None),
    (1, 2, 1, 300, 300, 16, 3, 170, None, None),     # sinks over two key blocks
    (1, 2, 1, 1500, 1500, 16, 30, 2, None, None),    # far rows in several chunks
    (1, 4, 1, 700, 700, 64, 20, 140, [650], 0),
]


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('n', [2, 60])
def test_attention_gradients_between_two_values_one_step_apart(cuda, dtype, n):
    """The output lies halfway between two numbers of its type: gradients that
    go by the rounded output are all wrong, those of the formula are exact.
    Short windows, whose few keys do not average that out."""
    dt, d = DTYPES[dtype], 64
    eps = torch.finfo(dt).eps
    q = torch.zeros(1, 1, 2, d, dtype=dt, device=cuda, requires_grad=True)
    k = torch.zeros(1, 1, n, d, dtype=dt, device=cuda)
    k[:, :, :2] = rand(cuda, 1, 1, 2, d, seed=1, dtype=dt)
    k[:, :, -2:] = k[:, :, :2]
    v = torch.ones(1, 1, n, d, dtype=dt, device=cuda)
    v[:, :, 0::2] += eps
    out = window_attention(q, k, v, window=n)
    (dq,) = torch.autograd.grad(out[:, :, 1].sum() / eps, q)
    # P = 1 / n, dP - delta = +-d / 2, so dq = d ** -0.5 / n * d / 2 * sum of
    # +-k; one rounding (dS is a power of two, or rounds once more by n).  dP
    # and delta are each a sum of d terms of 1 / eps in 32 bits, off by
    # d * 2^-24 of d / eps at most: in fp32 that is more than their difference.
    sign = torch.where(torch.arange(n, device=cuda) % 2 == 0, 1.0, -1.0).double()
    terms = sign[:, None] * k[0, 0].double()
    want = d ** -0.5 / n * d / 2 * terms.sum(0)
    sums = 2 * d * 2.0 ** -24 * d / eps
    tol = ((2 * eps + 2.0 ** -12) * d / 2 + sums) * d ** -0.5 / n * terms.abs().sum(0)
    ref.check('dq', dq[0, 0, 1], want.cpu(), tol.cpu())


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('d', [16, 64, 128])
def test_a_token_that_sees_itself_alone(cuda, d, dtype):
    dt = DTYPES[dtype]
    q, k, v, do = (rand(cuda, 2, 4, 90, d, seed=s, dtype=dt) for s in range(4))
    for x in (q, k, v):
        x.requires_grad_()
    out = window_attention(q, k, v, window=1)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    # powers of 2 are off by the scores' 32-bit rounding, 40 * 2^-24: below half
    # a step of the 16-bit types, which give the values back as they are
    off = 2.0 ** -18 if dtype == 'fp32' else 0.0
    for got, want in ((out, v), (dv, do)):
        assert bool(((got - want).abs() <= off * want.abs()).all())
    assert not bool(dq.any()) and not bool(dk.any())


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('d', [24, 64, 88, 128])
def test_attention_with_many_heads(cuda, d, dtype):
    """Enough blocks that no two waves share keys; sinks over two groups of
    keys, far rows in chunks."""
    dt = DTYPES[dtype]
    q, k, v, do = (rand(cuda, 2, 27, 600, d, seed=s, dtype=dt) for s in range(4))
    for x in (q, k, v):
        x.requires_grad_()
    out = window_attention(q, k, v, window=70, sinks=35)
    got = (out, *torch.autograd.grad(out, (q, k, v), do))
    want, tol = ref.attention(q, k, v, window=70, sinks=35, do=do)
    for name, *x in zip(('out', 'dq', 'dk', 'dv'), got, want, tol):
        ref.check(name, *x)


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('case', ATTN, ids=lambda c: '-'.join(str(x) for x in c[:8]))
def test_attention_matches_formula(cuda, case, dtype):
    b, hq, hk, tq, tk, d, window, sinks, lengths, start = case
    dt = DTYPES[dtype]
    q, k, v, do = (rand(cuda, b, h, t, d, seed=s, dtype=dt) for s, (h, t) in
                   enumerate([(hq, tq), (hk, tk), (hk, tk), (hq, tq)]))
    ln = None
    if lengths is not None:
        ln = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        for i, n in enumerate(lengths):
            k[i, :, n:] = float('nan')
            v[i, :, n:] = float('inf')
    st = torch.tensor(start, dtype=torch.int32, device=cuda) if isinstance(start, list) else start
    conf = dict(window=window, sinks=sinks, lengths=ln, q_start=st)
    want, tol = ref.attention(q, k, v, do=do, **conf)
    x = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention(*x, **conf)
    got = [out, *torch.autograd.grad(out, x, do)]
    for name, g, w, t in zip(('out', 'dq', 'dk', 'dv'), got, want, tol):
        ref.check(name, g, w, t)
    with torch.no_grad():
        assert torch.equal(window_attention(*x, **conf), out)


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('d', [16, 64, 128])
def test_keys_that_no_row_sees_may_hold_anything(cuda, d, dtype):
    """A chunk of rows behind a cache, whose older entries are stale."""
    dt = DTYPES[dtype]
    q, do = (rand(cuda, 1, 4, 4, d, seed=s, dtype=dt) for s in range(2))
    k, v = (rand(cuda, 1, 2, 64, d, seed=s, dtype=dt) for s in (2, 3))
    conf = dict(window=8, sinks=3)
    x = [t.requires_grad_() for t in (q, k, v)]
    want = [window_attention(*x, **conf)]
    want += torch.autograd.grad(want[0], x, do)
    with torch.no_grad():
        for bad, at in ((float('nan'), 40), (float('inf'), 52), (float('nan'), 3)):
            k[:, :, at] = bad
            v[:, :, at] = bad
    got = [window_attention(*x, **conf)]
    got += torch.autograd.grad(got[0], x, do)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('d', [16, 64, 128])
def test_rows_of_padding_may_hold_anything(cuda, d, dtype):
    dt = DTYPES[dtype]
    q, k, v, do = (rand(cuda, 2, h, 130, d, seed=s, dtype=dt) for s, h in enumerate((4, 2, 2, 4)))
    conf = dict(window=40, sinks=1, lengths=torch.tensor([130, 71], dtype=torch.int32, device=cuda),
                q_start=0)
    x = [t.requires_grad_() for t in (q, k, v)]
    want = [window_attention(*x, **conf)]
    want += torch.autograd.grad(want[0], x, do)
    with torch.no_grad():
        for t in (q, k, v, do):
            t[1, :, 71:] = float('nan')
    got = [window_attention(*x, **conf)]
    got += torch.autograd.grad(got[0], x, do)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('tq, hq', [(1, 1), (1, 300), (70, 1)])
def test_fp16_rows_of_small_probabilities(cuda, tq, hq):
    """4096 keys of 2^-20.6 each beside one of 1, which has no value: the
    output is their sum.  Off by the rounding of the probabilities and of the
    output, half a step of 2^-11 each, and of the scores in 32 bits."""
    n, d = 4097, 64
    q = torch.ones(1, 1, tq, d, dtype=torch.half, device=cuda)
    k = torch.zeros(1, 1, n, d, dtype=torch.half, device=cuda)
    k[:, :, 0] = 1.785
    v = torch.ones_like(k)
    v[:, :, 0] = 0.0
    want = ref.attention(q, k, v, window=n)[0][0]
    # many heads: one block goes over all keys of a row
    out = window_attention(*(x.expand(1, hq, -1, d) for x in (q, k, v)), window=n)
    err = ((out.cpu().double() - want).abs() / want).max()
    assert float(err) <= 2.0 ** -10 + 2.0 ** -16, float(err)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('d', [16, 64, 96, 128])
@pytest.mark.parametrize('heads', [1, 30])
def test_short_windows_round_their_gradients_once(cuda, heads, d, dtype):
    """8 keys of probability 1/8 each (queries of 0, or keys of 0), so that
    probabilities and outputs are exact in 32 bits: what is left of the
    gradients' error is their own rounding, half a step, and terms of second
    order: what o's rounding took away is itself rounded (u^2 of o, or half of
    fp16's smallest step), and so is what the rounding of P (dP - delta) did."""
    dt, n, rows, w = DTYPES[dtype], 263, 256, 8
    u, tiny = ref.half(dt), ref.smallest(dt)
    x, v = (rand(cuda, 1, heads, t, d, seed=s) for s, t in ((0, n), (1, n)))
    do = rand(cuda, 1, heads, rows, d, seed=2, dtype=dt)
    v, some = v.to(dt), (x + 16.0).to(dt)
    for name in ('dq', 'dk'):
        q = torch.zeros_like(do) if name == 'dq' else some[:, :, :rows].contiguous()
        k = torch.zeros_like(some) if name == 'dk' else some
        leaf = (q if name == 'dq' else k).requires_grad_()
        (got,) = torch.autograd.grad(window_attention(q, k, v, window=w), leaf, do)
        V, D, K, Q = (y.detach().cpu().double() for y in (v, do, k, q))
        see = (torch.arange(n) >= torch.arange(rows)[:, None]) & (
            torch.arange(n) < torch.arange(rows)[:, None] + w)
        p = (see / w).double()
        o = p @ V
        dp, delta = D @ V.transpose(2, 3), (D * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        size = D.abs() @ V.abs().transpose(2, 3) + (D.abs() * o.abs()).sum(-1, keepdim=True)
        e = p * ((D.abs() * (u * u * o.abs() + tiny)).sum(-1, keepdim=True)
                 + 2.0 ** -24 * 4 * (d + 16) * size) + u * u * ds.abs()
        f = d ** -0.5
        if name == 'dq':
            want, off = f * ds @ K, f * (e + 2.0 ** -20 * ds.abs()) @ K.abs()
        else:
            want = f * ds.transpose(2, 3) @ Q
            off = f * (e + 2.0 ** -20 * ds.abs()).transpose(2, 3) @ Q.abs()
        # half a step of a number of this size (frexp: below 2^exponent)
        half_step = u * torch.ldexp(torch.ones(()).double(), torch.frexp(want.abs() + off)[1] - 1)
        ref.check(name, got, want, off + torch.maximum(half_step, torch.tensor(tiny).double()))


def _signs(dev, n, d):
    """[1, 1, n, d] of rows +1, -1, +1, .."""
    x = torch.where(torch.arange(n, device=dev) % 2 == 0, 1.0, -1.0).half()
    return x[:, None].expand(n, d)[None, None].contiguous()


def test_fp16_small_gradients_of_queries(cuda):
    """4096 products P (dP - delta) of +-2^-26, below fp16, whose sum is not:
    all numbers are powers of two and the answer exact."""
    n, d = 4096, 64
    q = torch.zeros(1, 1, 1, d, dtype=torch.half, device=cuda, requires_grad=True)
    kv = _signs(cuda, n, d)
    do = torch.full((1, 1, 1, d), 2.0 ** -20, dtype=torch.half, device=cuda)
    (dq,) = torch.autograd.grad(window_attention(q, kv, kv, window=n), q, do)
    assert bool((dq == 2.0 ** -17).all()), dq[0, 0, 0, :4]


@pytest.mark.parametrize('d', [64, 128])
def test_fp16_small_gradients_of_keys(cuda, d):
    """512 rows of 4096 equally weighted keys each: products of +-2^-32 d."""
    n, rows = 4096, 512
    q = torch.ones(1, 1, rows, d, dtype=torch.half, device=cuda)
    k = torch.ones(1, 1, n + rows, d, dtype=torch.half, device=cuda, requires_grad=True)
    v = _signs(cuda, n + rows, d)
    do = torch.full_like(q, 2.0 ** -20)
    (dk,) = torch.autograd.grad(window_attention(q, k, v, window=n, scale=0.125), k, do)
    # keys that all rows see; factor 1/8 on the sum
    assert torch.equal(dk[:, :, rows:n], v[:, :, rows:n] * (d * 2.0 ** -26)), dk[0, 0, rows]


def test_fp16_small_gradients_of_values(cuda):
    """Keys of probability 2^-27 or less under large upstream gradients: off
    by the rounding of the probabilities and of the result, 2^-11 each, and of
    the scores (27 times a few 2^-24).  The last keys' results lie under 2^-14
    (one row: 2^-17), where fp16 has a step of 2^-24 and half of it, 2^-25, is
    no 2^-11 of the value."""
    n, d = 1024, 64
    q = torch.ones(1, 1, n, d, dtype=torch.half, device=cuda)
    k = torch.zeros_like(q)
    k[:, :, 0] = 2.34
    v = torch.zeros_like(q).requires_grad_()
    do = torch.full_like(q, 2.0 ** 10)
    (dv,) = torch.autograd.grad(window_attention(q, k, v, window=n), v, do)
    want = ref.attention(q, k, v, window=n, do=do)[0][3][0, 0, 1:]
    ref.check('dv', dv[0, 0, 1:], want, (2.0 ** -10 + 2.0 ** -16) * want + 2.0 ** -25)


def test_fp16_large_gradients(cuda):
    """P (dP - delta) of 2^18, behind fp16's end, under gradients that are
    not: powers of two once more."""
    n, d = 70, 64
    q = torch.zeros(1, 1, n, d, dtype=torch.half, device=cuda, requires_grad=True)
    v = _signs(cuda, n, d)
    k = (v / 64).requires_grad_()
    do = torch.full_like(q, 2.0 ** 13)
    dq, dk = torch.autograd.grad(window_attention(q, k, v, window=2), (q, k), do)
    assert bool((dq[0, 0, 1:] == 2.0 ** 10).all()), dq[0, 0, :, 0]
    assert not bool(dk.any())


@pytest.mark.parametrize('d', [16, 64, 128])
@pytest.mark.parametrize('factor', [2.0 ** -7, 2.0 ** 9])
def test_fp16_gradients_follow_the_upstream_scale(cuda, factor, d):
    """A power of two on the upstream gradient is one on every gradient, bit
    for bit, as long as the results are normal numbers of fp16.  2^-14 itself
    is left out: 2^-14 (1 - 2^-11) rounds up to it from below, where the step
    is 2^-24, and is a number of its own at any other scale."""
    q, k, v, do = (rand(cuda, 1, h, 700, d, seed=s).half() for s, h in enumerate((4, 2, 2, 4)))
    do = torch.where(do.abs() < 2.0 ** -7, 0.0, do)
    x = [t.requires_grad_() for t in (q, k, v)]
    got = []
    for f in (1.0, factor):
        got.append(torch.autograd.grad(window_attention(*x, window=600, sinks=4), x, do * f))
    for a, b in zip(*got):
        a, b = a.float(), b.float()
        keep = (a.abs() > 2.0 ** -14) & (b.abs() > 2.0 ** -14)
        assert float(keep.float().mean()) > 0.5
        assert torch.equal(a[keep] * factor, b[keep])


def test_fp16_gradients_beside_an_infinite_one(cuda):
    """An infinite upstream gradient reaches its own sequence and head."""
    q, k, v, do = (rand(cuda, 2, 2, 90, 32, seed=s).half().requires_grad_() for s in range(4))
    x, do = (q, k, v), do.detach()
    want = torch.autograd.grad(window_attention(*x, window=20), x, do)
    do[0, 1, 50, 3] = float('inf')
    got = torch.autograd.grad(window_attention(*x, window=20), x, do)
    for a, b in zip(got, want):
        assert torch.equal(a[1], b[1]) and torch.equal(a[0, 0], b[0, 0])
        assert not bool(a[0, 1].isfinite().all())


@pytest.mark.parametrize('dtype', sorted(DTYPES))
def test_attention_at_the_smallest_scale(cuda, dtype):
    """Scores of 0: the mean over the keys that a row sees.  Off by half a
    step of the output, and of the probabilities' type for each term."""
    dt = DTYPES[dtype]
    q, k, v = (rand(cuda, 1, 2, 100, 64, seed=s, dtype=dt) for s in range(3))
    out = window_attention(q, k, v, window=30, scale=2.0 ** -126)
    want, tol = ref.attention(q, k, v, window=30, scale=2.0 ** -126)
    ref.check('out', out, want[0], tol[0])


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('window', [8, 200])
def test_attention_with_offloaded_tensors(cuda, window, dtype):
    """Saved-tensor hooks hand tensors back contiguous, whatever they were:
    the output lies [B, T, H, D] in memory, the operands are slices."""
    b, t, h, d = 2, 90, 3, 32
    qkv = rand(cuda, b, t, h, 3 * d, seed=1, dtype=DTYPES[dtype]).requires_grad_()
    do = rand(cuda, b, h, t, d, seed=2, dtype=DTYPES[dtype])

    def call():
        q, k, v = qkv.permute(0, 2, 1, 3).split(d, dim=-1)
        return window_attention(q, k, v, window=window, sinks=2)

    (want,) = torch.autograd.grad(call(), qkv, do)
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        out = call()
    assert torch.equal(torch.autograd.grad(out, qkv, do)[0], want)


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('hq, hk', [(2, 2), (6, 2)])
def test_attention_to_a_single_key_of_any_stride(cuda, dtype, hq, hk):
    """[B, H, D] made [B, H, 1, D] with a token stride of 1 or 0: it says
    nothing, and nothing goes by it."""
    dt, b, d = DTYPES[dtype], 3, 40
    q, k, v, do = (rand(cuda, b, h, d, seed=s, dtype=dt) for s, h in enumerate((hq, hk, hk, hq)))
    want, tol = ref.attention(*(x[:, :, None] for x in (q, k, v)), window=4, do=do[:, :, None])
    for view in (lambda x: x.unsqueeze(-1).transpose(2, 3),
                 lambda x: x.as_strided((*x.shape[:2], 1, d), (*x.stride()[:2], 0, 1))):
        x = [view(t).requires_grad_() for t in (q, k, v)]
        out = window_attention(*x, window=4)
        for name, *y in zip(('out', 'dq', 'dk', 'dv'),
                            (out, *torch.autograd.grad(out, x, view(do))), want, tol):
            ref.check(name, *y)


TOKEN = [
    # b, hq, hk, tq, tk, d, window, sinks, lengths
    (1, 2, 2, 1, 1, 64, 1, 0, None),
    (3, 8, 2, 1, 300, 64, 40, 4, [300, 7, 0]),
    (2, 8, 1, 1, 2100, 128, 2100, 0, None),
    (2, 5, 1, 1, 1999, 80, 700, 3, [1999, 640]),
    (1, 4, 2, 3, 5000, 32, 5000, 0, None),
    (1, 3, 3, 1, 4097, 16, 64, 200, None),
    (1, 40, 1, 1, 3001, 64, 3001, 0, None),
    (1, 40, 1, 7, 3001, 64, 1000, 10, None),
]


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('case', TOKEN, ids=lambda c: '-'.join(str(x) for x in c[:8]))
def test_attention_tokens_match_formula(cuda, case, dtype):
    b, hq, hk, tq, tk, d, window, sinks, lengths = case
    dt = DTYPES[dtype]
    q, k, v = (rand(cuda, b, h, t, d, seed=s, dtype=dt) for s, (h, t) in
               enumerate([(hq, tq), (hk, tk), (hk, tk)]))
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda)
    for i in range(b):
        n = tk if lengths is None else lengths[i]
        k[i, :, n:] = float('nan')
        v[i, :, n:] = float('nan')
        if tq == 1 and n - window > sinks:  # what no row sees any more
            k[i, :, sinks:n - window] = float('inf')
            v[i, :, sinks:n - window] = float('nan')
    conf = dict(window=window, sinks=sinks, lengths=ln)
    want, tol = ref.attention(q, k, v, **conf)
    ref.check('out', window_attention(q, k, v, **conf), want[0], tol[0])
    # the same rows with a backward pass to follow
    out = window_attention(q.requires_grad_(), k, v, **conf)
    ref.check('out', out, want[0], tol[0])


@pytest.mark.parametrize('dtype', ['bf16', 'fp32'])
def test_attention_strides_and_scale(cuda, dtype):
    dt = DTYPES[dtype]
    b, h, t, d = 2, 3, 77, 32
    qkv = rand(cuda, b, t, h, 3 * d, seed=1, dtype=dt).requires_grad_()
    do = rand(cuda, b, h, d, t, seed=2, dtype=dt).transpose(2, 3)  # rows not contiguous
    q, k, v = qkv.permute(0, 2, 1, 3).split(d, dim=-1)
    conf = dict(window=20, sinks=2, scale=0.31)
    want, tol = ref.attention(q, k, v, do=do, **conf)
    out = window_attention(q, k, v, **conf)
    assert out.transpose(1, 2).is_contiguous()
    (g,) = torch.autograd.grad(out, qkv, do)
    g = g.permute(0, 2, 1, 3).split(d, dim=-1)
    for name, x, w, e in zip(('out', 'dq', 'dk', 'dv'), (out, *g), want, tol):
        ref.check(name, x, w, e)
    # rows at odd addresses, and one key head shared without a copy
    odd = torch.empty(b * t * h * d + 3, dtype=dt, device=cuda)[3:].view(b, h, t, d)
    odd.copy_(q.detach())
    kk, vv = (x.detach()[:, :1].expand(b, h, t, d) for x in (k, v))
    want, tol = ref.attention(odd, kk, vv, do=do, **conf)
    x = [odd.requires_grad_(), kk.requires_grad_(), vv.requires_grad_()]
    out = window_attention(*x, **conf)
    for name, g2, w, e in zip(('out', 'dq', 'dk', 'dv'), (out, *torch.autograd.grad(out, x, do)),
                              want, tol):
        ref.check(name, g2, w, e)


def test_attention_differences(cuda):
    """The gradient's component along a direction, by central differences of
    an fp32 call: step e has an error of e^2 / 6 times the third derivative
    (of order 1 for inputs of order 1) and 2^-24 |f| / e of rounding."""
    b, h, t, d = 1, 2, 70, 16
    x = [rand(cuda, b, h, t, d, seed=s) * 0.5 for s in range(3)]
    do = rand(cuda, b, h, t, d, seed=7)
    along = [rand(cuda, b, h, t, d, seed=10 + s) for s in range(3)]

    def f(a):
        return (window_attention(*a, window=9, sinks=2).double() * do.double()).sum()

    leaves = [a.clone().requires_grad_() for a in x]
    grads = torch.autograd.grad(f(leaves), leaves)
    for i in range(3):
        norm = float(along[i].double().norm())
        step = 1e-2 / norm
        lo, hi = ([a + s * step * w if j == i else a for j, (a, w) in enumerate(zip(x, along))]
                  for s in (-1, 1))
        want = float((f(hi) - f(lo)) / (2 * step)) / norm
        got = float((grads[i].double() * along[i].double()).sum()) / norm
        size = float(grads[i].double().norm())
        assert abs(got - want) <= 1e-2 * size / norm ** 0.5 + 2e-3, (i, got, want)


# --------------------------------------------------------------- rotary
@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('layout', ['interleaved', 'halves'])
@pytest.mark.parametrize('b, hq, hk, t, d, sections, ladder', [
    (1, 1, 1, 1, 2, (1,), 'shared'),
    (2, 3, 3, 17, 64, (32,), 'shared'),
    (2, 4, 1, 33, 128, (16, 24, 24), 'shared'),
    (3, 2, 2, 5, 40, (4, 3, 2), 'per_axis'),
    (1, 2, 1, 300, 18, (5, 4), 'per_axis'),
    (2, 5, 2, 1, 80, (8, 8), 'shared'),
    (1, 2, 2, 9, 256, (128,), 'shared'),
    (2, 2, 1, 0, 16, (8,), 'shared'),
])
def test_rotary_matches_formula(cuda, dtype, layout, b, hq, hk, t, d, sections, ladder):
    dt = DTYPES[dtype]
    # views whose rows are not next to each other
    q = rand(cuda, b, t, hq, d, seed=1, dtype=dt).transpose(1, 2).requires_grad_()
    k = rand(cuda, b, hk, t, d + 2, seed=2, dtype=dt)[..., :d].requires_grad_()
    gq, gk = rand(cuda, b, hq, t, d, seed=3, dtype=dt), rand(cuda, b, hk, t, d, seed=4, dtype=dt)
    g = torch.Generator().manual_seed(5)
    conf = dict(sections=sections, ladder=ladder, layout=layout)
    for pos in (torch.randint(-5, 4096, (t, len(sections)), generator=g, dtype=torch.int32),
                torch.randint(2 ** 30, 2 ** 31, (b, t, len(sections)), generator=g)):
        pos = pos.to(cuda)
        out = rotary_axes(q, k, pos, **conf)
        grads = torch.autograd.grad(out, (q, k), (gq, gk))
        for name, x, got in (('q', q, out[0]), ('k', k, out[1])):
            ref.check(name, got, *ref.rotary(x, pos, **conf))
        for name, x, got in (('dq', gq, grads[0]), ('dk', gk, grads[1])):
            ref.check(name, got, *ref.rotary(x, pos, sign=-1.0, **conf))


def test_rotary_passes_the_rest_through(cuda):
    q = rand(cuda, 1, 2, 3, 32)
    q[..., 20:] = float('inf')
    q[0, 0, 0, 31] = float('nan')
    pos = torch.arange(3, device=cuda)[:, None]
    for layout in ('interleaved', 'halves'):
        out, _ = rotary_axes(q, q, pos, sections=(10,), layout=layout)
        assert torch.equal(out[..., 20:].isnan(), q[..., 20:].isnan())
        assert torch.equal(out[..., 20:].isinf(), q[..., 20:].isinf())
        assert bool(out[..., :20].isfinite().all())


# -------------------------------------------------------------- distill
def _teacher(dev, n, v, k, tau, rest, seed):
    g = torch.Generator().manual_seed(seed)
    full = torch.randn(n, v, generator=g) * 2.5
    t, i = full.topk(k, dim=-1)
    r = (full / tau).scatter(-1, i, float('-inf')).logsumexp(-1) if rest else None
    return t.to(dev), i.to(dev), None if r is None else r.to(dev)


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('n, v, k, tau, reduction', [
    (1, 1, 1, 1.0, 'mean'),
    (3, 7, 2, 1.0, 'sum'),
    (5, 8, 8, 2.0, 'mean'),
    (4, 255, 5, 0.5, 'none'),
    (6, 512, 64, 2.0, 'mean'),
    (9, 1001, 100, 1.0, 'none'),
    (2, 33278, 20, 1.5, 'mean'),
    (3, 5003, 1024, 1.0, 'sum'),
    (2100, 130, 4, 1.0, 'mean'),      # one block a row
])
def test_distill_matches_formula(cuda, dtype, rest, n, v, k, tau, reduction):
    dt = DTYPES[dtype]
    z = (rand(cuda, n, v, seed=n) * 2).to(dt).requires_grad_()
    t, i, r = _teacher(cuda, n, v, k, tau, rest, v)
    if rest and k == v:
        r = None  # nothing is left
    up = rand(cuda, n, seed=9) if reduction == 'none' else torch.tensor(0.37, device=cuda)
    loss = topk_distill_loss(z, t, i, teacher_rest=r, temperature=tau, reduction=reduction)
    assert loss.dtype == torch.float32
    want = ref.distill(z, t, i, rest=r, temperature=tau, reduction=reduction, upstream=up)
    ref.check('loss', loss, *want[:2])
    tol = want[3]
    if n >= 256 and dtype != 'fp16':
        # the forward stored the gradient, and the factor 0.37 is multiplied
        # into what it stored: (1 + u)(1 + u) - 1 = 2 u + u^2, of which the
        # bound holds one u
        tol = tol + (ref.half(dt) + ref.half(dt) ** 2) * want[2].abs()
    ref.check('dz', *torch.autograd.grad(loss, z, up), want[2], tol)
    with torch.no_grad():
        assert torch.equal(topk_distill_loss(z, t, i, teacher_rest=r, temperature=tau,
                                             reduction=reduction), loss)


@pytest.mark.parametrize('dtype', ['bf16', 'fp32'])
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('v, k', [(5, 2), (8 * 1024, 7), (8 * 1024 + 9, 64), (33278, 20), (60001, 3)])
def test_distill_rows_in_registers(cuda, dtype, rest, v, k):
    """256 rows and more: the forward writes the gradient.  One upstream
    factor is 1, one is not, and a second backward pass of the same graph
    computes its own."""
    n = 256 if v < 9000 else 257
    dt = DTYPES[dtype]
    z = (rand(cuda, n, v, seed=n) * 2).to(dt).requires_grad_()
    t, i, r = _teacher(cuda, n, v, k, 2.0, rest, v)
    i[3] = -1
    i[7, k - 1] = -5
    loss = topk_distill_loss(z, t, i, teacher_rest=r, temperature=2.0, weight=0.75)
    want = [0.75 * x for x in ref.distill(z, t, i, rest=r, temperature=2.0)]
    one = torch.ones((), device=cuda)
    ref.check('loss', loss, *want[:2])
    (first,) = torch.autograd.grad(loss, z, one, retain_graph=True)
    kept = first.clone()
    ref.check('dz', first, want[2], want[3])
    (again,) = torch.autograd.grad(loss, z, one)
    assert again.data_ptr() != first.data_ptr()
    ref.check('dz again', again, want[2], want[3])
    # multiplied afterwards: the gradient is rounded once more
    loss = topk_distill_loss(z, t, i, teacher_rest=r, temperature=2.0) * 0.75
    (g,) = torch.autograd.grad(loss, z, one)
    ref.check('dz', g, want[2], want[3] + 2 * ref.half(dt) * want[2].abs())
    assert torch.equal(first, kept)
    summed = topk_distill_loss(z, t, i, teacher_rest=r, temperature=2.0, reduction='sum')
    want = ref.distill(z, t, i, rest=r, temperature=2.0, reduction='sum')
    ref.check('sum', summed, *want[:2])
    ref.check('dz of sum', *torch.autograd.grad(summed, z), *want[2:])


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('k', [100, 512, 513, 1024])
@pytest.mark.parametrize('dtype, v', [('fp32', 32000), ('bf16', 65536)])
def test_distill_many_entries_in_registers(cuda, dtype, v, k, rest):
    """Up to twice as many entries as the block has threads, with columns that
    several entries name, on one side of the 512th and across it."""
    n, dt = 256, DTYPES[dtype]
    z = (rand(cuda, n, v, seed=n) * 2).to(dt).requires_grad_()
    t, i, r = _teacher(cuda, n, v, k, 2.0, rest, v)
    i[2, 0] = i[2, k - 1]
    i[5, k - 3] = i[5, k - 1] = i[5, 1]
    i[9] = -1
    i[11, k // 2:] = -1
    loss = topk_distill_loss(z, t, i, teacher_rest=r, temperature=2.0, reduction='sum')
    want = ref.distill(z, t, i, rest=r, temperature=2.0, reduction='sum')
    ref.check('loss', loss, *want[:2])
    ref.check('dz', *torch.autograd.grad(loss, z), *want[2:])


def test_distill_rows_in_registers_alone(cuda):
    """Bad rows, views and no rows that count, where the forward writes the
    gradient."""
    n, v, k = 300, 1030, 5
    full = rand(cuda, n, v + 5, seed=2, dtype=torch.bfloat16)
    view = full[:, 3:v + 3].requires_grad_()      # rows at odd addresses
    t, i, r = _teacher(cuda, n, v, k, 1.0, True, 5)
    want = ref.distill(view, t, i, rest=r)
    loss = topk_distill_loss(view, t, i, teacher_rest=r)
    ref.check('loss', loss, *want[:2])
    ref.check('dz', *torch.autograd.grad(loss, view), *want[2:])
    i[4, 1] = i[4, 2]
    i[5, 0] = v
    z = view.detach().clone()
    z[6, 100] = float('nan')
    z[7] = float('-inf')
    z.requires_grad_()
    (g,) = torch.autograd.grad(topk_distill_loss(z, t, i, teacher_rest=r), z)
    bad = g.isnan().any(dim=-1)
    assert bad[5:8].all() and int(bad.sum()) == 3
    loss = topk_distill_loss(z, t, torch.full_like(i, -1), teacher_rest=r)
    (g,) = torch.autograd.grad(loss, z)
    assert float(loss.detach()) == 0.0 and bool((g == 0).all())


def test_distill_stored_gradient_and_saved_tensor_hooks(cuda):
    """The gradient that the forward wrote goes through the hooks: moved to the
    host and back, to other strides and odd addresses, or made anew by a
    checkpoint, the answer is the same, and a second backward pass works."""
    n, v = 256, 1036
    z = rand(cuda, n, v, seed=1).requires_grad_()
    t, i, _ = _teacher(cuda, n, v, 3, 1.0, False, 1)
    one = torch.ones((), device=cuda)
    (want,) = torch.autograd.grad(topk_distill_loss(z, t, i), z, one)

    def odd(x):
        if x.dim() < 2:
            return x.cuda()
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=cuda)[1:].view(x.shape)
        return y.copy_(x)

    def strided(x):
        return x.cuda().transpose(-1, -2).contiguous().transpose(-1, -2) if x.dim() > 1 else x.cuda()

    for unpack in (torch.Tensor.cuda, odd):
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(
                lambda x: seen.append(tuple(x.shape)) or x.cpu(), unpack):
            loss = topk_distill_loss(z, t, i)
        assert seen.count((1, n, v)) == 2, seen
        (first,) = torch.autograd.grad(loss, z, one, retain_graph=True)
        assert torch.equal(first, want)
        first.zero_()
        # formed anew from the logits: the same formula, its factors multiplied
        # in another order, a few dozen roundings of 2^-24 at most
        (again,) = torch.autograd.grad(loss, z, one)
        torch.testing.assert_close(again, want, rtol=2.0 ** -18, atol=0)
    for reduction in ('mean', 'none'):            # the gradient stored, and not
        up = one if reduction == 'mean' else torch.full((n,), 1.0 / n, device=cuda)
        with torch.autograd.graph.saved_tensors_hooks(torch.Tensor.cpu, strided):
            loss = topk_distill_loss(z, t, i, reduction=reduction)
        (g,) = torch.autograd.grad(loss, z, up)
        torch.testing.assert_close(g, want, rtol=2.0 ** -18, atol=0)
    loss = torch.utils.checkpoint.checkpoint(topk_distill_loss, z, t, i, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(loss, z, one)[0], want)


@pytest.mark.parametrize('rest', [False, True])
def test_distill_padding_repeats_views_and_int32(cuda, rest):
    b, t, v, k = 3, 9, 1037, 6
    z = rand(cuda, b, t + 1, v + 3, seed=1, dtype=torch.bfloat16).requires_grad_()
    view = z[:, :-1, 1:v + 1]                    # odd rows and strides
    tt, ii, rr = _teacher(cuda, b * t, v, k, 1.3, rest, 4)
    tt, ii = tt.view(b, t, k), ii.view(b, t, k).to(torch.int32)
    ii[0, 3:] = -1                               # padding rows
    ii[1, 2, 4:] = -1                            # fewer entries
    ii[2, 5, 1] = ii[2, 5, 3]                    # an index twice
    tt[2, 6, 0] = float('-inf')                  # an entry without mass
    rr = None if rr is None else rr.view(b, t)
    loss = topk_distill_loss(view, tt, ii, teacher_rest=rr, temperature=1.3)
    want = ref.distill(view, tt, ii, rest=rr, temperature=1.3)
    ref.check('loss', loss, *want[:2])
    (g,) = torch.autograd.grad(loss, z)
    assert bool((g[:, -1] == 0).all()) and bool((g[..., 0] == 0).all())
    assert bool((g[0, 3:] == 0).all())
    ref.check('dz', g[:, :-1, 1:v + 1], *want[2:])
    # nothing to learn from at all
    none = topk_distill_loss(view, tt, torch.full_like(ii, -1), teacher_rest=rr)
    assert float(none.detach()) == 0.0 and bool((torch.autograd.grad(none, z)[0] == 0).all())


@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
@pytest.mark.parametrize('dtype, n', [('fp16', 300), ('bf16', 20), ('fp32', 20)])
def test_distill_weight(cuda, dtype, n, reduction):
    z = rand(cuda, n, 700, seed=1, dtype=DTYPES[dtype]).requires_grad_()
    t, i, r = _teacher(cuda, n, 700, 9, 1.0, True, 6)
    loss = topk_distill_loss(z, t, i, teacher_rest=r, weight=-0.5, reduction=reduction)
    up = torch.full_like(loss, 2.0)
    # -0.5 and 2 are powers of two: no rounding of their own
    want = ref.distill(z, t, i, rest=r, reduction=reduction, upstream=torch.ones(n) * -1.0)
    ref.check('loss', loss, -0.5 * want[0], 0.5 * want[1])
    ref.check('dz', *torch.autograd.grad(loss, z, up), *want[2:])


def test_distill_bad_rows_stay_alone(cuda):
    n, v, k = 6, 300, 4
    z = rand(cuda, n, v, seed=3)
    t, i, r = _teacher(cuda, n, v, k, 1.0, True, 5)
    good = topk_distill_loss(z, t, i, teacher_rest=r, reduction='none')
    z2, i2 = z.clone(), i.clone()
    i2[1, 2] = v                                  # behind the vocabulary
    i2[2, 0] = 2 ** 40
    z2[3, 17] = float('nan')
    z2[4, i[4, 1]] = float('-inf')                # the student excludes an entry
    z2.requires_grad_()
    loss = topk_distill_loss(z2, t, i2, teacher_rest=r, reduction='none')
    assert loss.isnan().tolist() == [False, True, True, True, False, False]
    assert float(loss[4]) == float('inf')
    assert torch.equal(loss[[0, 5]], good[[0, 5]])
    (g,) = torch.autograd.grad(loss, z2, torch.ones_like(loss))
    assert bool(g[[0, 4, 5]].isfinite().all()) and bool(g[[1, 2, 3]].isnan().any(dim=-1).all())
    # masked columns (-inf) that no entry names carry no probability
    z3 = z.clone()
    z3[:, :100] = float('-inf')
    keep = (i >= 100).all(dim=-1)
    z3.requires_grad_()
    loss = topk_distill_loss(z3, t, i, teacher_rest=r, reduction='none')
    (g,) = torch.autograd.grad(loss, z3, torch.ones_like(loss))
    assert bool(g[keep].isfinite().all())
    assert bool((g[keep][:, :100] == 0).all())


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('tau', [0.5, 1.0, 3.0])
@pytest.mark.parametrize('stored', [False, True])
def test_distill_lowest_values(cuda, stored, tau, rest, dtype):
    z, t, i, r, want = lowest_case(DTYPES[dtype], tau, rest)
    copies = 60 if stored else 1                  # 300 rows: the forward writes the gradient
    zz, tt, ii = (x.repeat(copies, 1).to(cuda) for x in (z, t, i))
    rr = r.repeat(copies).to(cuda) if rest else None
    zz.requires_grad_()
    conf = dict(teacher_rest=rr, temperature=tau)
    loss = topk_distill_loss(zz, tt, ii, reduction='none', **conf)
    ref.check('loss', loss, want[0].repeat(copies), want[1].repeat(copies))
    total = loss.sum() if not stored else topk_distill_loss(zz, tt, ii, reduction='sum', **conf)
    if stored:
        bound = want[1].sum() * copies + 2.0 ** -24 * want[0].sum().abs() * copies
        ref.check('sum', total, want[0].sum() * copies, bound)
    (g,) = torch.autograd.grad(total, zz)
    ref.check('dz', g, want[2].repeat(copies, 1), want[3].repeat(copies, 1))


@pytest.mark.parametrize('dtype', sorted(DTYPES))
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('n', [3, 256])
def test_distill_rows_of_one_large_value(cuda, n, rest, dtype):
    """A constant on a row's logits changes nothing: its columns are equal, and
    so are their powers, whatever the base of them rounds to."""
    t, i, r = _teacher(cuda, n, 40001, 20, 0.7, rest, 5)
    z = torch.full((n, 40001), 60000.0, dtype=DTYPES[dtype], device=cuda)
    z *= torch.where(torch.arange(n, device=cuda) % 2 == 0, 1.0, -1.0).to(z.dtype)[:, None]
    z.requires_grad_()
    want = ref.distill(torch.zeros_like(z), t, i, rest=r, temperature=0.7)
    loss = topk_distill_loss(z, t, i, teacher_rest=r, temperature=0.7)
    ref.check('loss', loss, *want[:2])
    ref.check('dz', *torch.autograd.grad(loss, z), *want[2:])


# ------------------------------------------------------------ in use
def _chain(x, conf):
    """The operators as a decoder's step runs them: qkv and logits from
    leaves, rotary, attention, a head, the loss; the leaves' gradients."""
    qkv, head = x
    q, k, v = qkv.permute(0, 2, 1, 3).split(conf['d'], dim=-1)
    q, k = rotary_axes(q, k, conf['pos'], sections=conf['sections'])
    o = window_attention(q, k, v, window=conf['window'], sinks=conf['sinks'])
    logits = o.transpose(1, 2).flatten(2) @ head
    loss = topk_distill_loss(logits, conf['teacher'], conf['index'], teacher_rest=conf['rest'],
                             temperature=2.0)
    return [loss, *torch.autograd.grad(loss, x)]


def _chain_inputs(dev, dtype, seed=0, b=2, t=70, h=4, d=16, v=333):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, t, h, 3 * d, generator=g)
    head = torch.randn(h * d, v, generator=g) * 0.3
    full = torch.randn(b, t, v, generator=g) * 2
    teacher, index = full.topk(8, dim=-1)
    rest = (full / 2).scatter(-1, index, float('-inf')).logsumexp(-1)
    conf = dict(d=d, window=16, sinks=2, sections=(3, 5), teacher=teacher.to(dev),
                index=index.to(dev), rest=rest.to(dev),
                pos=torch.randint(0, 900, (t, 2), generator=g).to(dev))
    return [x.to(dtype).to(dev).requires_grad_() for x in (qkv, head)], conf


def test_chain_matches_64_bits(cuda):
    """fp32 operators against the same chain in 64 bits on the CPU.  Each
    operator is within 2^-20 of its operands' size (the bounds above at these
    sizes), the matrix product within 64 roundings of 2^-24; the chain's
    gradient passes seven of them: 2^-16 of the gradient's largest element."""
    x, conf = _chain_inputs(cuda, torch.float32)
    got = _chain(x, conf)
    want = _chain([t.detach().cpu().double().requires_grad_() for t in x],
                  {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in conf.items()})
    for g, w in zip(got, want):
        assert float((g.cpu().double() - w).abs().max()) <= 2.0 ** -16 * float(w.abs().max())


def test_chain_repeats_bit_for_bit_on_any_stream(cuda):
    x, conf = _chain_inputs(cuda, torch.bfloat16, t=300)
    first = _chain(x, conf)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    answers = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            answers.append(_chain(x, conf))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for a in answers:
        assert all(torch.equal(p, q) for p, q in zip(first, a))


def test_chain_in_two_graphs(cuda):
    """Forward and backward captured twice, replayed with new inputs in turn
    and with eager work in between: every replay equals the eager answer."""
    graphs = []
    for n in range(2):
        x, conf = _chain_inputs(cuda, torch.bfloat16, seed=n, t=200 + 30 * n)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _chain(x, conf)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _chain(x, conf)
        graphs.append((g, x, conf, out))
    for rep in range(4):
        for n, (g, x, conf, out) in enumerate(graphs):
            new, _ = _chain_inputs(cuda, torch.bfloat16, seed=10 * rep + n + 5, t=200 + 30 * n)
            with torch.no_grad():
                for a, b in zip(x, new):
                    a.copy_(b)
            g.replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in out]
            eager = _chain(x, conf)
            assert all(torch.equal(a, b) for a, b in zip(kept, eager)), (rep, n)


def test_fp16_attention_in_a_graph_beside_eager_passes(cuda):
    """Forward and backward captured once, replayed with upstream gradients of
    very different sizes and eager passes in between."""
    q, k, v, do = (rand(cuda, 2, h, 600, 64, seed=s).half() for s, h in enumerate((4, 2, 2, 4)))
    ln = torch.tensor([600, 333], dtype=torch.int32, device=cuda)
    x = [t.requires_grad_() for t in (q, k, v)]

    def call():
        out = window_attention(*x, window=90, sinks=3, lengths=ln, q_start=0)
        return [out, *torch.autograd.grad(out, x, do)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = call()
    for seed, size in ((5, 1.0), (6, 2.0 ** -12), (7, 2.0 ** 11), (8, 1.0)):
        with torch.no_grad():
            do.copy_(rand(cuda, 2, 4, 600, 64, seed=seed).half() * size)
            q.copy_(rand(cuda, 2, 4, 600, 64, seed=seed + 10).half())
            ln[1] = 100 * (seed - 4)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in kept]
        for a, b in zip(got, call()):
            assert torch.equal(a, b), seed
            assert bool(a.isfinite().all()), seed


def test_offsets_behind_32_bits(cuda):
    """Operands of more than 2^31 elements: what lies at their end is what a
    small call on a copy of it gives, bit for bit."""
    d, tk = 128, 2 ** 24 + 77
    k = torch.zeros(1, 1, tk, d, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    q = rand(cuda, 1, 2, 3, d, seed=1, dtype=torch.bfloat16)
    for x, s in ((k, 2), (v, 3)):
        x[:, :, -200:] = rand(cuda, 1, 1, 200, d, seed=s, dtype=torch.bfloat16)
        x[:, :, :5] = rand(cuda, 1, 1, 5, d, seed=s + 5, dtype=torch.bfloat16)
    got = window_attention(q, k, v, window=150, sinks=5)
    kk, vv = (torch.cat([x[:, :, :5], x[:, :, -200:]], dim=2) for x in (k, v))
    want, tol = ref.attention(q, kk, vv, window=150, sinks=5)
    ref.check('out', got, want[0], tol[0])
    del k, v

    hk, tk = 9, 2 ** 21 + 5
    k = torch.zeros(1, hk, tk, d, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    q = rand(cuda, 1, hk, 3, d, seed=11, dtype=torch.bfloat16)
    do = rand(cuda, 1, hk, 3, d, seed=12, dtype=torch.bfloat16)
    for x, s in ((k, 13), (v, 14)):
        x[:, -1:, -200:] = rand(cuda, 1, 1, 200, d, seed=s, dtype=torch.bfloat16)
        x.requires_grad_()
    out = window_attention(q, k, v, window=150)
    got = torch.autograd.grad(out, (k, v), do)
    ends = [x.detach()[:, -1:, -200:] for x in (k, v)]
    want, tol = ref.attention(q[:, -1:], *ends, window=150, do=do[:, -1:])
    for i, name in enumerate(('dk', 'dv')):
        ref.check(name, got[i][:, -1:, -200:], want[2 + i], tol[2 + i])
        assert not bool(got[i][:, -1, :-200].any())
    del k, v, got, out

    b, h, t = 70, 16, 16384                       # 2.35e9 elements
    x = torch.zeros(b, h, t, d, dtype=torch.bfloat16, device=cuda)
    x[-1, -1, -9:] = rand(cuda, 9, d, seed=4, dtype=torch.bfloat16)
    pos = torch.arange(t, device=cuda)[:, None]
    one = x[-1:, -1:, -9:].clone()
    _, big = rotary_axes(x[:, :1], x, pos, sections=(64,))
    _, small = rotary_axes(one, one, pos[-9:], sections=(64,))
    assert torch.equal(big[-1:, -1:, -9:], small)
    del x, big

    n, vocab = 43000, 50304                       # 2.16e9 logits
    z = torch.zeros(n, vocab, dtype=torch.bfloat16, device=cuda)
    z[-3:] = rand(cuda, 3, vocab, seed=5, dtype=torch.bfloat16)
    t3, i3, _ = _teacher(cuda, 3, vocab, 6, 1.0, False, 8)
    idx = torch.full((n, 6), -1, device=cuda)
    idx[-3:] = i3
    tl = torch.zeros(n, 6, device=cuda)
    tl[-3:] = t3
    z.requires_grad_()
    loss = topk_distill_loss(z, tl, idx)
    want = ref.distill(z[-3:], t3, i3)
    ref.check('loss', loss, *want[:2])
    (g,) = torch.autograd.grad(loss, z)
    ref.check('dz', g[-3:], *want[2:])
    assert not bool(g[:-3].any())


def test_too_large_is_refused_on_the_host(cuda):
    one = torch.zeros(1, 1, 1, 8, device=cuda)
    many = one.expand(2 ** 25, 1, 1, 8)
    with pytest.raises(RuntimeError, match='too large'):
        window_attention(many, many, many, window=1)
    with pytest.raises(RuntimeError, match='row blocks'):
        window_attention(one.expand(1, 1, 2 ** 24, 8), one, one, window=1)
    with pytest.raises(RuntimeError, match='too large'):
        rotary_axes(one.expand(2, 1, 2 ** 30, 8), one.expand(2, 1, 2 ** 30, 8),
                    torch.zeros(1, 1, dtype=torch.int32, device=cuda).expand(2 ** 30, 1),
                    sections=(4,))
    row = torch.zeros(1, 1, device=cuda)
    with pytest.raises(RuntimeError, match='too many rows'):
        topk_distill_loss(row.expand(2 ** 24, 1), row.expand(2 ** 24, 1),
                          torch.zeros(1, 1, dtype=torch.int32, device=cuda).expand(2 ** 24, 1))


def test_more_heads_than_offsets_reach_are_refused(cuda):
    """64 tokens of 65536 heads of 128 in fp32 are 2^31 bytes."""
    x = torch.zeros(1, 2, 65536, 128, device=cuda).transpose(1, 2)
    for heads, fits in ((65536, False), (32768, True)):
        y = x[:, :heads] if not fits else x[:, :heads].contiguous()
        if fits:
            assert not bool(window_attention(y, y, y, window=1).any())
        else:
            with pytest.raises(RuntimeError, match='too large'):
                window_attention(y, y, y, window=1)


def test_more_sinks_than_a_launch_joins_are_refused(cuda):
    q, k = (torch.zeros(1, 1, t, 128, dtype=torch.bfloat16, device=cuda).requires_grad_()
            for t in (520, 16385))
    x = [y.expand(4096, -1, -1, -1) for y in (q, k, k)]
    out = window_attention(*x, window=1, sinks=16384)
    with pytest.raises(RuntimeError, match='too large'):
        torch.autograd.grad(out, (q, k), torch.zeros_like(out))


def test_gradients_of_gradients_are_refused(cuda):
    q = rand(cuda, 1, 1, 4, 8).requires_grad_()
    z = rand(cuda, 2, 9).requires_grad_()
    pos = torch.arange(4, device=cuda)[:, None]
    t, i, _ = _teacher(cuda, 2, 9, 2, 1.0, False, 1)
    for out, leaf in ((window_attention(q, q, q, window=2).sum(), q),
                      (rotary_axes(q, q, pos, sections=(4,))[0].sum(), q),
                      (topk_distill_loss(z, t, i), z)):
        with pytest.raises(RuntimeError, match='gradients of gradients'):
            torch.autograd.grad(out, leaf, create_graph=True)


def test_forward_mode_is_refused(cuda):
    q, z = rand(cuda, 1, 1, 4, 8), rand(cuda, 2, 9)
    pos = torch.arange(4, device=cuda)[:, None]
    t, i, _ = _teacher(cuda, 2, 9, 2, 1.0, False, 1)
    with torch.autograd.forward_ad.dual_level():
        dq, dz = (torch.autograd.forward_ad.make_dual(x, x) for x in (q, z))
        for call in (lambda: window_attention(dq, q, q, window=2),
                     lambda: window_attention(q, q.clone().requires_grad_(), dq, window=2),
                     lambda: rotary_axes(q, dq, pos, sections=(4,)),
                     lambda: topk_distill_loss(dz, t, i)):
            with pytest.raises(RuntimeError, match='forward-mode'):
                call()


@pytest.mark.parametrize('layout', ['interleaved', 'halves'])
@pytest.mark.parametrize('learns', [0, 1])
def test_rotary_turns_what_needs_a_gradient(cuda, learns, layout):
    x = [rand(cuda, 2, h, 7, 32, seed=h) for h in (3, 2)]
    do = [rand(cuda, 2, h, 7, 32, seed=h + 5) for h in (3, 2)]
    pos = torch.arange(7, device=cuda)[:, None]
    x[learns].requires_grad_()
    out = rotary_axes(*x, pos, sections=(16,), layout=layout)
    (g,) = torch.autograd.grad(out, x[learns], do)
    ref.check('dx', g, *ref.rotary(do[learns], pos, sections=(16,), layout=layout, sign=-1.0))


def test_results_are_tensors_of_their_own(cuda):
    """In-place operations on what a frozen part gave, as on the CPU: the
    attention's output is no view of a buffer that autograd knows."""
    q, z = rand(cuda, 2, 4, 6, 16), rand(cuda, 5, 9)
    pos = torch.arange(6, device=cuda)[:, None]
    t, i, _ = _teacher(cuda, 5, 9, 2, 1.0, False, 1)
    with torch.no_grad():
        outs = [window_attention(q, q, q, window=3), *rotary_axes(q, q, pos, sections=(8,)),
                topk_distill_loss(z, t, i, reduction='none')]
    for out in outs:
        adapter = torch.full_like(out, 2.0).requires_grad_()
        want = out + adapter.detach()
        out += adapter
        assert torch.equal(out, want)
        (g,) = torch.autograd.grad(out.sum(), adapter)
        assert bool((g == 1).all())


@pytest.mark.parametrize('dtype', sorted(DTYPES))
def test_nothing_at_all(cuda, dtype):
    dt = DTYPES[dtype]
    for shapes in (((0, 4, 5, 16), (0, 2, 7, 16)), ((2, 4, 0, 16), (2, 2, 7, 16)),
                   ((2, 4, 5, 16), (2, 2, 0, 16)), ((2, 0, 5, 16), (2, 2, 7, 16))):
        q, k, v = (rand(cuda, *s, dtype=dt).requires_grad_() for s in (*shapes, shapes[1]))
        out = window_attention(q, k, v, window=3, sinks=1)
        assert out.shape == q.shape and not bool(out.any())
        for x, g in zip((q, k, v), torch.autograd.grad(out, (q, k, v), torch.ones_like(out))):
            assert g.shape == x.shape and not bool(g.any())
    for lead in ((0,), (2, 0), (0, 3), (3, 0, 2)):
        z = rand(cuda, *lead, 11, dtype=dt).requires_grad_()
        t, i = rand(cuda, *lead, 3), torch.zeros(*lead, 3, dtype=torch.int64, device=cuda)
        for reduction in ('none', 'sum', 'mean'):
            loss = topk_distill_loss(z, t, i, teacher_rest=rand(cuda, *lead), reduction=reduction)
            assert loss.shape == (lead if reduction == 'none' else ()) and not bool(loss.any())
            (g,) = torch.autograd.grad(loss.sum(), z)
            assert g.shape == z.shape
    pos = torch.zeros(5, 1, dtype=torch.int64, device=cuda)
    q, k = rand(cuda, 0, 2, 5, 16, dtype=dt), rand(cuda, 0, 1, 5, 16, dtype=dt)
    assert [x.shape for x in rotary_axes(q, k, pos, sections=(8,))] == [q.shape, k.shape]
    q, k = (rand(cuda, 2, h, 5, 16, dtype=dt).requires_grad_() for h in (0, 1))
    out = rotary_axes(q, k, pos, sections=(8,))
    assert torch.equal(out[1], k)
    assert torch.equal(torch.autograd.grad(out[1].sum(), k)[0], torch.ones_like(k))


def test_one_operand_learns(cuda):
    q, k, v = (rand(cuda, 1, 2, 40, 16, seed=s) for s in range(3))
    do = rand(cuda, 1, 2, 40, 16, seed=5)
    want, tol = ref.attention(q, k, v, window=7, do=do)
    k.requires_grad_()
    out = window_attention(q, k, v, window=7)
    ref.check('dk', torch.autograd.grad(out, k, do)[0], want[2], tol[2])
    pos = torch.arange(40, device=cuda)[:, None]
    a, b = rotary_axes(q, k, pos, sections=(8,))
    (g,) = torch.autograd.grad(b, k, do)          # q's output is not used
    ref.check('dk', g, *ref.rotary(do, pos, sections=(8,), sign=-1.0))
