"""Decoder operators on the CPU: what they refuse, the torch formulas against
64 bits and against differences."""
from __future__ import annotations

import pytest
import torch

from distributed_kfac_pytorch_amd.ops.attention import window_attention
from distributed_kfac_pytorch_amd.ops.distill import topk_distill_loss
from distributed_kfac_pytorch_amd.ops.rotary import rotary_axes
from tests import lm_reference as ref


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ------------------------------------------------------------- refusals
def _qkv(b=1, hq=2, hk=1, t=4, d=8, dtype=torch.float32):
    return rand(b, hq, t, d, dtype=dtype), rand(b, hk, t, d, dtype=dtype), rand(b, hk, t, d, dtype=dtype)


@pytest.mark.parametrize('change, error', [
    (dict(window=0), ValueError),
    (dict(sinks=-1), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(scale=float('nan')), ValueError),
    (dict(lengths=torch.tensor([4])), ValueError),                       # int64
    (dict(lengths=torch.tensor([4, 4], dtype=torch.int32)), ValueError),  # two sequences
    (dict(q_start=torch.tensor([0.0])), ValueError),
])
def test_attention_refuses_options(change, error):
    q, k, v = _qkv()
    with pytest.raises(error):
        window_attention(q, k, v, **{'window': 2, **change})


@pytest.mark.parametrize('shapes, error', [
    (((1, 2, 4, 8), (1, 1, 4, 8), (1, 1, 5, 8)), ValueError),     # v unlike k
    (((1, 3, 4, 8), (1, 2, 4, 8), (1, 2, 4, 8)), ValueError),     # heads do not divide
    (((2, 2, 4, 8), (1, 1, 4, 8), (1, 1, 4, 8)), ValueError),     # batch
    (((1, 2, 4, 12), (1, 1, 4, 12), (1, 1, 4, 12)), ValueError),  # head size
    (((1, 2, 4, 136), (1, 1, 4, 136), (1, 1, 4, 136)), ValueError),
    (((1, 2, 4, 8), (1, 0, 4, 8), (1, 0, 4, 8)), ValueError),
    (((2, 4, 8), (1, 4, 8), (1, 4, 8)), ValueError),
])
def test_attention_refuses_shapes(shapes, error):
    q, k, v = (rand(*s) for s in shapes)
    with pytest.raises(error):
        window_attention(q, k, v, window=2)


@pytest.mark.parametrize('scale', [1e-46, 2.0 ** -127, -1.0, 1e39, float('inf')])
def test_attention_refuses_a_scale_that_32_bits_do_not_hold(scale):
    q, k, v = _qkv()
    with pytest.raises(ValueError, match='scale'):
        window_attention(q, k, v, window=2, scale=scale)


def test_attention_refuses_types():
    q, k, v = _qkv()
    with pytest.raises(TypeError):
        window_attention(q.half(), k, v, window=2)
    with pytest.raises(TypeError):
        window_attention(q.int(), k.int(), v.int(), window=2)


@pytest.mark.parametrize('change, error', [
    (dict(sections=()), ValueError),
    (dict(sections=(0, 2)), ValueError),
    (dict(sections=(5,)), ValueError),
    (dict(sections=(2, 2)), ValueError),          # positions have one axis
    (dict(base=0.0), ValueError),
    (dict(ladder='none'), ValueError),
    (dict(layout='none'), ValueError),
])
def test_rotary_refuses(change, error):
    q, k, _ = _qkv()
    with pytest.raises(error):
        rotary_axes(q, k, torch.arange(4)[:, None], **{'sections': (4,), **change})


def test_rotary_refuses_operands():
    q, k, _ = _qkv()
    with pytest.raises(TypeError):
        rotary_axes(q, k, torch.arange(4.0)[:, None], sections=(4,))
    with pytest.raises(TypeError):
        rotary_axes(q, k.half(), torch.arange(4)[:, None], sections=(4,))
    with pytest.raises(ValueError):
        rotary_axes(q, k[:, :, :3], torch.arange(4)[:, None], sections=(4,))
    with pytest.raises(ValueError):
        rotary_axes(q, k, torch.arange(4), sections=(4,))
    with pytest.raises(ValueError):
        rotary_axes(q[..., :7], k[..., :7], torch.arange(4)[:, None], sections=(3,))


@pytest.mark.parametrize('change, error', [
    (dict(temperature=0.0), ValueError),
    (dict(temperature=float('inf')), ValueError),
    (dict(reduction='avg'), ValueError),
    (dict(weight=float('nan')), ValueError),
    (dict(teacher_rest=torch.zeros(2)), ValueError),
    (dict(teacher_rest=torch.zeros(3, dtype=torch.int64)), ValueError),
])
def test_distill_refuses_options(change, error):
    with pytest.raises(error):
        topk_distill_loss(rand(3, 9), rand(3, 2), torch.zeros(3, 2, dtype=torch.int64), **change)


@pytest.mark.parametrize('change', [
    dict(temperature=1e-39), dict(temperature=1e39), dict(temperature=1e20), dict(temperature=1e-20),
    dict(temperature=-1.0), dict(weight=1e39), dict(weight=-float('inf'))])
def test_distill_refuses_factors_that_32_bits_do_not_hold(change):
    with pytest.raises(ValueError, match=next(iter(change))):
        topk_distill_loss(rand(3, 9), rand(3, 2), torch.zeros(3, 2, dtype=torch.int64), **change)


@pytest.mark.parametrize('z, t, i, error', [
    (rand(3, 9), rand(3, 2), torch.zeros(3, 3, dtype=torch.int64), ValueError),
    (rand(3, 9), rand(2, 2), torch.zeros(2, 2, dtype=torch.int64), ValueError),
    (rand(3, 9), rand(3, 0), torch.zeros(3, 0, dtype=torch.int64), ValueError),
    (rand(3, 9), rand(3, 1025), torch.zeros(3, 1025, dtype=torch.int64), ValueError),
    (rand(3, 9), rand(3, 2), torch.zeros(3, 2), TypeError),
    (rand(3, 9), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int64), TypeError),
    (torch.zeros(3, 9, dtype=torch.int32), rand(3, 2), torch.zeros(3, 2, dtype=torch.int64), TypeError),
    (rand(3, 0), rand(3, 2), torch.zeros(3, 2, dtype=torch.int64), ValueError),
])
def test_distill_refuses_operands(z, t, i, error):
    with pytest.raises(error):
        topk_distill_loss(z, t, i)


def test_the_kernels_refuse_tangents():
    """Before anything else, so this shows on the CPU too; the CPU's formulas
    carry them."""
    from distributed_kfac_pytorch_amd.ops import _native

    q, z = rand(1, 1, 4, 8), rand(1, 2, 9)
    pos, t, i = torch.arange(4)[:, None], rand(2, 2), torch.zeros(2, 2, dtype=torch.int64)
    table = torch.zeros(4, 2, dtype=torch.float64)
    with torch.autograd.forward_ad.dual_level():
        dq, dz = (torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)) for x in (q, z))
        lib = _native.native()
        if lib is not None:
            for call in (lambda: lib.window_attention(q, q, dq, None, None, 2, 0, 0, False, 1.0),
                         lambda: lib.rotary_axes(dq, q, pos, table, False),
                         lambda: lib.topk_distill_loss(dz, t, i, None, 1.0, 1.0, 2, [1, 2])):
                with pytest.raises(RuntimeError, match='forward-mode'):
                    call()
        for out in (window_attention(q, q, dq, window=2), rotary_axes(dq, q, pos, sections=(4,))[0],
                    topk_distill_loss(dz[0], t, i)):
            assert torch.autograd.forward_ad.unpack_dual(out).tangent is not None


# -------------------------------------------------------- against 64 bits
@pytest.mark.parametrize('hq, hk, tq, tk, window, sinks, lengths, start', [
    (2, 2, 7, 7, 3, 0, None, None),
    (4, 2, 9, 9, 2, 3, None, None),
    (4, 1, 1, 9, 4, 2, [9, 3, 0], None),
    (3, 3, 6, 6, 2, 1, [6, 4, 0], 0),
    (2, 1, 5, 8, 20, 0, [8, 2, 5], None),     # fewer tokens than rows
    (2, 1, 4, 8, 3, 1, None, -2),
    (2, 1, 3, 0, 3, 1, None, None),           # no keys
])
def test_attention_formula(hq, hk, tq, tk, window, sinks, lengths, start):
    b = 3
    q, k, v, do = (rand(b, h, t, 8, seed=s) for s, (h, t) in
                   enumerate([(hq, tq), (hk, tk), (hk, tk), (hq, tq)]))
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    if lengths is not None:
        for i, n in enumerate(lengths):  # what lies behind a sequence is not read
            k[i, :, n:] = float('nan')
            v[i, :, n:] = float('inf')
    conf = dict(window=window, sinks=sinks, lengths=ln, q_start=start)
    want, tol = ref.attention(q, k, v, do=do, **conf)
    x = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention(*x, **conf)
    got = [out, *torch.autograd.grad(out, x, do)]
    for name, g, w, t in zip(('out', 'dq', 'dk', 'dv'), got, want, tol):
        ref.check(name, g, w, t)


def test_rows_of_padding_may_hold_anything():
    q, k, v, do = (rand(2, h, 6, 8, seed=s) for s, h in enumerate((4, 2, 2, 4)))
    conf = dict(window=2, sinks=1, lengths=torch.tensor([6, 3], dtype=torch.int32), q_start=0)
    want, tol = ref.attention(q, k, v, do=do, **conf)
    for x in (q, k, v, do):
        x[1, :, 3:] = float('nan')
    x = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention(*x, **conf)
    got = [out, *torch.autograd.grad(out, x, do)]
    for name, g, w, t in zip(('out', 'dq', 'dk', 'dv'), got, want, tol):
        ref.check(name, g, w, t)


def test_keys_that_no_row_sees_may_hold_anything():
    q, do = (rand(1, 4, 4, 8, seed=s) for s in range(2))
    k, v = (rand(1, 2, 64, 8, seed=s) for s in (2, 3))
    conf = dict(window=8, sinks=3)
    want, tol = ref.attention(q, k, v, do=do, **conf)
    for x in (k, v):
        x[:, :, 3], x[:, :, 40] = float('nan'), float('inf')
    x = [t.requires_grad_() for t in (q, k, v)]
    out = window_attention(*x, **conf)
    got = [out, *torch.autograd.grad(out, x, do)]
    for name, g, w, t in zip(('out', 'dq', 'dk', 'dv'), got, want, tol):
        ref.check(name, g, w, t)


def test_autocast_changes_nothing():
    q, k, v = _qkv(2, 4, 2, 9)
    pos, (z, t, i, r) = torch.arange(9)[:, None], _distill_case(rest=True)

    def call(*x):
        turned = rotary_axes(*x[:2], pos, sections=(4,))
        return (window_attention(*turned, x[2], window=4, sinks=1), *turned,
                topk_distill_loss(x[3], t, i, teacher_rest=r))

    x = [a.requires_grad_() for a in (q, k, v, z)]
    want = call(*x)
    with torch.autocast('cpu', dtype=torch.bfloat16):
        got = call(*x)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b)
    for a, b in zip(*(torch.autograd.grad(sum(y.sum() for y in out), x) for out in (got, want))):
        assert torch.equal(a, b)
    q = torch.empty(1, 2, 4, 8, device='meta')        # a device without autocast
    assert window_attention(q, q, q, window=2).shape == q.shape


def test_attention_output_is_a_tensor_of_its_own():
    """[B, T, H, D] in memory and no view: in-place operations on what a frozen
    part gave are allowed."""
    q = rand(2, 4, 6, 8)
    with torch.no_grad():
        out = window_attention(q, q, q, window=3)
    assert out.transpose(1, 2).is_contiguous() and out._base is None
    adapter = torch.ones_like(out).requires_grad_()
    out += adapter
    assert bool((torch.autograd.grad(out.sum(), adapter)[0] == 1).all())


def test_attention_differences():
    q, k, v = (t.double().requires_grad_() for t in _qkv(2, 4, 2, 5))
    ln = torch.tensor([5, 3], dtype=torch.int32)
    assert torch.autograd.gradcheck(
        lambda *a: window_attention(*a, window=2, sinks=1, lengths=ln, q_start=0), (q, k, v))


@pytest.mark.parametrize('layout', ['interleaved', 'halves'])
@pytest.mark.parametrize('ladder', ['shared', 'per_axis'])
def test_rotary_formula_and_differences(layout, ladder):
    q, k = rand(2, 3, 5, 18), rand(2, 1, 5, 18, seed=1)
    pos = torch.randint(-9, 10 ** 6, (2, 5, 3), generator=torch.Generator().manual_seed(3))
    conf = dict(sections=(3, 1, 4), ladder=ladder, layout=layout, base=500.0)
    for g, x in zip(rotary_axes(q, k, pos, **conf), (q, k)):
        ref.check('turned', g, *ref.rotary(x, pos, **conf))
    assert torch.autograd.gradcheck(lambda a, b: rotary_axes(a, b, pos, **conf),
                                    (q.double().requires_grad_(), k.double().requires_grad_()))


def test_rotary_keeps_no_tensor_of_another_mode():
    """A call under a fake-tensor mode or inference mode leaves nothing behind
    that a later call would trip over, and the other way round."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from distributed_kfac_pytorch_amd.ops import rotary

    def call(**kw):
        q, pos = torch.ones(1, 2, 4, 24, **kw), torch.arange(4)[:, None]
        return rotary_axes(q, q, pos, sections=(11,), base=77.0)[0]

    key = ((11,), 77.0, 'shared')
    with FakeTensorMode():
        assert call().shape == (1, 2, 4, 24)
        assert rotary._table(*key).shape == (11, 2)
    with torch.inference_mode():
        call()
        kept = rotary._table(*key)
    call(requires_grad=True).sum().backward()
    table = rotary._table(*key)
    assert type(table) is torch.Tensor and not table.is_inference() and table is kept
    with FakeTensorMode():
        call()


def test_rotary_one_axis_is_the_models_rotation():
    from distributed_kfac_pytorch_amd.models.gpt_neox import _rotary

    q, k = rand(2, 3, 9, 16), rand(2, 3, 9, 16, seed=1)
    got = rotary_axes(q, k, torch.arange(9)[:, None], sections=(8,))
    for g, x in zip(got, (q, k)):
        torch.testing.assert_close(g, _rotary(x), rtol=0, atol=2e-5)


def _distill_case(n=4, v=23, k=5, seed=0, rest=False, tau=1.0, dtype=torch.float32):
    z = rand(n, v, seed=seed) * 3
    full = z * 0.5 + rand(n, v, seed=seed + 1) * 2
    t, i = full.topk(k, dim=-1)
    r = (full / tau).scatter(-1, i, float('-inf')).logsumexp(-1) if rest else None
    return z.to(dtype), t, i, r


def lowest_case(dtype, tau, rest, v=40, k=5):
    """Rows that are masked with the type's lowest value: some of the student's
    logits, all of them, some of the teacher's entries, all of them.  The
    answers are those of a row in which nothing is masked where only the mask
    is left, and of no probability (2^-288 for the student, which has no place
    in any type) in the mask's place where something is."""
    low = torch.finfo(dtype).min
    z, t, i, r = _distill_case(n=5, v=v, k=k, rest=rest, tau=tau, dtype=dtype)
    clean_z, clean_t = z.clone(), t.clone()
    spare = [c for c in range(v) if c not in i[1].tolist()][:9]  # none of the teacher's
    z[1, spare], clean_z[1, spare] = low, -200.0 * tau
    z[2], clean_z[2] = low, 0.0
    t[3, 2:], clean_t[3, 2:] = torch.finfo(torch.float32).min, float('-inf')
    t[4], clean_t[4] = torch.finfo(torch.float32).min, 0.0
    if rest:
        r[4] = float('-inf')     # nothing beside the masked entries
    want = ref.distill(clean_z, clean_t, i, rest=r, temperature=tau, reduction='none')
    assert all(bool(x.isfinite().all()) for x in want)
    return z, t, i, r, want


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('k, twist', [(1, ''), (5, ''), (5, 'padded'), (5, 'twice'), (23, ''),
                                      (5, 'all padded')])
def test_distill_formula(rest, reduction, k, twist):
    z, t, i, r = _distill_case(k=k, rest=rest, tau=1.5)
    if twist == 'padded':
        i[1] = -1
        i[2, 3:] = -7
    elif twist == 'all padded':
        i[:] = -1
    elif twist == 'twice':
        i[0, 1] = i[0, 3]
    up = rand(4, seed=9) if reduction == 'none' else torch.tensor(0.3)
    z.requires_grad_()
    loss = topk_distill_loss(z, t, i, teacher_rest=r, temperature=1.5, reduction=reduction)
    want = ref.distill(z, t, i, rest=r, temperature=1.5, reduction=reduction, upstream=up)
    ref.check('loss', loss, *want[:2])
    ref.check('dz', *torch.autograd.grad(loss, z, up), *want[2:])


def test_distill_differences_and_dense_limit():
    z, t, i, r = _distill_case(rest=True)
    z = z.double()
    assert torch.autograd.gradcheck(
        lambda a: topk_distill_loss(a, t, i, teacher_rest=r), (z.requires_grad_(),))
    # every column an entry: the divergence of the whole distributions
    t = rand(4, 23, seed=5).double()
    i = torch.argsort(t, dim=-1, descending=True)
    got = topk_distill_loss(z, t.gather(-1, i), i)
    dense = torch.nn.functional.kl_div(torch.log_softmax(z, -1), torch.softmax(t, -1),
                                       reduction='batchmean')
    torch.testing.assert_close(got, dense)


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('tau', [0.5, 1.0, 3.0])
def test_distill_lowest_values(tau, rest):
    z, t, i, r, want = lowest_case(torch.float32, tau, rest)
    z.requires_grad_()
    loss = topk_distill_loss(z, t, i, teacher_rest=r, temperature=tau, reduction='none')
    ref.check('loss', loss, *want[:2])
    ref.check('dz', *torch.autograd.grad(loss, z, torch.ones_like(loss)), *want[2:])


def test_distill_rows_of_padding_may_hold_anything():
    z, t, i, _ = _distill_case()
    i[1:3] = -1
    want = ref.distill(z, t, i)
    z[1], z[2, 3] = float('-inf'), float('nan')
    z.requires_grad_()
    loss = topk_distill_loss(z, t, i)
    ref.check('loss', loss, *want[:2])
    ref.check('dz', *torch.autograd.grad(loss, z), *want[2:])


def test_distill_index_behind_the_vocabulary_is_nan():
    z, t, i, _ = _distill_case()
    i[2, 1] = 23
    loss = topk_distill_loss(z, t, i, reduction='none')
    assert loss.isnan().tolist() == [False, False, True, False]
