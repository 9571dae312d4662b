"""GPT-NeoX with windowed attention, position axes and distillation."""
from __future__ import annotations

import copy
import warnings

import pytest
import torch

from distributed_kfac_pytorch_amd.models.gpt_neox import GPTNeoX
from distributed_kfac_pytorch_amd.models.gpt_neox import gpt_neox_pipeline_layers
from distributed_kfac_pytorch_amd.neox.pipeline import PipelineModule
from distributed_kfac_pytorch_amd.neox.preconditioner import GPTNeoXKFACPreconditioner
from distributed_kfac_pytorch_amd.neox.topology import PipeModelDataParallelTopology
from distributed_kfac_pytorch_amd.utils.training import TopKDistillLoss
from distributed_kfac_pytorch_amd.warnings import ExperimentalFeatureWarning
from tests import lm_reference as ref
from tests.test_examples import _run

warnings.filterwarnings('ignore', category=ExperimentalFeatureWarning)

SHAPE = dict(vocab=64, hidden=64, layers=2, heads=4)


def _tokens(b=3, t=21, seed=0):
    return torch.randint(0, 64, (b, t), generator=torch.Generator().manual_seed(seed))


def test_default_model_is_unchanged():
    """Without the new options the blocks hold the same weights and run the
    same calls: logits bit for bit those of a block-by-block reference."""
    from distributed_kfac_pytorch_amd.models.gpt_neox import _rotary

    model, tok = GPTNeoX(**SHAPE), _tokens()
    x = model.embed_in(tok)
    for blk in model.layers:
        a, h = blk.attention, blk.input_layernorm(x)
        qkv = a.query_key_value(h).view(3, 21, 4, 48)
        q, k, v = qkv.permute(0, 2, 1, 3).split(16, dim=-1)
        o = torch.nn.functional.scaled_dot_product_attention(_rotary(q), _rotary(k), v,
                                                             is_causal=True)
        x = x + a.dense(o.permute(0, 2, 1, 3).reshape(3, 21, 64)) + blk.mlp(
            blk.post_attention_layernorm(x))
    assert torch.equal(model(tok), model.embed_out(model.final_layer_norm(x)))


def test_window_of_the_whole_sequence_is_full_attention():
    full = GPTNeoX(**SHAPE)
    windowed = GPTNeoX(**SHAPE, attention_window=64)
    windowed.load_state_dict(full.state_dict())
    tok = _tokens()
    # rotary angles of at most 20 radians in 32 bits against 64: 20 * 2^-24
    # of a rotated element; two layers of products of 64 terms on top
    torch.testing.assert_close(windowed(tok), full(tok), rtol=0, atol=1e-4)


def test_window_hides_and_sinks_show():
    """A token that lies outside every later window changes no later logit
    of a one-layer model; as a sink it does."""
    tok = _tokens(1, 12)
    other = tok.clone()
    other[0, 0] = (tok[0, 0] + 1) % 64
    shape = dict(SHAPE, layers=1)
    for sinks, same in ((0, True), (1, False)):
        model = GPTNeoX(**shape, attention_window=4, attention_sinks=sinks)
        a, b = model(tok), model(other)
        assert torch.equal(a[:, 4:], b[:, 4:]) is same
        assert not torch.equal(a[:, :4], b[:, :4])


def test_positions_have_axes():
    model, tok = GPTNeoX(**SHAPE, rotary_sections=(2, 3, 3)), _tokens(2, 12)
    i = torch.arange(12)
    grid = torch.stack([i // 6, i // 3 % 2, i % 3], dim=-1)
    text = i[:, None].expand(12, 3)
    assert torch.equal(model(tok), model(tok, text))
    assert not torch.equal(model(tok), model(tok, grid))
    assert torch.equal(model(tok, grid), model(tok, grid.expand(2, 12, 3)))
    # scores see differences of positions only
    torch.testing.assert_close(model(tok, grid + 7), model(tok, grid), rtol=0, atol=1e-4)


def test_refused_options():
    with pytest.raises(ValueError):
        GPTNeoX(**SHAPE, attention_sinks=2)
    with pytest.raises(ValueError):
        GPTNeoX(**SHAPE, attention_window=0)
    with pytest.raises(ValueError):
        GPTNeoX(**dict(SHAPE, hidden=48), attention_window=4)   # heads of 12
    with pytest.raises(ValueError):
        GPTNeoX(**SHAPE)(_tokens(), torch.arange(21)[:, None])
    with pytest.raises(ValueError):
        GPTNeoX(**SHAPE, rotary_sections=(5, 5))(_tokens())


def test_pipeline_layers_have_the_window():
    whole = GPTNeoX(**SHAPE, attention_window=5, attention_sinks=1)
    x = tok = _tokens()
    for make in gpt_neox_pipeline_layers(**SHAPE, attention_window=5, attention_sinks=1):
        x = make()(x)
    assert torch.equal(x, whole(tok))


def test_distill_module():
    z = torch.randn(4, 9, 33, generator=torch.Generator().manual_seed(1)).requires_grad_()
    best, index = torch.randn(4, 9, 33, generator=torch.Generator().manual_seed(2)).topk(5)
    loss = TopKDistillLoss(temperature=2.0, weight=0.25)(z, best, index)
    want = [0.25 * w for w in ref.distill(z, best, index, temperature=2.0)]
    ref.check('loss', loss, *want[:2])
    ref.check('dz', *torch.autograd.grad(loss, z), *want[2:])


def test_cli_window_and_teacher(tmp_path):
    base = ['examples/torch_gpt_neox.py', '--steps', '2', '--seq-len', '16', '--micro-batch', '2',
            '--factor-update-steps', '1', '--inv-update-steps', '2', '--log-interval', '1',
            '--no-cuda', '--backend', 'gloo']
    teacher = str(tmp_path / 'teacher.pt')
    assert _run(base + ['--save', teacher])[-1]['tokens_per_s'] > 0
    lines = _run(base + ['--attention-window', '5', '--attention-sinks', '1', '--teacher', teacher,
                         '--distill-topk', '8'])
    assert [line['step'] for line in lines if 'step' in line] == [1, 2]
    assert all(line['loss'] == line['loss'] for line in lines)


def test_cli_teacher_keeps_its_window(tmp_path):
    """A teacher that was trained with a window is evaluated with it."""
    from distributed_kfac_pytorch_amd.utils.training import load_checkpoint
    from examples.torch_gpt_neox import MODELS
    from examples.torch_gpt_neox import load_teacher

    path = str(tmp_path / 'teacher.pt')
    _run(['examples/torch_gpt_neox.py', '--steps', '1', '--seq-len', '16', '--micro-batch', '2',
          '--attention-window', '5', '--attention-sinks', '1', '--save', path,
          '--no-cuda', '--backend', 'gloo'])
    sizes = {n: MODELS['tiny'][n] for n in ('vocab', 'hidden', 'layers', 'heads')}
    teacher = load_teacher(path, sizes['vocab'], sizes, None)
    state = load_checkpoint(path)
    windowed, full = GPTNeoX(**sizes, attention_window=5, attention_sinks=1), GPTNeoX(**sizes)
    for m in (windowed, full):
        m.load_state_dict(state['model'])
    tok = torch.randint(0, sizes['vocab'], (2, 16), generator=torch.Generator().manual_seed(1))
    assert torch.equal(teacher(tok), windowed(tok))
    assert not torch.equal(teacher(tok), full(tok))
    # a checkpoint that says nothing: the model's sizes, all tokens seen
    del state['config']
    torch.save(state, path)
    assert torch.equal(load_teacher(path, sizes['vocab'], sizes, None)(tok), full(tok))
    with pytest.raises(ValueError, match='vocabulary'):
        load_teacher(path, sizes['vocab'] + 1, sizes, None)


def _grads(model, tok, teacher):
    logits = model(tok[:, :-1])
    best, index = teacher
    loss = TopKDistillLoss(2.0)(logits, best, index)
    return logits, loss, torch.autograd.grad(loss, list(model.parameters()))


@pytest.mark.gpu
def test_model_on_the_gpu_matches_64_bits(cuda):
    """fp32 on the GPU against the same model in 64 bits: the model is two
    blocks of operators that are each within 2^-18 of their operands' size
    (products of 64 to 256 terms in 32 bits, library GEMMs among them), some
    twenty of them in a row forward and as many backward: 2^-12 of a
    gradient's largest element."""
    gpu = GPTNeoX(**SHAPE, attention_window=16, attention_sinks=2, rotary_sections=(3, 5))
    cpu = copy.deepcopy(gpu).double()
    gpu = gpu.to(cuda)
    tok = _tokens(2, 71)
    g = torch.Generator().manual_seed(4)
    best, index = torch.randn(2, 70, 64, generator=g).topk(6)
    logits, loss, grads = _grads(gpu, tok.to(cuda), (best.to(cuda), index.to(cuda)))
    wl, wloss, wgrads = _grads(cpu, tok, (best, index))
    for a, b in ((logits, wl), (loss, wloss), *zip(grads, wgrads)):
        assert float((a.cpu().double() - b).abs().max()) <= 2.0 ** -12 * float(b.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [None, torch.bfloat16, torch.float16])
def test_kfac_step_on_the_gpu(cuda, dtype):
    """K-FAC over the windowed model with distillation: every factor and
    preconditioned gradient is finite, and all eight linears are registered."""
    topo = PipeModelDataParallelTopology(num_pp=1, num_mp=1, num_dp=1)
    model = PipelineModule(
        [lambda: GPTNeoX(**SHAPE, attention_window=16, attention_sinks=2)], topo, rank=0).to(cuda)
    pre = GPTNeoXKFACPreconditioner(model, factor_update_steps=1, inv_update_steps=1, lr=0.1)
    assert len(pre._layers) == 8
    tok = _tokens(4, 65).to(cuda)
    best, index = torch.randn(4, 64, 64, device=cuda).topk(6)
    for _ in range(2):
        model.zero_grad(set_to_none=False)
        with torch.autocast('cuda', dtype=dtype or torch.bfloat16, enabled=dtype is not None):
            logits = model(tok[:, :-1])
        assert logits.dtype == (dtype or torch.float32)
        TopKDistillLoss(2.0)(logits, best, index).backward()
        pre.step()
        assert all(bool(p.grad.isfinite().all()) for p in model.parameters())
