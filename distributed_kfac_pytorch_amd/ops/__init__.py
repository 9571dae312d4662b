"""Native-op layer: every hot tensor op of K-FAC, with a gfx950 HIP kernel
for GPU tensors and the reference's PyTorch math for CPU tensors.

Modules:
    _native       extension loader and GPU policy (fail loudly if missing)
    factors       SYRK factor accumulation, conv patch extraction
    linalg        batched eigensolver, damped SPD inverse
    precondition  eigen-basis scaling, KL-clip reduction, in-place grad write
    comm_pack     triangle / bucket packing for collectives
    attention     causal attention with a sliding window and sinks
    rotary        rotary positions with several axes
    distill       distillation from a teacher's top logits
"""
from distributed_kfac_pytorch_amd.ops import attention
from distributed_kfac_pytorch_amd.ops import comm_pack
from distributed_kfac_pytorch_amd.ops import distill
from distributed_kfac_pytorch_amd.ops import factors
from distributed_kfac_pytorch_amd.ops import linalg
from distributed_kfac_pytorch_amd.ops import precondition
from distributed_kfac_pytorch_amd.ops import rotary
from distributed_kfac_pytorch_amd.ops._native import available as native_available
from distributed_kfac_pytorch_amd.ops._native import native
from distributed_kfac_pytorch_amd.ops.attention import window_attention
from distributed_kfac_pytorch_amd.ops.distill import topk_distill_loss
from distributed_kfac_pytorch_amd.ops.rotary import rotary_axes

__all__ = [
    'attention',
    'comm_pack',
    'distill',
    'factors',
    'linalg',
    'precondition',
    'rotary',
    'native',
    'native_available',
    'rotary_axes',
    'topk_distill_loss',
    'window_attention',
]
