"""B200-native (sm_100a) gated causal attention block.

Drop-in for xTimeCrystal/memory_efficient_attn_layer: ``fused_attn``,
``FusedAttentionFunction`` and ``CausalSoftmaxAttention`` keep the reference's
names and call surface; the work runs in hand-written tcgen05/TMA kernels in
``libmea.so`` (C ABI in ``include/mea.h``).
"""
from ._lib import MeaError, check_device_status
from .clip import clip_grad_norm_, grad_norm
from .dp import allreduce_grads, overlap_grad_allreduce
from .fused_attn import FusedAttentionFunction, fused_attn
from .module import CausalSoftmaxAttention, Yarn
from .norm import LayerNorm, LayerNormFunction, layer_norm
from .optim import ShardedAdamW
from .packed import PackedAttentionFunction, packed_attention

__all__ = ["fused_attn", "FusedAttentionFunction", "CausalSoftmaxAttention", "Yarn", "allreduce_grads",
           "overlap_grad_allreduce", "packed_attention", "PackedAttentionFunction", "layer_norm", "LayerNormFunction",
           "LayerNorm", "clip_grad_norm_", "grad_norm", "ShardedAdamW", "MeaError", "check_device_status"]
