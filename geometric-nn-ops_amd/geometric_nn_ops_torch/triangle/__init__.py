"""Triangle (protein-folding) ops (reference geometric_nn_ops_torch/triangle/__init__.py:6-14)."""

from ._attention_pair_bias import attention_pair_bias
from ._cross_attention import cross_attention
from ._fused_linear import fused_linear
from ._gated_linear import gated_linear
from ._layer_norm import layer_norm
from ._qk_norm_rotary import qk_norm_rotary
from ._relative_position import relative_position_bias
from ._triattn import triangle_attention
from ._trimul import triangle_multiplicative_update

__all__ = [
    "attention_pair_bias",
    "cross_attention",
    "fused_linear",
    "gated_linear",
    "layer_norm",
    "qk_norm_rotary",
    "relative_position_bias",
    "triangle_attention",
    "triangle_multiplicative_update",
]
