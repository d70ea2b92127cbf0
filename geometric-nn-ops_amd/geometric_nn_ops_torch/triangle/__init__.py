"""Triangle (protein-folding) ops (reference geometric_nn_ops_torch/triangle/__init__.py:6-14)."""

from ._attention_pair_bias import attention_pair_bias
from ._fused_linear import fused_linear
from ._layer_norm import layer_norm
from ._relative_position import relative_position_bias
from ._triattn import triangle_attention
from ._trimul import triangle_multiplicative_update

__all__ = [
    "attention_pair_bias",
    "fused_linear",
    "layer_norm",
    "relative_position_bias",
    "triangle_attention",
    "triangle_multiplicative_update",
]
