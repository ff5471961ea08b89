"""ops3d_b200 -- Flash Deformable 3D Attention for NVIDIA B200 (sm_100a).

Drop-in for the ``ops3d.flash_deform_attn`` entry points of cell-observatory/ops3d: hand-written
CUDA kernels behind a C ABI (``include/fda_b200.h``, ``libfda_b200.so``), a thin torch binding
(``ops3d_b200._C``) and the autograd wrapper ``FlashDeformAttnFunction``.  CUDA only.
"""
from ._extension import _C
from .experts import (CombineRowsFunction, DispatchRowsFunction, ExpertFeedForward, RouteExpertsFunction, RowOrder, combine_rows,
                      dispatch_rows, route_experts)
from .flash_deform_attn import FlashDeformAttnFunction, findspec, findspec_bwd
from .linear import FeedForward, FusedLinearFunction, GroupedLinear, fused_linear, grouped_linear, linear_timeouts
from .norm import LayerNorm, LayerNormFunction, layer_norm

__all__ = ["FlashDeformAttnFunction", "findspec", "findspec_bwd", "fused_linear", "grouped_linear", "FusedLinearFunction",
           "GroupedLinear", "FeedForward", "linear_timeouts", "layer_norm", "LayerNorm", "LayerNormFunction", "route_experts", "RouteExpertsFunction", "dispatch_rows",
           "DispatchRowsFunction", "RowOrder", "combine_rows", "CombineRowsFunction", "ExpertFeedForward", "_C"]
# The layer around the operator lives in ops3d_b200.msda3d (MSDeformAttn3D); imported on demand.
