"""dynconv: MI355X-native dynamic short convolutions (headwise and lowrank).

Public API (same as the reference's headwise.py / lowrank.py):
    headwise_dynamic_convolution(x, weight, static_w=None, residual=False)
    lowrank_dynamic_convolution(x, z, U, static_w=None, residual=False)

Beyond the reference's operators: lowrank_dynamic_convolution_grouped (the
q / k / v convolutions of one layer in one launch per direction, README.md:57-110)
and the README's LowRankDynamicShortConvolution module, plus its grouped form.

Behind the convolutions of a layer: linear_attention with a decay for each head (whole
sequences) and linear_attention_step (single tokens), group_norm with its gate, the
convolutions' single-token form lowrank_dynamic_convolution_step(_grouped), and
DynamicLinearAttention, a layer of all of them.

The operators are torch.autograd.Functions backed by hand-written gfx950 HIP kernels
in libdynconv.so, reached through a C ABI (include/dynconv.h, include/dynconv_layer.h).
"""

from .headwise import headwise_dynamic_convolution, _HeadwiseDynamicConvolutionFn  # noqa: F401
from .lowrank import lowrank_dynamic_convolution, _LowrankDynamicConvolutionFn  # noqa: F401
from .lowrank import lowrank_dynamic_convolution_grouped  # noqa: F401
from .lowrank import lowrank_dynamic_convolution_step, lowrank_dynamic_convolution_step_grouped  # noqa: F401
from .linattn import linear_attention, linear_attention_step  # noqa: F401
from .norm import group_norm  # noqa: F401
from .modules import LowRankDynamicShortConvolution, GroupedLowRankDynamicShortConvolution  # noqa: F401
from .modules import DynamicLinearAttention, LayerState  # noqa: F401
from ._capi import LIB_PATH, load as load_library  # noqa: F401

__all__ = [
    "headwise_dynamic_convolution",
    "lowrank_dynamic_convolution",
    "lowrank_dynamic_convolution_grouped",
    "lowrank_dynamic_convolution_step",
    "lowrank_dynamic_convolution_step_grouped",
    "linear_attention",
    "linear_attention_step",
    "group_norm",
    "LowRankDynamicShortConvolution",
    "GroupedLowRankDynamicShortConvolution",
    "DynamicLinearAttention",
    "LayerState",
    "load_library",
    "LIB_PATH",
]
