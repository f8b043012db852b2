"""Import path of the operators behind the convolutions, beside headwise.py and lowrank.py.

    from linattn import linear_attention, linear_attention_step, group_norm, DynamicLinearAttention
    from linattn import gated_delta_rule, gated_delta_rule_step, residual_norm, DynamicDeltaRule, DynamicDeltaStack

resolves to dynamic-conv1d_amd/dynconv/linattn.py, delta.py, norm.py and modules.py.
"""

import os as _os
import sys as _sys

_PKG_DIR = _os.path.join(_os.path.dirname(_os.path.abspath(__file__)), "dynamic-conv1d_amd")
if _PKG_DIR not in _sys.path:
    _sys.path.insert(0, _PKG_DIR)

from dynconv.linattn import linear_attention, linear_attention_step  # noqa: E402,F401
from dynconv.delta import gated_delta_rule, gated_delta_rule_step  # noqa: E402,F401
from dynconv.norm import group_norm, residual_norm  # noqa: E402,F401
from dynconv.modules import DynamicDeltaRule, DynamicDeltaStack, DynamicLinearAttention, LayerState  # noqa: E402,F401
