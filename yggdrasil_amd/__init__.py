"""yggdrasil_amd -- MI355X-native (gfx950) MoE-HLM expert layer.

A from-scratch HIP implementation of Yggdrasil's MoE-HLM expert layer
(``holograph/models/hlm_block.py:154-183``): CliffordRouter top-k gating,
token dispatch, grouped CliffordLinear expert products with the grade-wise
activation fused, and the weighted combine, behind the C ABI declared in
``include/ygg_moe.h`` and the torch module ``CliffordMoELayer``; the pre-norm
and residual around it (``hlm_block.py:144-151``) as ``CliffordMoEBlockFFN``.
fp32 layers train through autograd; bf16 layers, the router, the norm and the
block do so on request (``bf16_grad``, ``router_grad``, ``grad``); the operators' gradients
are in ``ops`` for callers who chain them.  Serving in int8: ``weight_format``
'int8_rows' (rows and weights), 'int8_pauli' (decode) and 'int8' (weights).
"""

from .layers import (CliffordLayerNorm, CliffordLinear, CliffordMoEBlockFFN, CliffordMoELayer,  # noqa: F401
                     MoEHLMConfig)
from . import ops  # noqa: F401

__all__ = ["CliffordMoELayer", "CliffordMoEBlockFFN", "CliffordLayerNorm", "CliffordLinear", "MoEHLMConfig", "ops"]
