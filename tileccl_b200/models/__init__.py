"""Model-level blocks built from the fused operators."""

from .tp_mlp import TPMLP, pack_gate_up, reference_forward
from .tp_moe import TPMoE, reference_moe_forward

__all__ = ["TPMLP", "TPMoE", "pack_gate_up", "reference_forward", "reference_moe_forward"]
