"""The gated activation of an expert with its inputs kept in 8 bits for the backward pass."""

from .glu_checkpoint import dequantize_checkpoint, glu_checkpoint, glu_checkpoint_bwd, pack_gate_up_checkpoint

__all__ = ["glu_checkpoint", "glu_checkpoint_bwd", "pack_gate_up_checkpoint", "dequantize_checkpoint"]
