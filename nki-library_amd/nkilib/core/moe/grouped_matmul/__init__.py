"""Products of the rows of every expert with its weights, and their gradients."""

from .grouped_matmul import expert_row_offsets, grouped_matmul, grouped_matmul_bwd

__all__ = ["expert_row_offsets", "grouped_matmul", "grouped_matmul_bwd"]
