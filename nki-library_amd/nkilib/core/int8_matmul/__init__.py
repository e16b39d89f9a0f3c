"""Products in 8-bit integers with a scale per token and per channel, dense and by expert."""

from .int8_matmul import grouped_int8_matmul, int8_matmul

__all__ = ["int8_matmul", "grouped_int8_matmul"]
