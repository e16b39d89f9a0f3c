from .rmsnorm_quant import RmsNormQuantKernelArgs, rmsnorm_quant_kernel
from .rmsnorm_quant_rows import dequantize_rows, rmsnorm_quant_rows, rmsnorm_quant_rows_bwd

__all__ = ["RmsNormQuantKernelArgs", "rmsnorm_quant_kernel", "rmsnorm_quant_rows", "rmsnorm_quant_rows_bwd", "dequantize_rows"]
