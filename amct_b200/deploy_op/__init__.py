from .npu_quantization_linear import NpuQuantizationLinear
from .weight_npu_quant_module import NpuWeightQuantizedLinear
from .fp8_block_linear import FP8BlockLinear

__all__ = ['NpuQuantizationLinear', 'NpuWeightQuantizedLinear', 'FP8BlockLinear']
