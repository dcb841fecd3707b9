import torch
import torch.nn.functional as F

from .base_quant_module import BaseQuantizeModule
from ..utils.data_utils import check_linear_input_dim


class FP8BlockQuant(BaseQuantizeModule):
    """Calibration module of the 'fp8_block' algorithm.  Both scales come from the data they scale (weight tiles at
    conversion, activations at run time), so there is nothing to observe: calibration passes run the original Linear.
    Algorithm attribute ``pow2_scale`` (bool, may be omitted): scales are powers of two.  The reference has no such path;
    this module plugs in through algorithm_register().
    """

    def __init__(self, ori_module, layer_name, quant_config):
        super().__init__(ori_module, layer_name, quant_config)
        self.ori_module = ori_module
        self.weight = ori_module.weight
        self.bias = ori_module.bias
        self.layer_name = layer_name
        attrs = (quant_config.get('algorithm') or {}).get('fp8_block') or {}
        pow2 = attrs.get('pow2_scale', False)
        if pow2 not in (True, False):
            raise ValueError(f'fp8_block pow2_scale only support bool [True, False], but got {pow2}')
        self.pow2_scale = pow2
        self.act_type = self.wts_type = 'float8_e4m3'

    @torch.no_grad()
    def forward(self, inputs):
        check_linear_input_dim(inputs)
        return F.linear(inputs, self.weight, self.bias)
