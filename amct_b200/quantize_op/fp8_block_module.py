import torch
import torch.nn.functional as F

from .base_quant_module import BaseQuantizeModule
from ..utils.data_utils import check_linear_input_dim


class FP8BlockQuant(BaseQuantizeModule):
    """Calibration module of the 'fp8_block' algorithm.  Both scales come from the data they scale (weight tiles at
    conversion, activations at run time), so there is nothing to observe: calibration passes run the original Linear.
    Algorithm attribute ``pow2_scale`` (bool, may be omitted): scales are powers of two.  The configuration has to ask for
    what the deploy module computes: symmetric ``float8_e4m3`` weights in groups of 128, symmetric ``float8_e4m3`` inputs per
    token.  The reference has no such path; this module plugs in through algorithm_register().
    """
    FOLLOWED = {'weights': {'quant_type': 'float8_e4m3', 'symmetric': True, 'strategy': 'group', 'group_size': 128},
                'inputs': {'enable_quant': True, 'quant_type': 'float8_e4m3', 'symmetric': True, 'strategy': 'token'}}

    def __init__(self, ori_module, layer_name, quant_config):
        super().__init__(ori_module, layer_name, quant_config)
        self.ori_module = ori_module
        self.weight = ori_module.weight
        self.bias = ori_module.bias
        self.layer_name = layer_name
        attrs = (quant_config.get('algorithm') or {}).get('fp8_block') or {}
        if set(attrs) - {'pow2_scale'}:
            raise ValueError(f'fp8_block only support attribute pow2_scale, but got {sorted(attrs)}')
        for part, fields in self.FOLLOWED.items():
            given = {'enable_quant': True, **(quant_config.get(part + '_cfg') or {})}
            for field, value in fields.items():
                if given.get(field) != value:
                    name = 'type' if field == 'quant_type' else field
                    raise ValueError(f'fp8_block {part} {name} only support {value}, but got {given.get(field)}')
        pow2 = attrs.get('pow2_scale', False)
        if pow2 not in (True, False):
            raise ValueError(f'fp8_block pow2_scale only support bool [True, False], but got {pow2}')
        self.pow2_scale = pow2
        self.act_type = self.wts_type = 'float8_e4m3'

    @torch.no_grad()
    def forward(self, inputs):
        check_linear_input_dim(inputs)
        return F.linear(inputs, self.weight, self.bias)
