"""Configurations of the 'fp8_block' algorithm: what it follows is taken, everything else refused by the field's name."""
import copy

import pytest
import torch

import amct_b200 as amct

CFG = {'batch_num': 1, 'quant_cfg': {'weights': {'type': 'float8_e4m3', 'symmetric': True, 'strategy': 'group', 'group_size': 128},
                                     'inputs': {'type': 'float8_e4m3', 'symmetric': True, 'strategy': 'token'}},
       'algorithm': {'fp8_block': {'pow2_scale': False}}}


def net():
    return torch.nn.Sequential(torch.nn.Linear(256, 130))


def changed(part, **fields):
    cfg = copy.deepcopy(CFG)
    cfg['quant_cfg'][part].update(fields)
    cfg['quant_cfg'][part] = {k: v for k, v in cfg['quant_cfg'][part].items() if v is not None}
    return cfg


@pytest.mark.parametrize('cfg', [CFG, {**CFG, 'algorithm': 'fp8_block'}, {**CFG, 'algorithm': {'fp8_block'}}, {**CFG, 'algorithm': {'fp8_block': {}}},
                                 changed('inputs', dynamic=True), changed('inputs', enable_quant=True)])
def test_taken(cfg):
    model = net()
    amct.quantize(model, cfg)
    assert type(model[0]).__name__ == 'FP8BlockQuant' and model[0].pow2_scale is False


@pytest.mark.parametrize('field,cfg', [
    ('weights type', changed('weights', type='int4')), ('weights type', changed('weights', type='int8')), ('weights type', changed('weights', type='hifloat8')),
    ('weights symmetric', changed('weights', symmetric=False)), ('weights group_size', changed('weights', group_size=32)),
    ('weights strategy', changed('weights', strategy='channel', group_size=None)), ('weights strategy', changed('weights', strategy='tensor', group_size=None)),
    ('inputs type', changed('inputs', type='int8')), ('inputs type', changed('inputs', type='hifloat8')), ('inputs strategy', changed('inputs', strategy='tensor')),
    ('inputs symmetric', changed('inputs', strategy='tensor', symmetric=False)), ('inputs enable_quant', changed('inputs', enable_quant=False)),
    ('inputs enable_quant', {**CFG, 'quant_cfg': {'weights': CFG['quant_cfg']['weights']}}),
    ('pow2', {**CFG, 'algorithm': {'fp8_block': {'pow2_scales': True}}})])
def test_refused(field, cfg):
    model = net()
    with pytest.raises(ValueError, match=field):
        amct.quantize(model, cfg)
    assert type(model[0]) is torch.nn.Linear


@pytest.mark.parametrize('algorithm', [{'hifloat8': {}}, {'minmax'}, {'gptq'}, {'awq': {'grids_num': 4}}, {'smoothquant': {'smooth_strength': 0.5}}])
@pytest.mark.parametrize('part', ['weights', 'inputs'])
def test_the_type_belongs_to_this_algorithm(algorithm, part):
    """None of the other algorithms here computes float8_e4m3: asked for it, they refuse instead of computing something else."""
    plain = 'hifloat8' if 'hifloat8' in algorithm else 'int8'
    cfg = {'batch_num': 1, 'quant_cfg': {'weights': {'type': plain, 'symmetric': True, 'strategy': 'channel'},
                                         'inputs': {'type': plain, 'symmetric': True, 'strategy': 'token'}}, 'algorithm': algorithm}
    cfg['quant_cfg'][part]['type'] = 'float8_e4m3'
    model = net().to(torch.bfloat16)
    with pytest.raises(ValueError, match='float8_e4m3'):
        amct.quantize(model, cfg)
    assert type(model[0]) is torch.nn.Linear
