"""Host side of the FP8 block and routing operators, on the CPU: argument types against the public header, refusals that
need no device, the 'fp8_block' algorithm's configuration, buffer types of its modules."""
import re

import pytest
import torch

import amct_b200 as amct
from amct_b200.backend import lib, ops
from amct_b200.deploy_op import FP8BlockLinear
from oracle import fp8_block as O


def test_argument_types_are_the_header_s():
    text = re.sub(r'/\*.*?\*/', '', open(lib.HEADER).read(), flags=re.S)
    for name, letters in lib._SIGNATURES.items():
        args = re.search(r'\b%s\(([^)]*)\)' % name, text, re.S).group(1).split(',')
        want = ''.join('p' if '*' in a else 'l' if 'int64_t' in a else 'i' for a in args)
        assert letters == want, name


def test_the_workspace_of_the_sort_begins_where_the_wrapper_allocates_it():
    few, handle = ops.MOE_FEW_ASSIGNMENTS, lib.load()
    assert handle.amct_moe_permute_workspace_bytes(few, 256) == 0
    assert handle.amct_moe_permute_workspace_bytes(few + 1, 256) >= 4 * 256


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros(2, 128), torch.zeros(2, 1, dtype=torch.int64)
    codes, scale = O.quant_tokens(x)
    plan = ops.MoePlan(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    for call in (lambda: ops.fp8_block_quant(x), lambda: ops.gemm_fp8_block(codes, scale, codes, scale[:1]),
                 lambda: ops.gemm_fp8_block_grouped(codes, scale, torch.zeros(2, dtype=torch.int32), codes[None], scale[None, :1]),
                 lambda: ops.moe_permute(x, ids, 1), lambda: ops.moe_unpermute(x, plan),
                 lambda: ops.moe_unpermute_backward(x, x, plan, torch.ones(2, 1))):
        with pytest.raises(lib.BackendError):
            call()


def test_permutation_of_codes_has_no_gradient():
    from amct_b200.experimental.quantization.deepseek_v3_2 import experts
    with pytest.raises(ValueError):
        experts.permute_tokens(torch.zeros(2, 4, dtype=torch.float64, requires_grad=True), torch.zeros(2, 1, dtype=torch.int64), 1)


CFG = {'batch_num': 1, 'quant_cfg': {'weights': {'type': 'float8_e4m3', 'symmetric': True, 'strategy': 'group', 'group_size': 128},
                                     'inputs': {'type': 'float8_e4m3', 'symmetric': True, 'strategy': 'token'}},
       'algorithm': {'fp8_block': {'pow2_scale': True}}}


def test_quantize_puts_the_calibration_module_in_place():
    net = torch.nn.Sequential(torch.nn.Linear(256, 130), torch.nn.ReLU(), torch.nn.Linear(130, 8))
    x = torch.randn(3, 256)
    want = net(x)
    amct.quantize(net, {**CFG, 'skip_layers': ['2']})
    assert type(net[0]).__name__ == 'FP8BlockQuant' and net[0].pow2_scale is True and type(net[2]) is torch.nn.Linear
    assert torch.equal(net(x), want)
    with pytest.raises(ValueError):
        amct.quantize(torch.nn.Sequential(torch.nn.Linear(8, 8)), {**CFG, 'algorithm': {'fp8_block': {'pow2_scale': 'yes'}}})


def test_checkpoint_tensors_and_buffer_types():
    codes, scale = O.quant_tiles(torch.randn(130, 200, generator=torch.Generator().manual_seed(1)))
    layer = FP8BlockLinear.from_checkpoint(codes, scale, torch.zeros(130, dtype=torch.bfloat16))
    assert sorted(layer.state_dict()) == ['bias', 'weight', 'weight_scale_inv']
    for moved in (layer.half(), layer.to(torch.bfloat16), layer.double(), layer.to('cpu')):
        assert moved.weight.dtype == torch.float8_e4m3fn and moved.weight_scale_inv.dtype == torch.float32 and moved.bias.dtype == torch.float32
        assert torch.equal(moved.weight.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(moved.weight_scale_inv, scale)
    other = FP8BlockLinear.from_checkpoint(torch.zeros(130, 200, dtype=torch.uint8), torch.ones(2, 2))
    other.load_state_dict({k: v for k, v in layer.state_dict().items() if k != 'bias'})
    assert torch.equal(other.weight.view(torch.uint8), codes.view(torch.uint8)) and other.bias is None
    with pytest.raises(ValueError):
        FP8BlockLinear.from_checkpoint(codes, scale[:1])
