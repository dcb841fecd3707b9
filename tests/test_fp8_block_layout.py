"""Weights of the FP8 block modules lie as the product reads them (rows that begin at multiples of 16 bytes), whatever they came
from and wherever the module was moved: the product must not lay a weight out again at every call."""
import copy

import pytest
import torch

from amct_b200.backend import ops
from amct_b200.deploy_op import FP8BlockLinear
from amct_b200.experimental.quantization.deepseek_v3_2.experts import FP8RoutedExperts
from oracle import fp8_block as O

F8 = torch.float8_e4m3fn


def as_read(codes):
    laid, ld = ops._rows16(codes)
    return laid.data_ptr() == codes.data_ptr() and ld % 16 == 0


def moves(module):
    yield module
    yield copy.deepcopy(module)
    yield module.half()
    yield module.to(torch.bfloat16)
    # what moving to another device does: a copy of every buffer
    yield module._apply(lambda t: t.clone(memory_format=torch.contiguous_format))
    yield module._apply(lambda t: t.clone())


@pytest.mark.parametrize('dtype', [F8, torch.uint8])
@pytest.mark.parametrize('n,k', [(130, 200), (5, 256), (3, 17), (1, 200)])
def test_linear(n, k, dtype):
    codes, scale = O.quant_tiles(torch.randn(n, k, generator=torch.Generator().manual_seed(k)))
    shifted = torch.empty(n * k + 32, dtype=torch.uint8)
    shifted = shifted[16 - shifted.data_ptr() % 16 + 1:][:n * k].view(n, k)
    shifted.copy_(codes.view(torch.uint8))
    for source in (codes.view(dtype), shifted.view(dtype), codes.view(dtype).t().contiguous().t()):
        for module in moves(FP8BlockLinear.from_checkpoint(source, scale)):
            assert as_read(module.weight) and module.weight.dtype == F8
            assert torch.equal(module.weight.view(torch.uint8), codes.view(torch.uint8)) and module.weight.shape == (n, k)
            again = FP8BlockLinear.from_checkpoint(torch.zeros(n, k, dtype=F8), scale)
            again.load_state_dict(module.state_dict())
            assert as_read(again.weight) and torch.equal(again.weight.view(torch.uint8), codes.view(torch.uint8))


def test_aligned_checkpoint_tensors_are_not_copied():
    codes, scale = O.quant_tiles(torch.randn(130, 256, generator=torch.Generator().manual_seed(1)))
    assert FP8BlockLinear.from_checkpoint(codes, scale).weight.data_ptr() == codes.data_ptr()


def test_experts():
    gen = torch.Generator().manual_seed(3)
    gate_up, down = (torch.randint(0, 120, s, generator=gen, dtype=torch.uint8) for s in ((3, 256, 200), (3, 200, 128)))
    for module in moves(FP8RoutedExperts(gate_up.view(F8), torch.ones(3, 2, 2), down, torch.ones(3, 2, 1))):
        assert as_read(module.gate_up_weight) and as_read(module.down_weight)
        assert torch.equal(module.gate_up_weight.view(torch.uint8), gate_up) and torch.equal(module.down_weight, down)
        assert module.gate_up_weight.dtype == F8 and module.gate_up_scale.dtype == torch.float32
