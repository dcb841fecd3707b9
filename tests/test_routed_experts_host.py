"""Host side of the routed experts of a checkpoint, on the CPU: expert numbers, shapes and types of what is passed in."""
import pytest
import torch

from amct_b200.experimental.quantization.deepseek_v3_2.experts import FP8RoutedExperts

F8 = torch.float8_e4m3fn


def checkpoint(numbers, hidden=256, inter=128):
    tensors = {}
    for e in numbers:
        for name, (n, k) in (('gate_proj', (inter, hidden)), ('up_proj', (inter, hidden)), ('down_proj', (hidden, inter))):
            tensors[f'mlp.{e}.{name}.weight'] = torch.full((n, k), e, dtype=torch.uint8).view(F8)
            tensors[f'mlp.{e}.{name}.weight_scale_inv'] = torch.full((-(-n // 128), -(-k // 128)), float(e))
    return tensors


@pytest.mark.parametrize('numbers', [range(0, 3), range(8, 13), [5]])
def test_first_expert_is_the_first_number(numbers):
    layer = FP8RoutedExperts.from_checkpoint(checkpoint(numbers), 'mlp', numbers, device='cpu')
    assert layer.first_expert == numbers[0]
    assert layer.gate_up_weight.view(torch.uint8)[:, 0, 0].tolist() == list(numbers) and layer.down_scale[:, 0, 0].tolist() == list(numbers)
    assert FP8RoutedExperts.from_checkpoint(checkpoint(numbers), 'mlp', numbers, numbers[0], device='cpu').first_expert == numbers[0]
    assert FP8RoutedExperts.from_checkpoint(checkpoint(numbers), 'mlp', (e for e in numbers), device='cpu').first_expert == numbers[0]


@pytest.mark.parametrize('numbers,kwargs', [([8, 10, 12], {}), ([3, 2], {}), ([4, 4], {}), ([], {}), (range(8, 13), {'first_expert': 0}),
                                            (range(8, 13), {'first_expert': 9})])
def test_numbers_that_cannot_be_routed_are_refused(numbers, kwargs):
    with pytest.raises(ValueError, match='expert'):
        FP8RoutedExperts.from_checkpoint(checkpoint(numbers), 'mlp', numbers, device='cpu', **kwargs)


def parts(experts=2, hidden=256, inter=128):
    return {'gate_up_weight': torch.zeros(experts, 2 * inter, hidden, dtype=F8), 'gate_up_scale': torch.ones(experts, 2 * inter // 128, hidden // 128),
            'down_weight': torch.zeros(experts, hidden, inter, dtype=F8), 'down_scale': torch.ones(experts, hidden // 128, inter // 128)}


@pytest.mark.parametrize('hidden,inter', [(256, 128), (200, 128), (130, 256)])
def test_parts_that_fit_are_taken(hidden, inter):
    p = parts(hidden=256, inter=inter)
    kb = -(-hidden // 128)
    p.update(gate_up_weight=torch.zeros(2, 2 * inter, hidden, dtype=torch.uint8), gate_up_scale=torch.ones(2, 2 * inter // 128, kb),
             down_weight=torch.zeros(2, hidden, inter, dtype=F8), down_scale=torch.ones(2, kb, inter // 128))
    assert FP8RoutedExperts(**p).gate_up_scale.shape == (2, 2 * inter // 128, kb)


@pytest.mark.parametrize('name,value', [
    ('gate_up_scale', torch.ones(2, 2, 1)), ('gate_up_scale', torch.ones(2, 1, 2)), ('gate_up_scale', torch.ones(1, 2, 2)), ('gate_up_scale', torch.ones(2, 2)),
    ('down_scale', torch.ones(2, 2, 2)), ('down_scale', torch.ones(3, 2, 1)), ('gate_up_scale', torch.ones(2, 2, 2).half()),
    ('down_scale', torch.ones(2, 2, 1).double()), ('gate_up_weight', torch.zeros(2, 256, 256)), ('down_weight', torch.zeros(2, 256, 128).bfloat16()),
    ('gate_up_weight', torch.zeros(256, 256, dtype=F8)), ('down_weight', torch.zeros(2, 256, 64, dtype=F8)), ('gate_up_weight', torch.zeros(2, 200, 256, dtype=F8))])
def test_parts_that_do_not_fit_are_refused(name, value):
    with pytest.raises(ValueError, match='must'):
        FP8RoutedExperts(**{**parts(), name: value})
