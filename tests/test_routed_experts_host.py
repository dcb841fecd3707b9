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
