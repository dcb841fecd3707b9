"""Plans of the routing operators that their callers made, on the CPU: refused before anything is read from them."""
import pytest
import torch

from amct_b200.backend import ops


def plan(offsets):
    return ops.MoePlan(torch.zeros(3, 2, dtype=torch.int32), offsets)


@pytest.mark.parametrize('offsets', [torch.zeros(5, dtype=torch.int64), torch.zeros(5, dtype=torch.int16), torch.zeros(5), torch.zeros(0, dtype=torch.int32),
                                     torch.zeros(1, dtype=torch.int32), torch.zeros(1, 5, dtype=torch.int32), torch.zeros((), dtype=torch.int32), None])
def test_offsets_of_another_type_or_shape_are_refused(offsets):
    """Four bytes are read at the last entry: of a 16-bit one they would lie past its end."""
    from amct_b200.experimental.quantization.deepseek_v3_2 import experts
    rows, w, g = torch.zeros(6, 8), torch.ones(3, 2), torch.zeros(3, 8)
    with pytest.raises(ValueError, match='offsets'):
        ops.moe_unpermute_backward(g, rows, plan(offsets), w)
    with pytest.raises(ValueError, match='offsets'):
        experts.unpermute_tokens(rows.requires_grad_(), plan(offsets), w)
