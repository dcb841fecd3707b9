"""The status word of the FP8 block product, on the CPU: anything but an int32 is refused, since four bytes are written to it."""
import pytest
import torch

from amct_b200.backend import lib, ops
from oracle import fp8_block as O


def calls(status):
    codes, scale = O.quant_tokens(torch.zeros(2, 128))
    yield lambda: ops.gemm_fp8_block(codes, scale, codes, scale[:1], status=status)
    yield lambda: ops.gemm_fp8_block_grouped(codes, scale, torch.zeros(2, dtype=torch.int32), codes[None], scale[None, :1], status=status)


@pytest.mark.parametrize('status', [torch.zeros(1), torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.uint8), torch.zeros(0, dtype=torch.int32)])
def test_another_type_or_nothing_is_refused(status):
    for call in calls(status):
        with pytest.raises(ValueError, match='status'):
            call()


def test_an_int32_gets_as_far_as_the_device():
    for call in calls(torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(lib.BackendError, match='CUDA'):
            call()
