"""The weighted sum keeps its rows for the backward pass only where a weight wants a gradient."""
import weakref

import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
    from amct_b200.backend import ops as o
    return o


def m():
    from amct_b200.experimental.quantization.deepseek_v3_2 import experts
    return experts


@pytest.mark.parametrize('weighted', ['none', 'plain', 'leaf'])
def test_rows_are_let_go(weighted):
    gen = torch.Generator().manual_seed(1)
    ids = torch.tensor([[0, 2], [1, -1], [2, 1]]).cuda()
    x = torch.randn(3, 8, generator=gen).cuda()
    w = None if weighted == 'none' else torch.rand(3, 2, generator=gen).cuda().requires_grad_(weighted == 'leaf')
    g = torch.randn(3, 8, generator=gen).cuda()
    _, plan = m().permute_tokens(x, ids, 3)
    leaf = torch.randn(6, 8, generator=gen).cuda().requires_grad_()
    rows = leaf * 1.0
    kept = weakref.ref(rows)
    out = m().unpermute_tokens(rows, plan, w)
    values = rows.detach().clone()
    del rows
    assert weighted == 'leaf' or kept() is None
    saved = [t for t in out.grad_fn.saved_tensors if t is not None and t.shape == values.shape]
    assert len(saved) == (1 if weighted == 'leaf' else 0)
    grads = torch.autograd.grad(out, [leaf] + ([w] if weighted == 'leaf' else []), g)
    want = ops().moe_unpermute_backward(g, values, plan, None if w is None else w.detach())
    assert torch.equal(grads[0].cpu(), want[0].cpu())
    if weighted == 'leaf':
        assert torch.equal(grads[1].cpu(), want[1].cpu())


def test_rows_may_be_left_out_where_no_weight_wants_a_gradient():
    row_map, offsets = torch.tensor([[1, 0], [2, -1]], dtype=torch.int32).cuda(), torch.tensor([0, 2, 3], dtype=torch.int32).cuda()
    plan, g, w = ops().MoePlan(row_map, offsets), torch.ones(2, 5).cuda(), torch.tensor([[2.0, 3.0], [4.0, 5.0]]).cuda()
    rows, none = ops().moe_unpermute_backward(g, None, plan, w, want_weights=False)
    assert none is None and rows[:, 0].tolist() == [3.0, 2.0, 4.0, 0.0] and rows.shape == (4, 5)
    rows, none = ops().moe_unpermute_backward(g, None, plan)
    assert none is None and rows[:, 4].tolist() == [1.0, 1.0, 1.0, 0.0]
    with pytest.raises(ValueError, match='rows'):
        ops().moe_unpermute_backward(g, None, plan, w)
    with pytest.raises(ValueError, match='grad_out'):
        ops().moe_unpermute_backward(g[:1], None, plan)
