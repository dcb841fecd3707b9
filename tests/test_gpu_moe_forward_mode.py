"""Forward-mode derivatives of the permutation: refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def m():
    from amct_b200.experimental.quantization.deepseek_v3_2 import experts
    return experts


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('leaf', [True, False])
def test_dual_tensors_are_refused(grad, leaf):
    """Whether or not the inputs want a gradient besides, and with gradients switched off."""
    ids = torch.tensor([[0, 2], [1, 0], [2, 1]]).cuda()
    x, rows, w = torch.ones(3, 8).cuda(), torch.ones(6, 8).cuda(), torch.ones(3, 2).cuda()
    _, plan = m().permute_tokens(x, ids, 4)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        def dual(t):
            return forward_ad.make_dual(t.clone().requires_grad_(leaf), torch.ones_like(t))
        for call in (lambda: m().permute_tokens(dual(x), ids, 4), lambda: m().unpermute_tokens(dual(rows), plan),
                     lambda: m().unpermute_tokens(dual(rows), plan, w), lambda: m().unpermute_tokens(rows, plan, dual(w))):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call()
        # inside a dual level what carries no tangent goes through
        out = m().unpermute_tokens(m().permute_tokens(x, ids, 4)[0], plan, w)
        assert torch.equal(out.cpu(), torch.full((3, 8), 2.0)) and forward_ad.unpack_dual(out).tangent is None
