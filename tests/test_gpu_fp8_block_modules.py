"""The FP8 block Linear through quantize() / convert() and from checkpoint tensors, and the routed experts of a checkpoint,
against the 64-bit restatement of the same steps."""
import pytest
import torch

import amct_b200 as amct
from oracle import fp8_block as O

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def linear64(x, w, bias=None, pow2=False, w_scale=None):
    """(value, bound): the Linear on the operands' codes, whose quantization is exact to the bit in the restatement; the bound
    is the product's (2^-13 of the sum of magnitudes, see the product's tests) plus the rounding to x's dtype."""
    a, a_scale = O.quant_tokens(x, pow2)
    b, b_scale = (w, w_scale) if w_scale is not None else O.quant_tiles(w, pow2)
    value, size = O.product(a, a_scale, b, b_scale, bias)
    return value, size * 2.0 ** -13 + value.abs() * half_step(x.dtype) * 1.01 + 1e-30


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('pow2', [False, True])
@pytest.mark.parametrize('bias', [False, True])
def test_linear_through_the_public_api(dtype, pow2, bias):
    torch.manual_seed(3)
    net = torch.nn.Sequential(torch.nn.Linear(200, 330, bias=bias)).to(dtype).cuda()
    w = net[0].weight.data.cpu().clone()
    b = net[0].bias.data.cpu().float() if bias else None
    cfg = {'batch_num': 1, 'quant_cfg': {'weights': {'type': 'float8_e4m3', 'symmetric': True, 'strategy': 'group', 'group_size': 128},
                                         'inputs': {'type': 'float8_e4m3', 'symmetric': True, 'strategy': 'token'}},
           'algorithm': {'fp8_block': {'pow2_scale': pow2}}}
    amct.quantize(net, cfg)
    x = torch.randn(2, 5, 200, generator=torch.Generator().manual_seed(1)).to(dtype)
    net(x.cuda())
    amct.convert(net)
    assert type(net[0]).__name__ == 'FP8BlockLinear'
    got = net(x.cuda())
    assert got.shape == (2, 5, 330) and got.dtype == dtype
    want, bound = linear64(x.reshape(10, 200), w, b, pow2)
    assert bool(((got.cpu().double().reshape(10, 330) - want).abs() <= bound).all())
    for rows in (0, 1, 17, 300):
        x = torch.randn(rows, 200, generator=torch.Generator().manual_seed(rows)).to(dtype)
        got = net(x.cuda())
        want, bound = linear64(x, w, b, pow2) if rows else (torch.zeros(0, 330, dtype=torch.float64), torch.zeros(0, 330))
        assert got.shape == (rows, 330) and bool(((got.cpu().double() - want).abs() <= bound).all())


def test_checkpoint_linear_agrees_with_its_dequantized_weight():
    """The module on a checkpoint's tensors against weight_dequant of the same tensors, which is exact in fp32."""
    from amct_b200.backend import ops
    from amct_b200.deploy_op import FP8BlockLinear
    codes, scale = O.quant_tiles(torch.randn(390, 512, generator=torch.Generator().manual_seed(5)) * 0.1)
    dequantized = ops.ckpt_block_dequant(codes.cuda(), scale.cuda(), out_dtype=torch.float32).cpu()
    layer = FP8BlockLinear.from_checkpoint(codes.cuda(), scale.cuda()).half()
    x = torch.randn(33, 512, generator=torch.Generator().manual_seed(6)).bfloat16()
    a, a_scale = O.quant_tokens(x)
    want = O.dequant_tokens(a, a_scale) @ dequantized.double().t()
    size = O.dequant_tokens(a, a_scale).abs() @ dequantized.double().abs().t()
    got = layer(x.cuda()).cpu().double()
    assert bool(((got - want).abs() <= size * (2.0 ** -13 + 2.0 ** -24) + want.abs() * half_step(torch.bfloat16) * 1.01).all())


@pytest.mark.parametrize('tokens', [0, 1, 3, 40, 700])
@pytest.mark.parametrize('index_dtype', [torch.int64, torch.int32])
def test_routed_experts_of_a_checkpoint(tokens, index_dtype):
    """moe_infer against the chain in 64 bits.  Between the two products the kernels' fp32 sums and the exact ones may fall on
    either side of a code's border (half a step, 2^-4 of the value, for single values): the result is compared by norm, with
    the second product's inputs off by at most 2^-4 each, independently, in a tenth of the places."""
    from amct_b200.experimental.quantization.deepseek_v3_2.experts import FP8RoutedExperts
    gen = torch.Generator().manual_seed(2)
    experts, hidden, inter, topk, first = 5, 256, 384, 3, 8
    tensors = {}
    for e in range(first, first + experts):
        for name, shape in (('gate_proj', (inter, hidden)), ('up_proj', (inter, hidden)), ('down_proj', (hidden, inter))):
            c, s = O.quant_tiles(torch.randn(shape, generator=gen) * 0.1)
            tensors[f'mlp.experts.{e}.{name}.weight'], tensors[f'mlp.experts.{e}.{name}.weight_scale_inv'] = c, s
    layer = FP8RoutedExperts.from_checkpoint(tensors, 'mlp.experts', range(first, first + experts), first_expert=first)
    assert tuple(layer.gate_up_weight.shape) == (experts, 2 * inter, hidden) and layer.gate_up_weight.dtype == F8
    x = torch.randn(tokens, hidden, generator=gen).bfloat16()
    ids = torch.randint(0, first + experts + 3, (tokens, topk), generator=gen)
    w = torch.rand(tokens, topk, generator=gen)
    got = layer(x.cuda(), ids.to(index_dtype).cuda(), w.cuda())
    assert got.shape == x.shape and got.dtype == x.dtype
    a, a_scale = O.quant_tokens(x)
    want = torch.zeros(tokens, hidden, dtype=torch.float64)
    for e in range(first, first + experts):
        for t, j in (ids == e).nonzero().tolist():
            def prod(name, codes, scale):
                return O.product(codes, scale, tensors[f'mlp.experts.{e}.{name}.weight'], tensors[f'mlp.experts.{e}.{name}.weight_scale_inv'])[0]
            g, u = (prod(n, a[t:t + 1], a_scale[t:t + 1]).bfloat16().double() for n in ('gate_proj', 'up_proj'))
            c, s = O.quant_tokens((g * torch.sigmoid(g) * u).float())
            want[t] += prod('down_proj', c, s)[0].bfloat16().double() * float(w[t, j])
    if float(want.norm()):
        assert float((got.cpu().double() - want).norm() / want.norm()) < 2.0 ** -4 * 0.32 + 2.0 ** -8
    untouched = (want == 0).all(1)
    assert not bool(got.cpu()[untouched].any())


def test_experts_calibrate_through_the_permutation():
    """A clip factor in front of the experts gets the gradient of the plain formula: tokens sorted by expert, one 16-bit
    Linear for each expert's rows, weighted sum."""
    from amct_b200.experimental.quantization.deepseek_v3_2 import experts as m
    gen = torch.Generator().manual_seed(4)
    tokens, topk, experts, hidden = 20, 2, 4, 32
    x = torch.randn(tokens, hidden, generator=gen)
    ids = torch.randint(0, experts, (tokens, topk), generator=gen)
    w = torch.rand(tokens, topk, generator=gen)
    mats = torch.randn(experts, hidden, hidden, generator=gen) * 0.2
    gain = torch.tensor([1.5], requires_grad=True)

    def loss(device, dtype, gain):
        xx, ww, mm = (t.to(device, dtype) for t in (x, w, mats))
        y = xx * gain
        if device == 'cpu':
            out = sum(torch.einsum('th,thk->tk', y, mm[ids[:, j]]) * ww[:, j:j + 1] for j in range(topk))
        else:
            rows, plan = m.permute_tokens(y, ids.cuda(), experts)
            at = plan.offsets.tolist()
            rows = torch.cat([rows[at[e]:at[e + 1]] @ mm[e] for e in range(experts)])
            out = m.unpermute_tokens(rows, plan, ww)
        return (out ** 2).sum()

    g64 = torch.tensor([1.5], dtype=torch.float64, requires_grad=True)
    (want,) = torch.autograd.grad(loss('cpu', torch.float64, g64), g64)
    gain = torch.tensor([1.5], device='cuda', requires_grad=True)
    (got,) = torch.autograd.grad(loss('cuda', torch.float32, gain), gain)
    # a sum of 640 squares and 2 * 32 products each, every step rounded by 2^-24, all terms of the outer sum positive
    assert abs(float(got) - float(want)) <= abs(float(want)) * (2 * 32 + 640) * 2.0 ** -24 * 4
