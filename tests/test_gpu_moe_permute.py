"""Tokens sorted by expert and back, and their gradients, against plain loops in 64 bits (oracle/fp8_block.py)."""
import pytest
import torch

from oracle import fp8_block as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def ops():
    from amct_b200.backend import ops as o
    return o


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def routing(tokens, topk, experts, seed, elsewhere=0.0, wide=True):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, topk), generator=gen)
    if elsewhere:
        away = torch.rand(ids.shape, generator=gen) < elsewhere
        ids = torch.where(away, torch.randint(0, 2, ids.shape, generator=gen) * (experts + 3) - 1, ids)   # -1 or experts + 2
    return ids if wide else ids.to(torch.int32)


CASES = [(1, 1, 1, 0.0), (1, 8, 256, 0.0), (3, 2, 4, 0.3), (16, 8, 256, 0.0), (128, 8, 32, 0.2), (129, 8, 32, 0.2), (700, 3, 7, 0.0),
         (513, 8, 1024, 0.1), (1100, 4, 3, 0.5), (40, 70, 16, 0.1), (5, 6, 10, 1.0)]


@pytest.mark.parametrize('tokens,topk,experts,elsewhere', CASES)
@pytest.mark.parametrize('wide', [True, False])
def test_plan_and_rows(tokens, topk, experts, elsewhere, wide):
    ids = routing(tokens, topk, experts, tokens + topk, elsewhere, wide)
    x = torch.randn(tokens, 40, generator=torch.Generator().manual_seed(3))
    scales = torch.rand(tokens, 3, generator=torch.Generator().manual_seed(4))
    rows, row_scales, plan = ops().moe_permute(x.cuda(), ids.cuda(), experts, scales=scales.cuda())
    row_map, offsets = O.plan(ids, experts)
    assert torch.equal(plan.row_map.cpu(), row_map) and torch.equal(plan.offsets.cpu(), offsets)
    assert torch.equal(rows.cpu(), O.permute(x, row_map)) and torch.equal(row_scales.cpu(), O.permute(scales, row_map))


@pytest.mark.parametrize('tokens,topk,experts', [(9000, 2, 64)])
def test_many_chunks_of_assignments(tokens, topk, experts):
    ids = routing(tokens, topk, experts, 11, 0.05)
    x = torch.arange(tokens, dtype=torch.float32)[:, None]
    rows, _, plan = ops().moe_permute(x.cuda(), ids.cuda(), experts)
    row_map, offsets = O.plan(ids, experts)
    assert torch.equal(plan.row_map.cpu(), row_map) and torch.equal(plan.offsets.cpu(), offsets)
    assert torch.equal(rows.cpu(), O.permute(x, row_map))


def test_all_assignments_to_one_expert_and_repeated_experts():
    for fill in (0, 5, 6):
        ids = torch.full((300, 4), fill)
        x = torch.randn(300, 8, generator=torch.Generator().manual_seed(1))
        rows, _, plan = ops().moe_permute(x.cuda(), ids.cuda(), 6)
        row_map, offsets = O.plan(ids, 6)
        assert torch.equal(plan.row_map.cpu(), row_map) and torch.equal(plan.offsets.cpu(), offsets)
        assert torch.equal(rows.cpu(), O.permute(x, row_map))


@pytest.mark.parametrize('dtype', DTYPES + [torch.uint8, torch.int8])
@pytest.mark.parametrize('hidden', [0, 1, 2, 7, 12, 16, 130, 1024, 2056])
def test_types_widths_and_strides(dtype, hidden):
    for tokens, topk in ((6, 3), (600, 2)):
        ids = routing(tokens, topk, 9, hidden, 0.2)
        base = torch.randint(-100, 100, (tokens, hidden + 5), generator=torch.Generator().manual_seed(2)).to(dtype)
        row_map, _ = O.plan(ids, 9)
        for x in (base[:, :hidden], base[:, 3:3 + hidden], base[:, :hidden].contiguous()):
            rows, _, _ = ops().moe_permute(x.cuda() if x.is_contiguous() else base.cuda()[:, 3:3 + hidden] if x.data_ptr() != base.data_ptr() else base.cuda()[:, :hidden], ids.cuda(), 9)
            assert rows.shape == (tokens * topk, hidden) and torch.equal(rows.cpu(), O.permute(x, row_map))


def test_codes_with_scales_as_the_quantizer_lays_them_out():
    x = torch.randn(50, 300, generator=torch.Generator().manual_seed(9)).cuda()
    ids = routing(50, 4, 8, 1, 0.1)
    codes, scale = ops().fp8_block_quant(x)
    rows, row_scales, plan = ops().moe_permute(codes, ids.cuda(), 8, scales=scale)
    row_map, _ = O.plan(ids, 8)
    assert rows.dtype == torch.float8_e4m3fn and rows.stride(0) % 16 == 0
    assert torch.equal(rows.view(torch.uint8).cpu(), O.permute(codes.view(torch.uint8).cpu(), row_map))
    assert torch.equal(row_scales.cpu(), O.permute(scale.cpu(), row_map))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('weight_dtype', [None] + DTYPES)
@pytest.mark.parametrize('tokens,topk,hidden', [(1, 1, 8), (2, 8, 1032), (7, 9, 33), (300, 6, 256), (3, 20, 2048)])
def test_unpermute(tokens, topk, hidden, dtype, weight_dtype):
    """fp32 sum of topk products: each of the topk fused steps rounds by 2^-24 of at most the sum of magnitudes, and the
    result once to dtype."""
    gen = torch.Generator().manual_seed(tokens * 7 + topk)
    ids = routing(tokens, topk, 12, 5, 0.2)
    row_map, offsets = O.plan(ids, 12)
    rows = torch.randn(tokens * topk, hidden, generator=gen).to(dtype)
    w = None if weight_dtype is None else torch.randn(tokens, topk, generator=gen).to(weight_dtype)
    plan = ops().MoePlan(row_map.cuda(), offsets.cuda())
    out = ops().moe_unpermute(rows.cuda(), plan, None if w is None else w.cuda())
    want, size = O.unpermute(rows, row_map, w)
    assert out.dtype == dtype
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert bool(((out.cpu().double() - want).abs() <= size * topk * 2.0 ** -24 * 1.01 + want.abs() * half_step(dtype) * 1.01 + tiny).all())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('weight_dtype', DTYPES)
@pytest.mark.parametrize('tokens,topk,hidden', [(1, 1, 8), (7, 9, 33), (300, 6, 256), (3, 20, 2048), (40, 8, 1000)])
def test_unpermute_backward(tokens, topk, hidden, dtype, weight_dtype):
    """grad_rows: one rounded product; grad_weights: an fp32 sum whose every partial sum (hidden / 256 per thread, then 13
    more) rounds by 2^-24 of at most the sum of magnitudes."""
    gen = torch.Generator().manual_seed(tokens + topk)
    ids = routing(tokens, topk, 12, 6, 0.2)
    row_map, offsets = O.plan(ids, 12)
    rows = torch.randn(tokens * topk, hidden, generator=gen).to(dtype)
    w = torch.randn(tokens, topk, generator=gen).to(weight_dtype)
    g = torch.randn(tokens, hidden, generator=gen).to(dtype)
    plan = ops().MoePlan(row_map.cuda(), offsets.cuda())
    gr, gw = ops().moe_unpermute_backward(g.cuda(), rows.cuda(), plan, w.cuda())
    want_r, want_w, size = O.unpermute_backward(g, rows, row_map, w)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert bool(((gr.cpu().double() - want_r).abs() <= want_r.abs() * (half_step(dtype) + 2.0 ** -24) * 1.01 + tiny).all())
    used = int(offsets[-1])
    assert not bool(gr[used:].any())
    steps = (hidden + 255) // 256 * 8 + 13
    assert gw.dtype == weight_dtype
    assert bool(((gw.cpu().double() - want_w).abs() <= size * steps * 2.0 ** -24 * 1.01 + want_w.abs() * half_step(weight_dtype) * 1.01).all())
    only_rows = ops().moe_unpermute_backward(g.cuda(), rows.cuda(), plan, w.cuda(), want_weights=False)
    only_weights = ops().moe_unpermute_backward(g.cuda(), rows.cuda(), plan, w.cuda(), want_rows=False)
    assert only_rows[1] is None and torch.equal(only_rows[0], gr) and only_weights[0] is None and torch.equal(only_weights[1], gw)


def test_rows_without_a_token_are_not_read():
    """NaN in rows that no assignment has, and a NaN weight of an assignment without a row, change nothing."""
    ids = torch.tensor([[0, -1], [1, 0]])
    row_map, offsets = O.plan(ids, 2)
    rows = torch.randn(4, 16, generator=torch.Generator().manual_seed(0))
    rows[3] = float('nan')
    w = torch.tensor([[0.5, float('nan')], [0.25, 0.75]])
    plan = ops().MoePlan(row_map.cuda(), offsets.cuda())
    out = ops().moe_unpermute(rows.cuda(), plan, w.cuda())
    assert bool(torch.isfinite(out).all())
    gr, gw = ops().moe_unpermute_backward(torch.ones(2, 16).cuda(), rows.cuda(), plan, w.cuda())
    assert bool(torch.isfinite(gr).all()) and bool(torch.isfinite(gw).all()) and float(gw[0, 1]) == 0


def test_empty_batches():
    o = ops()
    for tokens, hidden in ((0, 16), (3, 0)):
        x = torch.zeros(tokens, hidden).cuda()
        ids = torch.zeros(tokens, 2, dtype=torch.int64).cuda()
        rows, _, plan = o.moe_permute(x, ids, 4)
        assert rows.shape == (2 * tokens, hidden) and plan.offsets.tolist() == [0] + [2 * tokens] * 4
        assert o.moe_unpermute(rows, plan).shape == (tokens, hidden)
        w = torch.ones(tokens, 2).cuda()
        gr, gw = o.moe_unpermute_backward(x, rows, plan, w)
        assert gr.shape == rows.shape and gw.shape == w.shape and not bool(gw.any())


def test_refusals():
    o = ops()
    x, ids = torch.zeros(4, 8).cuda(), torch.zeros(4, 2, dtype=torch.int64).cuda()
    for args in ((x, ids[:3], 4), (x, ids.float(), 4), (x.double(), ids, 4), (x[0], ids, 4), (x, ids[:, :0], 4)):
        with pytest.raises(ValueError):
            o.moe_permute(*args)
    with pytest.raises(ValueError):
        o.moe_permute(x, ids, 4, scales=torch.zeros(3, 2).cuda())
    for experts in (0, 1025):
        with pytest.raises(o._l.BackendError):
            o.moe_permute(x, ids, experts)
    rows, _, plan = o.moe_permute(x, ids, 4)
    with pytest.raises(ValueError):
        o.moe_unpermute(rows[:5], plan)
    with pytest.raises(ValueError):
        o.moe_unpermute(rows, plan, torch.ones(4, 3).cuda())
    with pytest.raises(ValueError):
        o.moe_unpermute_backward(x[:2], rows, plan, torch.ones(4, 2).cuda())


# ------------------------------------------------------------------------------------------------- through autograd
def experts_module():
    from amct_b200.experimental.quantization.deepseek_v3_2 import experts
    return experts


def test_gradients_against_the_formula_and_against_differences():
    """sum(c * unpermute(permute(x) * scale_e, w)) in fp32: autograd of the kernels against autograd of plain torch
    operations in 64 bits, and against central differences of the kernels' own forward (the map is bilinear, so their only
    error is fp32 rounding: 2^-24 of the sum of magnitudes over the step)."""
    m = experts_module()
    gen = torch.Generator().manual_seed(21)
    tokens, topk, experts, hidden = 13, 3, 5, 24
    ids = routing(tokens, topk, experts, 8, 0.2)
    x = torch.randn(tokens, hidden, generator=gen)
    w = torch.rand(tokens, topk, generator=gen)
    c = torch.randn(tokens, hidden, generator=gen)
    factor = torch.randn(tokens * topk, 1, generator=gen)

    def loss(xx, ww):
        rows, plan = m.permute_tokens(xx, ids.cuda(), experts)
        return (m.unpermute_tokens(rows * factor.cuda(), plan, ww) * c.cuda()).double().sum()

    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    gx, gw = torch.autograd.grad(loss(xg, wg), (xg, wg))
    row_map, _ = O.plan(ids, experts)
    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    valid = row_map >= 0
    f = torch.where(valid, factor.double()[row_map.long().clamp(min=0), 0], torch.zeros((), dtype=torch.float64))
    want = (((x64[:, None, :] * f[:, :, None]) * w64[:, :, None]).sum(1) * c.double()).sum()
    ex, ew = torch.autograd.grad(want, (x64, w64))
    assert torch.allclose(gx.cpu().double(), ex, rtol=0, atol=float(ex.abs().max()) * 16 * 2.0 ** -24)
    assert torch.allclose(gw.cpu().double(), ew, rtol=0, atol=float((x.abs() @ c.abs().t()).max()) * float(factor.abs().max()) * 40 * 2.0 ** -24)
    h = 0.25
    size = float((x.abs()[:, None] * factor.abs().max() * w.abs()[:, :, None]).sum() * c.abs().max())
    for t, i in ((0, 0), (7, 5), (12, 23)):
        d = torch.zeros_like(x)
        d[t, i] = h
        diff = (loss((x + d).cuda(), wg) - loss((x - d).cuda(), wg)).item() / (2 * h)
        assert abs(diff - float(gx[t, i])) <= size * 2.0 ** -23 / h
    for t, j in ((0, 0), (9, 2)):
        d = torch.zeros_like(w)
        d[t, j] = h
        diff = (loss(xg, (w + d).cuda()) - loss(xg, (w - d).cuda())).item() / (2 * h)
        assert abs(diff - float(gw[t, j])) <= size * 2.0 ** -23 / h


def test_gradient_shortcuts():
    """Broadcast output gradients (stride 0), inputs that want no gradient, and rows used twice outside the operator."""
    m = experts_module()
    ids = routing(10, 2, 4, 3).cuda()
    x = torch.randn(10, 16, generator=torch.Generator().manual_seed(4)).cuda().requires_grad_()
    rows, plan = m.permute_tokens(x, ids, 4)
    y = m.unpermute_tokens(rows, plan, torch.ones(10, 2).cuda())
    y.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))
    w = torch.rand(10, 2).cuda().requires_grad_()
    m.unpermute_tokens(rows.detach(), plan, w).sum().backward()
    assert torch.allclose(w.grad, rows.detach()[plan.row_map.long()].sum(2), atol=1e-5)
    rows, plan = m.permute_tokens(x, ids, 4)
    y = m.unpermute_tokens(rows, plan) + m.unpermute_tokens(rows, plan)
    x.grad = None
    y.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 4.0))


def test_more_than_two_gigabytes_of_rows():
    """Row addresses beyond 32 bits, in bytes and in elements."""
    o = ops()
    tokens, topk, hidden = 1 << 15, 8, 16384
    x = torch.randint(0, 256, (tokens, hidden), dtype=torch.uint8, device='cuda')
    ids = torch.randint(0, 64, (tokens, topk), device='cuda')
    rows, _, plan = o.moe_permute(x, ids, 64)
    for t in (0, 1, tokens // 2, tokens - 1):
        assert torch.equal(rows[plan.row_map[t].long()], x[t].expand(topk, hidden))
    assert int(plan.row_map.max()) == tokens * topk - 1 and torch.equal(rows[-1], x[(plan.row_map == tokens * topk - 1).nonzero()[0, 0]])
    y = o.moe_unpermute(rows[:, :1].expand(-1, hidden)[:, :8].to(torch.float32), plan)
    assert torch.equal(y[:, 0], x[:, 0].float() * topk)


def test_backward_captured_and_replayed():
    """A training step's dispatch and combine inside a CUDA graph, replayed with other values and other routing."""
    m = experts_module()
    tokens, topk, experts, hidden = 30, 2, 4, 64
    x, w = torch.zeros(tokens, hidden, device='cuda', requires_grad=True), torch.zeros(tokens, topk, device='cuda', requires_grad=True)
    ids = torch.zeros(tokens, topk, dtype=torch.int64, device='cuda')
    c = torch.randn(tokens, hidden, device='cuda')

    def step():
        rows, plan = m.permute_tokens(x, ids, experts)
        return torch.autograd.grad((m.unpermute_tokens(rows, plan, w) * c).sum(), (x, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gx, gw = step()
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(tokens, hidden, generator=gen))
            w.copy_(torch.rand(tokens, topk, generator=gen))
            ids.copy_(torch.randint(-1, experts, (tokens, topk), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        want_x, want_w = step()
        assert torch.equal(gx, want_x) and torch.equal(gw, want_w)
