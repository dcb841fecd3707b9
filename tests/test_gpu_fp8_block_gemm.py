"""The product of E4M3 operands with a scale for each block of 128, dense and grouped by expert, against the 64-bit
restatement (oracle/fp8_block.py).

Tolerance.  With S = sum over all terms of |a_scale b_scale a b|: the tensor core sums the 128 products of a K block (each
exact: 8 significant bits) with at least 13 bits kept below the largest term, so the blocks' sums are off by at most
2^-13 S altogether; every one of the K / 128 fused steps that fold them rounds by at most 2^-24 S, the product of the two
scales by 2^-24 S, the bias and the cluster's joins by 2^-24 S each; the result is rounded once.  Small whole numbers
with power-of-two scales are exact in all of these steps, and are tested for equality."""
import pytest
import torch

from oracle import fp8_block as O

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def ops():
    from amct_b200.backend import ops as o
    return o


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, size, k, dtype):
    bound = size * (2.0 ** -13 + ((k + 127) // 128 + 12) * 2.0 ** -24) + want.abs() * half_step(dtype) * 1.01
    top = torch.finfo(dtype).max
    g = got.cpu().double()
    return bool(((g - want).abs() <= bound + torch.finfo(dtype).tiny).all()) if float(want.abs().max() if want.numel() else 0) < top else False


def operands(m, n, k, seed):
    gen = torch.Generator().manual_seed(seed)
    a, a_scale = O.quant_tokens(torch.randn(m, k, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen)))
    b, b_scale = O.quant_tiles(torch.randn(n, k, generator=gen) * 0.05 * torch.exp(torch.randn(n, 1, generator=gen)))
    return a, a_scale, b, b_scale


def whole(rows, k, gen, lo=-2, hi=3):
    return torch.randint(lo, hi, (rows, k), generator=gen).float().to(F8)


def pow2(shape, gen):
    return 2.0 ** torch.randint(-3, 4, shape, generator=gen).float()


def cuda(*tensors):
    return [t.cuda() for t in tensors]


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 8, 16), (3, 130, 100), (15, 127, 256), (16, 256, 144), (17, 300, 1000), (32, 128, 4096), (33, 129, 384),
          (64, 1000, 512), (65, 257, 640), (127, 64, 128), (128, 384, 2048), (129, 256, 128), (200, 513, 1040), (300, 1000, 272), (777, 700, 1536),
          (1, 2048, 7168), (40, 4100, 2100)]


@pytest.mark.parametrize('m,n,k', SHAPES)
def test_whole_numbers_are_exact(m, n, k):
    gen = torch.Generator().manual_seed(m * 31 + n * 7 + k)
    a, b = whole(m, k, gen), whole(n, k, gen)
    a_scale, b_scale = pow2((m, O.blocks(k)), gen), pow2((O.blocks(n), O.blocks(k)), gen)
    bias = torch.randint(-8, 9, (n,), generator=gen).float()
    want, _ = O.product(a, a_scale, b, b_scale, bias)
    got = ops().gemm_fp8_block(*cuda(a, a_scale, b, b_scale), bias=bias.cuda(), out_dtype=torch.float32)
    assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize('m,n,k', SHAPES)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('bias_dtype', [None, torch.bfloat16, torch.float32])
def test_product(m, n, k, dtype, bias_dtype):
    a, a_scale, b, b_scale = operands(m, n, k, m + n + k)
    bias = None if bias_dtype is None else torch.randn(n, generator=torch.Generator().manual_seed(1)).to(bias_dtype)
    want, size = O.product(a, a_scale, b, b_scale, bias)
    got = ops().gemm_fp8_block(*cuda(a, a_scale, b, b_scale), bias=None if bias is None else bias.cuda(), out_dtype=dtype)
    assert got.dtype == dtype and close(got, want, size, k, dtype)
    again = ops().gemm_fp8_block(*cuda(a, a_scale, b, b_scale), bias=None if bias is None else bias.cuda(), out_dtype=dtype)
    assert torch.equal(got, again)


def test_the_quantizer_s_layout_and_a_whole_linear():
    """x and w through the quantizers and the product as a user runs them; the same bits whatever the scales' strides."""
    gen = torch.Generator().manual_seed(3)
    for m, n, k in ((5, 300, 520), (150, 260, 1000), (1, 128, 128)):
        x, w = torch.randn(m, k, generator=gen).bfloat16(), (torch.randn(n, k, generator=gen) * 0.1).bfloat16()
        xc, xs = ops().fp8_block_quant(x.cuda())
        wc, ws = ops().fp8_block_quant(w.cuda(), block='tile')
        got = ops().gemm_fp8_block(xc, xs, wc, ws)
        want, size = O.product(*O.quant_tokens(x), *O.quant_tiles(w))
        assert close(got, want, size, k, torch.bfloat16)
        for a_s in (xs.contiguous(), torch.stack([xs, xs], 2)[:, :, 1]):
            for b_s in (ws.t().contiguous().t(), ws.contiguous()):
                assert torch.equal(ops().gemm_fp8_block(xc, a_s, wc, b_s), got)


def test_codes_in_other_layouts():
    a, a_scale, b, b_scale = cuda(*operands(20, 140, 256, 9))
    want = ops().gemm_fp8_block(a, a_scale, b, b_scale)
    wide = torch.zeros(20, 300, dtype=torch.uint8).cuda()
    wide[:, 5:261] = a.view(torch.uint8)
    assert torch.equal(ops().gemm_fp8_block(wide[:, 5:261], a_scale, b, b_scale), want)                 # unaligned rows, uint8
    assert torch.equal(ops().gemm_fp8_block(a.view(torch.uint8).t().contiguous().t(), a_scale, b, b_scale), want)
    big = torch.zeros(40, 272, dtype=torch.uint8).cuda()
    big[::2, :256] = a.view(torch.uint8)
    assert torch.equal(ops().gemm_fp8_block(big.view(F8)[::2, :256], a_scale, b, b_scale), want)


@pytest.mark.parametrize('m', [3, 70, 260])
def test_out_is_written_where_it_should_be_and_nowhere_else(m):
    a, a_scale, b, b_scale = cuda(*operands(m, 133, 256, m))
    want = ops().gemm_fp8_block(a, a_scale, b, b_scale)
    for width, first in ((133, 0), (140, 0), (200, 16), (151, 7)):
        buf = torch.full((m + 2, width), 7.0, dtype=torch.bfloat16).cuda()
        out = buf[1:-1, first:first + 133]
        assert ops().gemm_fp8_block(a, a_scale, b, b_scale, out=out) is out
        assert torch.equal(out, want)
        buf[1:-1, first:first + 133] = 7.0
        assert bool((buf == 7).all())


# tiles enough that the 128 x 256 kernel takes them; every remainder of columns and rows that its stores treat apart
MANY_TILES = [(70, 9601, 256), (500, 2435, 300), (777, 1502, 1100), (1300, 900, 272), (1290, 1024, 4300), (9500, 33, 128), (4900, 160, 130),
              (2405, 512, 640), (9473, 1, 48)]


@pytest.mark.parametrize('m,n,k', MANY_TILES)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('bias_dtype', [None, torch.float16])
def test_product_of_many_tiles(m, n, k, dtype, bias_dtype):
    test_product(m, n, k, dtype, bias_dtype)


@pytest.mark.parametrize('m,n,k', MANY_TILES)
def test_whole_numbers_of_many_tiles_are_exact(m, n, k):
    test_whole_numbers_are_exact(m, n, k)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('n', [1, 31, 32, 33, 64, 95, 96, 97, 127, 128, 129, 160, 224, 255, 256, 257, 389])
def test_out_of_many_tiles_is_written_where_it_should_be_and_nowhere_else(n, dtype):
    """Rows of `out` that begin at any element and lie any distance apart."""
    m = 9600 if n <= 128 else 4900
    a, a_scale, b, b_scale = cuda(*operands(m, n, 128, n))
    want = ops().gemm_fp8_block(a, a_scale, b, b_scale, out_dtype=torch.float32).to(dtype)
    for width, first in ((n, 0), (n + 1, 0), (n + 1, 1), (n + 5, 2), (n + 8 - n % 8, 0), (n + 15 - n % 8, 3)):
        buf = torch.full((m + 2, width), 7.0, dtype=dtype).cuda()
        out = buf[1:-1, first:first + n]
        ops().gemm_fp8_block(a, a_scale, b, b_scale, out=out)
        assert torch.equal(out, want)
        buf[1:-1, first:first + n] = 7.0
        assert bool((buf == 7).all())


@pytest.mark.parametrize('m', [4, 140])
def test_nan_codes_and_scales(m):
    a, a_scale, b, b_scale = operands(m, 200, 300, 2)
    a.view(torch.uint8)[2, 150] = 0x7f
    b_scale[1, 2] = float('inf')
    got = ops().gemm_fp8_block(*cuda(a, a_scale, b, b_scale)).cpu()
    assert bool(torch.isnan(got[2]).all())
    keep = [i for i in range(m) if i != 2]
    assert bool(torch.isfinite(got[keep][:, :128]).all()) and not bool(torch.isfinite(got[keep][:, 128:]).any())


def test_empty_and_refused():
    o = ops()
    a, a_scale, b, b_scale = cuda(*operands(4, 130, 256, 1))
    assert o.gemm_fp8_block(a[:0], a_scale[:0], b, b_scale).shape == (0, 130)
    assert o.gemm_fp8_block(a, a_scale, b[:0], b_scale[:0]).shape == (4, 0)
    for bad in ((a.float(), a_scale, b, b_scale), (a, a_scale[:, :1], b, b_scale), (a, a_scale, b, b_scale[:1]), (a, a_scale.double(), b, b_scale),
                (a[:, :128], a_scale[:, :1], b, b_scale), (a[0], a_scale, b, b_scale), (a[:, :0], a_scale[:, :0], b[:, :0], b_scale[:, :0])):
        with pytest.raises(ValueError):
            o.gemm_fp8_block(*bad)
    with pytest.raises(ValueError):
        o.gemm_fp8_block(a, a_scale, b, b_scale, bias=torch.zeros(129).cuda())
    with pytest.raises(ValueError):
        o.gemm_fp8_block(a, a_scale, b, b_scale, out_dtype=torch.int32)
    with pytest.raises(ValueError):
        o.gemm_fp8_block(a, a_scale, b, b_scale, out=torch.empty(130, 4, dtype=torch.bfloat16).cuda().t())
    with pytest.raises(o._l.BackendError):
        o.gemm_fp8_block(a.cpu(), a_scale, b, b_scale)
    with pytest.raises(ValueError):
        o.gemm_fp8_block_grouped(a, a_scale, torch.zeros(3, dtype=torch.int32).cuda(), b[None], b_scale[None])
    with pytest.raises(ValueError):
        o.gemm_fp8_block_grouped(a, a_scale, torch.zeros(2, dtype=torch.int64).cuda(), b[None], b_scale[None])


# --------------------------------------------------------------------------------------------------------- grouped
def grouped_operands(rows, experts, n, k, seed):
    gen = torch.Generator().manual_seed(seed)
    a, a_scale = O.quant_tokens(torch.randn(rows, k, generator=gen))
    parts = [O.quant_tiles(torch.randn(n, k, generator=gen) * 0.1) for _ in range(experts)]
    return a, a_scale, torch.stack([p[0].view(torch.uint8) for p in parts]).view(F8), torch.stack([p[1] for p in parts])


GROUPS = {
    'even': [0, 5, 10, 15, 20], 'empty_groups': [0, 0, 17, 17, 33], 'one_expert_has_all': [0, 0, 0, 90, 90], 'none': [0, 0, 0, 0, 0],
    'tail': [0, 3, 3, 40, 77], 'late_start': [9, 12, 60, 61, 300], 'long': [0, 300, 301, 1000, 1003], 'tile_edges': [0, 128, 256, 257, 512],
    'sixteens': [0, 16, 32, 33, 65],
}


@pytest.mark.parametrize('offsets', list(GROUPS.values()), ids=list(GROUPS))
@pytest.mark.parametrize('n,k', [(128, 256), (130, 400), (300, 128)])
@pytest.mark.parametrize('more', [0, 13])
def test_grouped(offsets, n, k, more):
    rows = max(1, offsets[-1] + more)
    a, a_scale, b, b_scale = grouped_operands(rows, 4, n, k, rows + n)
    out = torch.full((rows, n), 7.0, dtype=torch.bfloat16).cuda()
    at = torch.tensor(offsets, dtype=torch.int32).cuda()
    got = ops().gemm_fp8_block_grouped(*cuda(a, a_scale), at, *cuda(b, b_scale), out=out)
    assert got is out
    for e in range(4):
        lo, hi = offsets[e], offsets[e + 1]
        want, size = O.product(a[lo:hi], a_scale[lo:hi], b[e], b_scale[e])
        assert close(got[lo:hi], want, size, k, torch.bfloat16)
    assert bool((got[:offsets[0]] == 7).all()) and bool((got[offsets[-1]:] == 7).all())


@pytest.mark.parametrize('rows', [40, 1500])
def test_grouped_offsets_out_of_order_stay_inside(rows):
    """Descending or out-of-range offsets are clamped to a running maximum within the rows."""
    a, a_scale, b, b_scale = grouped_operands(rows, 5, 130, 256, 3)
    at = torch.tensor([-4, 20, 10, 30, rows + 500, 2], dtype=torch.int32).cuda()
    got = ops().gemm_fp8_block_grouped(*cuda(a, a_scale), at, *cuda(b, b_scale))
    for e, (lo, hi) in enumerate([(0, 20), (20, 20), (20, 30), (30, rows), (rows, rows)]):
        want, size = O.product(a[lo:hi], a_scale[lo:hi], b[e], b_scale[e])
        assert close(got[lo:hi], want, size, 256, torch.bfloat16)


@pytest.mark.parametrize('rows', [700, 3000])
def test_grouped_many_experts(rows):
    gen = torch.Generator().manual_seed(rows)
    experts, n, k = 1024, 16, 64
    cuts = torch.sort(torch.randint(0, rows + 1, (experts - 1,), generator=gen)).values
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([rows])]).to(torch.int32)
    a, b = whole(rows, k, gen), whole(experts * n, k, gen).view(experts, n, k)
    a_scale, b_scale = pow2((rows, 1), gen), pow2((experts, 1, 1), gen)
    got = ops().gemm_fp8_block_grouped(*cuda(a, a_scale, offsets, b, b_scale), out_dtype=torch.float32).cpu().double()
    expert = torch.searchsorted(offsets[1:].contiguous().long(), torch.arange(rows), right=True)
    want = torch.einsum('rk,rnk->rn', a.double() * a_scale.double(), b.double()[expert] * b_scale.double()[expert])
    assert torch.equal(got, want)


def test_grouped_weights_that_are_not_packed():
    a, a_scale, b, b_scale = cuda(*grouped_operands(50, 4, 130, 250, 8))
    at = torch.tensor([0, 10, 20, 45, 50], dtype=torch.int32).cuda()
    want = ops().gemm_fp8_block_grouped(a, a_scale, at, b, b_scale)
    wide = torch.zeros(4, 140, 272, dtype=torch.uint8).cuda()
    wide[:, :130, :250] = b.view(torch.uint8)
    spread = torch.stack([b_scale, b_scale], 3)[..., 0]
    assert torch.equal(ops().gemm_fp8_block_grouped(a, a_scale, at, wide.view(F8)[:, :130, :250], spread), want)


# ------------------------------------------------------------------------------------------- streams, graphs, modules
def test_other_streams_and_two_at_once():
    first, second = operands(8, 512, 1024, 1), operands(400, 512, 1024, 2)
    a, b = cuda(*first), cuda(*second)
    want_a, want_b = ops().gemm_fp8_block(*a), ops().gemm_fp8_block(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            got.append((ops().gemm_fp8_block(*a), want_a))
        with torch.cuda.stream(s2):
            got.append((ops().gemm_fp8_block(*b), want_b))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in got)


def test_expert_layer_matches_its_parts_and_replays_from_a_graph():
    """FP8RoutedExperts: sorted tokens, both grouped products, SwiGLU with quantization and the weighted sum, against the
    same chain expert by expert through the dense product; captured and replayed with other inputs."""
    from amct_b200.experimental.quantization.deepseek_v3_2.experts import FP8RoutedExperts
    o = ops()
    gen = torch.Generator().manual_seed(12)
    experts, hidden, inter, topk = 6, 256, 128, 3
    gu = [o.fp8_block_quant((torch.randn(2 * inter, hidden, generator=gen) * 0.1).cuda(), block='tile') for _ in range(experts)]
    dn = [o.fp8_block_quant((torch.randn(hidden, inter, generator=gen) * 0.1).cuda(), block='tile') for _ in range(experts)]
    layer = FP8RoutedExperts(torch.stack([c.view(torch.uint8) for c, _ in gu]).view(F8), torch.stack([s for _, s in gu]),
                             torch.stack([c.view(torch.uint8) for c, _ in dn]).view(F8), torch.stack([s for _, s in dn]), first_expert=2)

    def by_hand(x, ids, w):
        out = torch.zeros_like(x, dtype=torch.float64)
        for e in range(experts):
            t, j = torch.nonzero(ids.cpu() == e + 2, as_tuple=True)
            if t.numel():
                t, j = t.cuda(), j.cuda()
                h = o.gemm_fp8_block(*o.fp8_block_quant(x[t]), *gu[e])
                y = o.gemm_fp8_block(*o.fp8_block_quant(h, act='swiglu'), *dn[e])
                out.index_add_(0, t, y.double() * w[t, j].double()[:, None])
        return out

    def inputs(tokens, seed):
        g = torch.Generator().manual_seed(seed)
        return (torch.randn(tokens, hidden, generator=g).bfloat16().cuda(), torch.randint(0, experts + 4, (tokens, topk), generator=g).cuda(),
                torch.rand(tokens, topk, generator=g).cuda())

    for tokens in (1, 5, 200, 900):
        x, ids, w = inputs(tokens, tokens)
        got, want = layer.moe_infer(x, ids, w), by_hand(x, ids, w)
        # the products' tiles differ between the two routes, so a sum may fall on the other side of a code's border:
        # compared by norm, at one code step (2^-3) for one value in a hundred at most plus bf16's rounding
        assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -3 * 0.1 + 2.0 ** -8
    x, ids, w = inputs(40, 1)
    layer(x, ids, w)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, ids, w)
    with torch.cuda.graph(other):
        z = layer(x, ids, w)
    for seed in (5, 6):
        nx, ni, nw = inputs(40, seed)
        x.copy_(nx), ids.copy_(ni), w.copy_(nw)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = layer(nx, ni, nw)
        assert torch.equal(y, want) and torch.equal(z, want)


def test_status_word_stays_clear():
    a, a_scale, b, b_scale = cuda(*operands(30, 300, 1000, 1))
    word = torch.zeros(1, dtype=torch.int32).cuda()
    ops().gemm_fp8_block(a, a_scale, b, b_scale, status=word)
    ops().raise_if_timed_out(word)
    assert int(word) == 0


def test_more_than_two_thousand_million_outputs():
    """Output addresses beyond 32 bits: the last rows of a 70000 x 32768 result."""
    gen = torch.Generator(device='cuda').manual_seed(1)
    m, n, k = 70000, 32768, 128
    a = torch.randint(0, 2, (m, k), generator=gen, device='cuda').float().to(F8)
    b = torch.randint(0, 2, (n, k), generator=gen, device='cuda').float().to(F8)
    a_scale, b_scale = torch.ones(m, 1).cuda(), torch.ones(n // 128, 1).cuda()
    got = ops().gemm_fp8_block(a, a_scale, b, b_scale)
    for r in (0, m // 2, m - 1):
        assert torch.equal(got[r].float(), b.float() @ a[r].float())


@pytest.mark.parametrize('rows', [60, 2000])
def test_grouped_captured_and_replayed_with_other_offsets(rows):
    a, a_scale, b, b_scale = cuda(*grouped_operands(rows, 4, 130, 256, 5))
    at = torch.tensor([0, 10, 20, 30, 60], dtype=torch.int32).cuda()
    out = torch.zeros(rows, 130, dtype=torch.bfloat16).cuda()
    ops().gemm_fp8_block_grouped(a, a_scale, at, b, b_scale, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops().gemm_fp8_block_grouped(a, a_scale, at, b, b_scale, out=out)
    for cuts in ([0, 0, 50, 50, rows], [5, 6, 7, 40, 59]):
        at.copy_(torch.tensor(cuts, dtype=torch.int32))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = ops().gemm_fp8_block_grouped(a, a_scale, at, b, b_scale, out=torch.full_like(out, 7))
        assert torch.equal(out, want)
