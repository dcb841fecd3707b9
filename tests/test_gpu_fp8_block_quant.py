"""E4M3 block quantization against the CPU restatement (oracle/fp8_block.py): codes and scales bit for bit, except behind
SwiGLU, whose fp32 product is held to the rounding of its steps."""
import pytest
import torch

from oracle import fp8_block as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def ops():
    from amct_b200.backend import ops as o
    return o


def same_codes(got, want):
    """Equal values; NaN where NaN (its sign is no information)."""
    g, w = got.cpu().float(), want.float()
    return torch.equal(torch.isnan(g), torch.isnan(w)) and torch.equal(torch.nan_to_num(g), torch.nan_to_num(w))


def same_scale(got, want):
    g = got.cpu()
    return g.shape == want.shape and torch.equal(torch.isnan(g), torch.isnan(want)) and torch.equal(torch.nan_to_num(g, posinf=1e38), torch.nan_to_num(want, posinf=1e38))


def make(rows, k, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=gen) * torch.exp(3 * torch.randn(rows, 1, generator=gen))
    x = x.clamp(-6e4, 6e4)
    if rows > 2:
        x[1] = 0
        x[2] *= 1e-6
    return x.to(dtype)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('pow2', [False, True])
@pytest.mark.parametrize('rows,k', [(1, 1), (1, 128), (2, 129), (3, 127), (5, 136), (4, 1000), (7, 300), (33, 512), (130, 264)])
def test_token_codes(rows, k, dtype, pow2):
    x = make(rows, k, dtype, rows * 1000 + k)
    codes, scale = ops().fp8_block_quant(x.cuda(), pow2_scale=pow2)
    want_c, want_s = O.quant_tokens(x, pow2)
    assert codes.shape == x.shape and codes.dtype == torch.float8_e4m3fn and (rows == 1 or codes.stride(0) % 16 == 0)
    assert same_scale(scale, want_s) and same_codes(codes, want_c)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('pow2', [False, True])
@pytest.mark.parametrize('n,k', [(1, 1), (128, 128), (129, 136), (100, 250), (300, 384), (257, 1000)])
def test_tile_codes(n, k, dtype, pow2):
    w = make(n, k, dtype, n + k)
    codes, scale = ops().fp8_block_quant(w.cuda(), block='tile', pow2_scale=pow2)
    want_c, want_s = O.quant_tiles(w, pow2)
    assert same_scale(scale, want_s) and same_codes(codes, want_c)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [3, 5000])
def test_extreme_magnitudes(dtype, rows):
    """Blocks whose scale is subnormal (becomes 1), near the border where the quotient leaves the normal range, and large."""
    exps = {torch.float16: [-24, -20, -14, 0, 14], torch.bfloat16: [-133, -126, -118, -100, -82, -80, 0, 100, 127], torch.float32: [-149, -130, -117, -90, -81, 0, 100, 127]}[dtype]
    gen = torch.Generator().manual_seed(5)
    x = torch.cat([(torch.randn(rows, 128, generator=gen).double().clamp(-1.9, 1.9) * 2.0 ** e) for e in exps], 1).to(dtype)
    codes, scale = ops().fp8_block_quant(x.cuda())
    want_c, want_s = O.quant_tokens(x)
    assert same_scale(scale, want_s) and same_codes(codes, want_c)


def test_rounding_ties():
    """Quotients that lie exactly between two codes (scale 1 exactly) go to the even one."""
    steps = torch.arange(0, 2 ** 11, dtype=torch.float32) / 2 ** 10            # all ties of the subnormal range and beyond
    vals = torch.cat([steps, torch.tensor([1.0625, 1.1875, 17.0, 19.0, 23.0, 432.0, 400.0, 416.0])])
    vals = torch.cat([vals, -vals])
    x = torch.zeros((vals.numel() + 126) // 127 * 127)
    x[:vals.numel()] = vals
    x = torch.cat([x.view(-1, 127), torch.full((x.numel() // 127, 1), 448.0)], 1)
    codes, scale = ops().fp8_block_quant(x.cuda())
    want_c, want_s = O.quant_tokens(x)
    assert bool((want_s == 1).all()) and same_scale(scale, want_s) and same_codes(codes, want_c)


@pytest.mark.parametrize('block', ['token', 'tile'])
def test_nan_and_infinity_stay_in_their_block(block):
    x = torch.randn(256, 384, generator=torch.Generator().manual_seed(2))
    x[3, 200] = float('nan')
    x[140, 300] = float('inf')
    codes, scale = ops().fp8_block_quant(x.cuda(), block=block)
    want_c, want_s = (O.quant_tokens if block == 'token' else O.quant_tiles)(x)
    assert same_scale(scale, want_s) and same_codes(codes, want_c)
    assert int((~torch.isfinite(scale)).sum()) == 2


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,k', [(1, 128), (5, 100), (9, 264), (700, 1024)])
def test_swiglu(rows, k, dtype):
    """v = silu(g) u in fp32.  The kernel's exponential and reciprocal are off by at most 2 + 1.4 |g| and 1 units of 2^-23
    (documented bounds of the fast functions and the rounding of -g log2(e)), the three other steps by 2^-24 each; silu's
    own sensitivity to exp is at most 1.  So v is within (4 + 1.4 |g|) 2^-23 of the exact value, and a code within half its
    step of v / scale plus that, times 448 at the top of the range."""
    x = make(rows, 2 * k, dtype, 7 * rows + k)
    codes, scale = ops().fp8_block_quant(x.cuda(), act='swiglu')
    g, u = x[:, :k].double(), x[:, k:].double()
    exact = g * torch.sigmoid(g) * u
    off = exact.abs() * (4 + 1.4 * g.abs()) * 2.0 ** -23 + 1e-38
    pad = O.blocks(k) * 128 - k

    def by_block(t):
        return torch.nn.functional.pad(t, (0, pad)).view(rows, -1, 128)

    top = by_block(exact).abs().amax(2)
    far = by_block(off).amax(2)
    s = scale.cpu().double()
    expect = torch.where(top / 448 < 2.0 ** -126, torch.ones_like(top), top / 448)
    assert bool(((s - expect).abs() <= far / 448 + expect * 2.0 ** -23).all())
    got = codes.cpu().double()
    sc = s.repeat_interleave(128, 1)[:, :k]
    q = exact / sc
    step = 2.0 ** (torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    assert bool(((got - q).abs() <= step / 2 * (1 + 1e-6) + off / sc + q.abs() * 2.0 ** -22).all())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [1, 2500])
def test_swiglu_gates_far_below_zero(dtype, rows):
    """silu is below 1e-80 for gates under -200, down to the type's lowest value: codes and scales are those of gates of zero,
    whatever the other half holds.  An infinite gate below zero is inf / inf, as in the formula."""
    gen = torch.Generator().manual_seed(rows)
    k = 384
    x = torch.randn(rows, 2 * k, generator=gen).to(dtype)
    x[:, k:] = (x[:, k:].float() * 100).to(dtype)
    low = [torch.finfo(dtype).min, torch.finfo(dtype).min / 1024, -2000.0, -200.0]
    zero = x.clone()
    for i in range(0, k, 5):
        x[:, i] = low[i % 4]
        zero[:, i] = 0
    codes, scale = ops().fp8_block_quant(x.cuda(), act='swiglu')
    want_c, want_s = ops().fp8_block_quant(zero.cuda(), act='swiglu')
    assert same_scale(scale, want_s.cpu()) and same_codes(codes, want_c.cpu())
    x[0, 130] = -float('inf')
    x[-1, 300] = float('inf')
    scale = ops().fp8_block_quant(x.cuda(), act='swiglu')[1].cpu()
    assert torch.isnan(scale[0, 1]) and torch.isinf(scale[-1, 2]) and int((~torch.isfinite(scale)).sum()) == 2


def test_strided_and_unaligned_inputs():
    base = make(40, 900, torch.bfloat16, 4).cuda()
    for view in (base[:, 3:700], base[::2, 8:520], base[:, ::2], base.t()[:300], base[5:6, 1:130]):
        codes, scale = ops().fp8_block_quant(view)
        want_c, want_s = O.quant_tokens(view.cpu())
        assert same_scale(scale, want_s) and same_codes(codes, want_c)
        codes, scale = ops().fp8_block_quant(view, block='tile')
        want_c, want_s = O.quant_tiles(view.cpu())
        assert same_scale(scale, want_s) and same_codes(codes, want_c)


@pytest.mark.parametrize('shape', [(256,), (2, 3, 256), (2, 3, 130), (0, 64), (2, 0, 64), (130,)])
def test_shapes(shape):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1))
    codes, scale = ops().fp8_block_quant(x.cuda())
    assert codes.shape == x.shape
    rows = x.numel() // shape[-1]
    assert tuple(scale.shape) == (rows, O.blocks(shape[-1]))
    if x.numel():
        want_c, want_s = O.quant_tokens(x.reshape(rows, -1))
        assert same_codes(codes.reshape(rows, -1), want_c) and same_scale(scale, want_s)


def test_refusals():
    o = ops()
    x = torch.randn(4, 130).cuda()
    for kwargs in ({'block': 'row'}, {'act': 'gelu'}, {'block': 'tile', 'act': 'swiglu'}):
        with pytest.raises(ValueError):
            o.fp8_block_quant(x, **kwargs)
    with pytest.raises(ValueError):
        o.fp8_block_quant(torch.randn(4, 129).cuda(), act='swiglu')
    with pytest.raises(ValueError):
        o.fp8_block_quant(torch.randn(2, 4, 128).cuda(), block='tile')
    with pytest.raises(o._l.BackendError):
        o.fp8_block_quant(x.double())
