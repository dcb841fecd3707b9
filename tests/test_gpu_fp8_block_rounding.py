"""The E4M3 block quantizer to the last bit of a code: the sign of a zero, and silu(g) u over the whole range of gates."""
import pytest
import torch

from oracle import fp8_block as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def ops():
    from amct_b200.backend import ops as o
    return o


def bytes_of(codes):
    return codes.cpu().contiguous().view(torch.uint8)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('block', ['token', 'tile'])
@pytest.mark.parametrize('pow2', [False, True])
@pytest.mark.parametrize('rows,k', [(4, 128), (3, 200), (5, 131), (6000, 136)])
def test_a_zero_keeps_its_sign(rows, k, block, dtype, pow2):
    """Byte for byte: -0 / s is -0, and so is what underflows below zero."""
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(k)).to(dtype)
    x[:, ::3] = -0.0
    x[:, 1::6] = 0.0
    x[1::2, 2::5] = -6e-8                          # far below half a step of the smallest code
    x[-1] = -0.0                                   # a block of zeros: scale 1
    codes, scale = ops().fp8_block_quant(x.cuda(), block=block, pow2_scale=pow2)
    want, want_s = (O.quant_tokens if block == 'token' else O.quant_tiles)(x, pow2)
    assert torch.equal(scale.cpu(), want_s) and torch.equal(bytes_of(codes), bytes_of(want))
    assert int((bytes_of(codes) == 0x80).sum()) > rows * k // 4


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [4, 6000])
def test_a_zero_behind_swiglu_keeps_its_sign(rows, dtype):
    """silu(g) u of zeros has the sign of g times that of u."""
    k = 128
    signs = torch.tensor([0.0, -0.0])
    g = signs.repeat(k // 2).expand(rows, k).clone()
    u = signs.repeat_interleave(2).repeat(k // 4).expand(rows, k).clone()
    u[:, 8:16] = 3.0
    u[:, 16:24] = -3.0
    g[:, 24:32] = 2.0
    g[:, 32:40] = -2.0
    codes, _ = ops().fp8_block_quant(torch.cat([g, u], 1).to(dtype).cuda(), act='swiglu')
    want = torch.where(torch.signbit(g) != torch.signbit(u), 0x80, 0).to(torch.uint8)
    zero = (g == 0) | (u == 0)
    assert torch.equal(bytes_of(codes)[zero], want[zero])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [3, 2000])
@pytest.mark.parametrize('low,high', [(-4.0, 4.0), (-86.9, -4.0), (-88.7, -87.1), (4.0, 200.0)])
def test_swiglu_error_does_not_grow_with_the_gate(low, high, rows, dtype):
    """One pair in every block, so that the block's scale is |silu(g) u| / 448.  The exponential's documented error is 2 units of
    2^-23; six further steps (its correction, 1 + exp, quotient, its remainder's rest, times u, the scale's division) round by at
    most 2^-24 each; the correction's ln 2 is off by 2.75e-9 of itself, which costs |g| times that.  silu's own sensitivity to
    the exponential is at most 1."""
    gen = torch.Generator().manual_seed(rows)
    blocks = 24
    g = torch.rand(rows, blocks, generator=gen) * (high - low) + low
    u = torch.exp(torch.randn(rows, blocks, generator=gen)) * (1e4 if dtype == torch.float16 else 1e8)
    u = u.clamp(max=6e4) if dtype == torch.float16 else u
    g, u = g.to(dtype), u.to(dtype)
    x = torch.zeros(rows, 2, blocks, 128, dtype=dtype)
    at = torch.randint(0, 128, (blocks,), generator=gen)
    x[:, 0, torch.arange(blocks), at] = g
    x[:, 1, torch.arange(blocks), at] = u
    _, scale = ops().fp8_block_quant(x.view(rows, -1).cuda(), act='swiglu')
    want = (g.double() * torch.sigmoid(g.double()) * u.double()).abs() / 448
    assert float(want.min()) > 2.0 ** -126
    bound = 2.0 ** -22 + 6 * 2.0 ** -24 + g.double().abs() * 2.8e-9
    assert bool(((scale.cpu().double() - want).abs() <= want * bound).all())
