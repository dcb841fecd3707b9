"""FP8 block quantization, the product of its operands, and the routing of tokens to experts, restated on the CPU.

Codes and scales follow the kernels' fp32 steps and are compared bit for bit; products and sums are formed in 64 bits.
The format is that of the checkpoints amct_pytorch/experimental/quantization/DeepSeekV3.2/deploy.py:48-90 reads; the routing is
that of modeling_deepseek_v3_2.py:522-611 of the same tree, written as plain loops.
"""
import torch

BLOCK, E4M3_MAX, TINY = 128, 448.0, 2.0 ** -126


def blocks(k):
    return (k + BLOCK - 1) // BLOCK


def block_scale(amax, pow2=False):
    """fp32 amax -> fp32 scale."""
    s = amax / torch.tensor(E4M3_MAX, dtype=torch.float32)
    p = torch.where(torch.isfinite(s) & (s > 0), 2.0 ** torch.ceil(torch.log2(s.double())), s.double()).float() if pow2 else s
    return torch.where(s < TINY, torch.ones_like(s), p)


def _codes(x, scale):
    return (x / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def quant_tokens(x, pow2=False):
    x = x.float()
    rows, k = x.shape
    scale = torch.empty(rows, blocks(k))
    codes = torch.empty(rows, k, dtype=torch.float8_e4m3fn)
    for b in range(blocks(k)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        scale[:, b] = block_scale(part.abs().amax(1), pow2)
        codes[:, b * BLOCK:(b + 1) * BLOCK] = _codes(part, scale[:, b:b + 1])
    return codes, scale


def quant_tiles(w, pow2=False):
    w = w.float()
    n, k = w.shape
    scale = torch.empty(blocks(n), blocks(k))
    codes = torch.empty(n, k, dtype=torch.float8_e4m3fn)
    for i in range(blocks(n)):
        for b in range(blocks(k)):
            part = w[i * BLOCK:(i + 1) * BLOCK, b * BLOCK:(b + 1) * BLOCK]
            scale[i, b] = block_scale(part.abs().amax(), pow2)
            codes[i * BLOCK:(i + 1) * BLOCK, b * BLOCK:(b + 1) * BLOCK] = _codes(part, scale[i, b])
    return codes, scale


def dequant_tokens(codes, scale):
    k = codes.shape[1]
    return codes.double() * scale.double().repeat_interleave(BLOCK, 1)[:, :k]


def dequant_tiles(codes, scale):
    n, k = codes.shape
    return codes.double() * scale.double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def product(a, a_scale, b, b_scale, bias=None):
    """(value, sum of magnitudes) in 64 bits."""
    x, w = dequant_tokens(a, a_scale), dequant_tiles(b, b_scale)
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def plan(ids, experts):
    """(row_map, offsets) for expert numbers [T, topk]."""
    tokens, topk = ids.shape
    row_map = torch.full((tokens, topk), -1, dtype=torch.int32)
    offsets = torch.zeros(experts + 1, dtype=torch.int32)
    groups = [[] for _ in range(experts)]
    for t, chosen in enumerate(ids.tolist()):
        for j, e in enumerate(chosen):
            if 0 <= e < experts:
                groups[e].append((t, j))
    at = 0
    for e, group in enumerate(groups):
        for t, j in group:
            row_map[t, j] = at
            at += 1
        offsets[e + 1] = at
    return row_map, offsets


def permute(x, row_map):
    rows = torch.zeros(row_map.numel(), *x.shape[1:], dtype=x.dtype)
    for t, places in enumerate(row_map.tolist()):
        for r in places:
            if r >= 0:
                rows[r] = x[t]
    return rows


def unpermute(rows, row_map, weights=None):
    """(value, sum of magnitudes) in 64 bits."""
    out = torch.zeros(row_map.shape[0], rows.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    for t, places in enumerate(row_map.tolist()):
        for j, r in enumerate(places):
            if r >= 0:
                term = rows[r].double() * (1.0 if weights is None else float(weights[t, j]))
                out[t] += term
                size[t] += term.abs()
    return out, size


def unpermute_backward(grad, rows, row_map, weights):
    """(grad_rows, grad_weights, sum of magnitudes of grad_weights) in 64 bits."""
    grad_rows = torch.zeros(rows.shape, dtype=torch.float64)
    grad_weights = torch.zeros(row_map.shape, dtype=torch.float64)
    size = torch.zeros_like(grad_weights)
    for t, places in enumerate(row_map.tolist()):
        for j, r in enumerate(places):
            if r >= 0:
                grad_rows[r] = grad[t].double() * float(weights[t, j])
                terms = grad[t].double() * rows[r].double()
                grad_weights[t, j], size[t, j] = terms.sum(), terms.abs().sum()
    return grad_rows, grad_weights, size
