"""What the FP8 block-scaled and routed-expert operators compute, on which sizes, and in which plain form.

Operators (E4M3 codes with one fp32 scale per block of 128):
  quant      activations -> codes and one scale per token and 128 channels, optionally behind silu(gate) * up;
             weights -> codes and one scale per 128 x 128 tile
  gemm       out[m, n] = sum_kb sa[m, kb] * sb[n / 128, kb] * dot(a[m, kb], b[n, kb]) (+ bias[n])
  grouped    the same product for rows sorted by expert, each row with its expert's weight
  permute    tokens copied to rows sorted by expert, and the gradient with respect to the tokens
  unpermute  rows weighted and summed back to tokens, and the gradients with respect to rows and weights
"""
import math

import torch

own = False                     # False: plain torch forms; True: the framework's kernels

BLOCK = 128
E4M3_MAX = 448.0
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32, 'fp8': torch.float8_e4m3fn}


def listed():
    return [
        # a decode batch's hidden states ahead of a quantized Linear: latency
        {'name': 'quant_decode', 'op': 'quant', 'rows': 16, 'k': 7168, 'dtype': 'bf16', 'block': 'token', 'act': 'none', 'pow2': False},
        # the routed experts' gate / up outputs of a prefill: SwiGLU and quantization ahead of the down projection
        {'name': 'quant_swiglu_prefill', 'op': 'quant', 'rows': 16383, 'k': 2048, 'dtype': 'bf16', 'block': 'token', 'act': 'swiglu', 'pow2': False},
        # converting the gate / up weight of a 70B-shape layer
        {'name': 'quant_weight', 'op': 'quant', 'rows': 28672, 'k': 8192, 'dtype': 'bf16', 'block': 'tile', 'act': 'none', 'pow2': False},
        # one token through an 8B-shape gate or up projection: the weight is read once
        {'name': 'gemm_decode', 'op': 'gemm', 'm': 1, 'n': 14336, 'k': 4096, 'out': 'bf16', 'bias': False},
        # a chunk of a prompt, sizes that end inside every tile, with a bias
        {'name': 'gemm_ragged', 'op': 'gemm', 'm': 777, 'n': 5001, 'k': 4000, 'out': 'fp16', 'bias': True},
        # prefill of a large projection
        {'name': 'gemm_prefill', 'op': 'gemm', 'm': 8192, 'n': 7168, 'k': 8192, 'out': 'bf16', 'bias': False},
        # a decode batch over the experts one of eight ranks holds: a few rows for each expert
        {'name': 'grouped_decode', 'op': 'grouped', 'tokens': 16, 'topk': 8, 'experts': 32, 'n': 4096, 'k': 7168, 'out': 'bf16'},
        # a prefill over the same experts, groups of unequal length that end inside tiles
        {'name': 'grouped_prefill', 'op': 'grouped', 'tokens': 2047, 'topk': 8, 'experts': 32, 'n': 4096, 'k': 7168, 'out': 'bf16'},
        # serving: a decode batch's codes and scales, sorted by expert
        {'name': 'permute_decode', 'op': 'permute', 'tokens': 8, 'topk': 8, 'experts': 256, 'hidden': 7168, 'dtype': 'fp8', 'elsewhere': 0.0, 'train': False},
        # calibrating the experts: forward and backward, an odd number of tokens, some experts on other ranks
        {'name': 'permute_train', 'op': 'permute', 'tokens': 8191, 'topk': 8, 'experts': 256, 'hidden': 7168, 'dtype': 'bf16', 'elsewhere': 0.1, 'train': True},
        # a decode batch's expert outputs back to tokens
        {'name': 'unpermute_decode', 'op': 'unpermute', 'tokens': 32, 'topk': 8, 'experts': 256, 'hidden': 7168, 'dtype': 'bf16', 'elsewhere': 0.0, 'train': False},
        # calibrating the experts: forward, and the gradients of rows and routing weights
        {'name': 'unpermute_train', 'op': 'unpermute', 'tokens': 8192, 'topk': 6, 'experts': 64, 'hidden': 4096, 'dtype': 'fp16', 'elsewhere': 0.0, 'train': True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(['quant', 'gemm', 'grouped', 'permute', 'unpermute'])
    if op == 'quant':
        block = rng.choice(['token', 'token', 'tile'])
        return {'op': op, 'rows': _log(rng, 1, 20000), 'k': _log(rng, 64, 8192), 'dtype': rng.choice(['bf16', 'fp16', 'fp32']),
                'block': block, 'act': rng.choice(['none', 'swiglu']) if block == 'token' else 'none', 'pow2': rng.random() < 0.3}
    if op == 'gemm':
        return {'op': op, 'm': _log(rng, 1, 8192), 'n': _log(rng, 64, 7168), 'k': _log(rng, 128, 8192),
                'out': rng.choice(['bf16', 'bf16', 'fp16']), 'bias': rng.random() < 0.4}
    if op == 'grouped':
        return {'op': op, 'tokens': _log(rng, 1, 2047), 'topk': rng.randint(1, 8), 'experts': rng.choice([8, 16, 27, 32]),
                'n': _log(rng, 128, 4096), 'k': _log(rng, 256, 7168), 'out': rng.choice(['bf16', 'fp16'])}
    train = rng.random() < 0.5
    return {'op': op, 'tokens': _log(rng, 1, 8000), 'topk': rng.randint(1, 8), 'experts': _log(rng, 8, 256), 'hidden': _log(rng, 100, 7168),
            'dtype': rng.choice(['bf16', 'fp16', 'fp32'] if train or op == 'unpermute' else ['bf16', 'fp16', 'fp8']),
            'elsewhere': rng.choice([0.0, 0.0, 0.3]), 'train': train}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _blocks(k):
    return (k + BLOCK - 1) // BLOCK


def _activations(rows, k, gen):
    """Hidden states as they come in earnest: a few channels stand far out, tokens differ in size."""
    x = torch.randn(rows, k, generator=gen, device='cuda')
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device='cuda'))
    return x * torch.where(torch.rand(k, generator=gen, device='cuda') < 0.01, 20.0, 1.0)


def _in_rows_of_16(codes):
    """Codes in rows that begin at multiples of 16 bytes, as the quantizer lays them out."""
    *lead, k = codes.shape
    pad = (k + 15) // 16 * 16
    buf = torch.zeros(*lead, pad, dtype=torch.uint8, device=codes.device)
    buf[..., :k] = codes.view(torch.uint8)
    return buf.view(torch.float8_e4m3fn)[..., :k]


def _block_major(scale):
    """Token scales [rows, blocks] stored block by block, as the quantizer lays them out."""
    return scale.t().contiguous().t()


def _routing(tokens, topk, experts, gen, elsewhere=0.0):
    """Expert numbers of every token without repeats, some experts more popular than others; `elsewhere` of them are -1."""
    logits = torch.randn(tokens, experts, generator=gen, device='cuda') + 0.7 * torch.randn(experts, generator=gen, device='cuda')
    ids = torch.sort(logits, dim=1, descending=True).indices[:, :topk]
    if elsewhere:
        ids = torch.where(torch.rand(ids.shape, generator=gen, device='cuda') < elsewhere, -1, ids)
    return ids.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op = case['op']
    s = {'case': case}
    if op == 'quant':
        width = case['k'] * (2 if case['act'] == 'swiglu' else 1)
        if case['block'] == 'tile':
            x = 0.02 * torch.randn(case['rows'], width, generator=gen, device='cuda')
        else:
            x = _activations(case['rows'], width, gen)
        s['x'] = x.to(DTYPES[case['dtype']])
    elif op == 'gemm':
        codes, scale = _token_codes(_activations(case['m'], case['k'], gen))
        s['a'], s['a_scale'] = _in_rows_of_16(codes), _block_major(scale)
        codes, s['b_scale'] = _tile_codes(0.02 * torch.randn(case['n'], case['k'], generator=gen, device='cuda'))
        s['b'] = _in_rows_of_16(codes)
        s['bias'] = torch.randn(case['n'], generator=gen, device='cuda') if case['bias'] else None
    elif op == 'grouped':
        ids = _routing(case['tokens'], case['topk'], case['experts'], gen).reshape(-1)
        s['offsets'] = _offsets(ids, case['experts'])
        codes, scale = _token_codes(_activations(ids.numel(), case['k'], gen))
        s['a'], s['a_scale'] = _in_rows_of_16(codes), _block_major(scale)
        w = 0.02 * torch.randn(case['experts'] * case['n'], case['k'], generator=gen, device='cuda')
        codes, scale = _tile_codes(w.view(case['experts'], case['n'], case['k']))
        s['b'], s['b_scale'] = _in_rows_of_16(codes), scale
        s['longest'] = int((s['offsets'][1:] - s['offsets'][:-1]).max())      # for the plain form's padded product
    else:
        s['ids'] = _routing(case['tokens'], case['topk'], case['experts'], gen, case['elsewhere'])
        n = s['ids'].numel()
        dtype = DTYPES[case['dtype']]
        if op == 'permute':
            x = _activations(case['tokens'], case['hidden'], gen)
            if case['dtype'] == 'fp8':
                codes, scale = _token_codes(x)
                s['x'], s['scales'] = _in_rows_of_16(codes), _block_major(scale)
            else:
                s['x'] = x.to(dtype).requires_grad_(case['train'])
                if case['train']:
                    s['grad'] = torch.randn(n, case['hidden'], generator=gen, device='cuda').to(dtype)
        else:
            s['rows'] = torch.randn(n, case['hidden'], generator=gen, device='cuda').to(dtype).requires_grad_(case['train'])
            w = torch.rand(case['tokens'], case['topk'], generator=gen, device='cuda') + 0.05
            s['weights'] = (w / w.sum(1, keepdim=True)).requires_grad_(case['train'])
            s['row_map'], s['offsets'] = _sorted_places(s['ids'], case['experts'])
            if case['train']:
                s['grad'] = torch.randn(case['tokens'], case['hidden'], generator=gen, device='cuda').to(dtype)
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _block_scale(amax, pow2):
    """amax / 448; 1 where that is below the smallest normal number (a block of zeros); pow2: the next power of two."""
    scale = amax / E4M3_MAX
    if pow2:
        scale = torch.ldexp(torch.ones_like(scale), torch.ceil(torch.log2(scale.double())).to(torch.int32))
    return torch.where(amax / E4M3_MAX < torch.finfo(torch.float32).tiny, torch.ones_like(scale), scale)


def _token_codes(x, pow2=False):
    rows, k = x.shape
    kb = _blocks(k)
    y = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    scale = _block_scale(y.abs().amax(2), pow2)
    codes = (y / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.view(rows, kb * BLOCK)[:, :k], scale


def _tile_codes(w, pow2=False):
    *lead, n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    y = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(*lead, nb, BLOCK, kb, BLOCK)
    scale = _block_scale(y.abs().amax((-3, -1)), pow2)
    codes = (y / scale[..., :, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.view(*lead, nb * BLOCK, kb * BLOCK)[..., :n, :k], scale


def _spread(scale, n, k):
    """Tile scales [.., ceil(n / 128), ceil(k / 128)] -> one for each element."""
    return scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _offsets(ids, experts):
    counts = (ids[:, None] == torch.arange(experts, device=ids.device)).sum(0) if ids.numel() * experts < 1 << 26 else torch.bincount(ids[ids >= 0], minlength=experts)
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)


def _sorted_places(ids, experts):
    """(row of every assignment, -1 where it has none; the first row of every expert)."""
    flat = ids.reshape(-1)
    valid = (flat >= 0) & (flat < experts)
    order = torch.sort(torch.where(valid, flat, experts), stable=True).indices
    place = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=order.device))
    return torch.where(valid, place, -1).to(torch.int32).view(ids.shape), _offsets(flat, experts)


def _plain_permute(s):
    case, x = s['case'], s['x'].detach()
    row_map, offsets = _sorted_places(s['ids'], case['experts'])
    n, topk = s['ids'].numel(), case['topk']
    flat = row_map.reshape(-1).long()
    valid = flat >= 0
    to = torch.where(valid, flat, n)                                            # assignments without a row: one row too many
    source = torch.full((n + 1,), -1, device=x.device).scatter_(0, to, torch.arange(n, device=x.device) // topk)
    filled = torch.arange(n, device=x.device) < offsets[-1]
    source = torch.where(filled, source[:n], 0)

    def gathered(t):
        return torch.where(filled[:, None], t[source], torch.zeros((), dtype=t.dtype, device=t.device))

    out = {'row_map': row_map, 'offsets': offsets}
    if case['dtype'] == 'fp8':
        out['rows'] = gathered(x.view(torch.uint8)).view(torch.float8_e4m3fn)
        out['row_scales'] = gathered(s['scales'])
        return out
    out['rows'] = gathered(x)
    if case['train']:
        g = s['grad'][flat.clamp(min=0)].float() * valid[:, None]
        out['grad_x'] = g.view(case['tokens'], topk, -1).sum(1).to(x.dtype)
    return out


def _plain_unpermute(s):
    case, rows, w = s['case'], s['rows'].detach(), s['weights'].detach()
    n, flat = s['row_map'].numel(), s['row_map'].reshape(-1).long()
    valid = flat >= 0
    picked = (rows[flat.clamp(min=0)].float() * valid[:, None]).view(*w.shape, -1)
    out = {'out': (picked * w[:, :, None]).sum(1).to(rows.dtype)}
    if case['train']:
        g = s['grad'].float()[:, None, :]
        out['grad_weights'] = (g * picked).sum(2)
        grad_rows = torch.zeros(n + 1, rows.shape[1], device=rows.device)
        grad_rows[torch.where(valid, flat, n)] = (g * w[:, :, None]).view(n, -1)
        out['grad_rows'] = grad_rows[:n].to(rows.dtype)
    return out


def _plain(s):
    case = s['case']
    if case['op'] == 'quant':
        x = s['x'].float()
        if case['act'] == 'swiglu':
            gate, up = x[:, :case['k']], x[:, case['k']:]
            x = gate / (1 + torch.exp(-gate)) * up
        codes, scale = (_tile_codes if case['block'] == 'tile' else _token_codes)(x, case['pow2'])
        return {'codes': codes, 'scale': scale}
    if case['op'] in ('gemm', 'grouped'):
        n, k = case['n'], case['k']
        a = s['a'].float() * s['a_scale'].repeat_interleave(BLOCK, 1)[:, :k]
        b = s['b'].float() * _spread(s['b_scale'], n, k)
        if case['op'] == 'gemm':
            out = a @ b.t()
            if s['bias'] is not None:
                out = out + s['bias']
        else:                                                                   # one padded product for all experts
            row = torch.arange(a.shape[0], device=a.device)
            expert = (row[:, None] >= s['offsets'][1:]).sum(1)
            place = row - s['offsets'][expert]
            padded = a.new_zeros(case['experts'], s['longest'], k)
            padded[expert, place] = a
            out = torch.bmm(padded, b.transpose(1, 2))[expert, place]
        return {'out': out.to(DTYPES[case['out']])}
    return _plain_permute(s) if case['op'] == 'permute' else _plain_unpermute(s)


# ---------------------------------------------------------------------------------------------- the framework's operators
def _kernels(s):
    from amct_b200.backend import ops
    from amct_b200.experimental.quantization.deepseek_v3_2 import experts
    case = s['case']
    op = case['op']
    if op == 'quant':
        codes, scale = ops.fp8_block_quant(s['x'], block=case['block'], act=None if case['act'] == 'none' else case['act'], pow2_scale=case['pow2'])
        return {'codes': codes, 'scale': scale}
    if op == 'gemm':
        return {'out': ops.gemm_fp8_block(s['a'], s['a_scale'], s['b'], s['b_scale'], bias=s['bias'], out_dtype=DTYPES[case['out']])}
    if op == 'grouped':
        return {'out': ops.gemm_fp8_block_grouped(s['a'], s['a_scale'], s['offsets'], s['b'], s['b_scale'], out_dtype=DTYPES[case['out']])}
    if op == 'permute':
        if case['dtype'] == 'fp8':
            rows, row_scales, plan = ops.moe_permute(s['x'], s['ids'], case['experts'], scales=s['scales'])
            return {'rows': rows, 'row_scales': row_scales, 'row_map': plan.row_map, 'offsets': plan.offsets}
        rows, plan = experts.permute_tokens(s['x'], s['ids'], case['experts'])
        out = {'rows': rows.detach(), 'row_map': plan.row_map, 'offsets': plan.offsets}
        if case['train']:
            out['grad_x'], = torch.autograd.grad(rows, s['x'], s['grad'])
        return out
    y = experts.unpermute_tokens(s['rows'], ops.MoePlan(s['row_map'], s['offsets']), s['weights'])
    out = {'out': y.detach()}
    if case['train']:
        out['grad_rows'], out['grad_weights'] = torch.autograd.grad(y, (s['rows'], s['weights']), s['grad'])
    return out


def run(state):
    return _kernels(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def _round_e4m3(v):
    """Nearest E4M3 value, ties to even, saturating: steps of 2^(e - 3), e not below -6."""
    _, e = torch.frexp(v.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(v), e - 4)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_quant(case, x):
    k, rows, tile = case['k'], case['rows'], case['block'] == 'tile'
    codes = torch.empty(rows, k, dtype=torch.float64, device=x.device)
    scale = torch.empty(_blocks(rows) if tile else rows, _blocks(k), dtype=torch.float64, device=x.device)
    for r in range(0, rows, 1024):                                              # some rows at a time: 64 bits are large
        y = x[r:r + 1024].double()
        if case['act'] == 'swiglu':
            y = y[:, :k] * torch.sigmoid(y[:, :k]) * y[:, k:]
        for b in range(_blocks(k)):
            part = y[:, b * BLOCK:(b + 1) * BLOCK]
            if tile:
                top = torch.stack([p.abs().max() for p in part.split(BLOCK)])
            else:
                top = part.abs().max(1).values
            sc = top / E4M3_MAX
            if case['pow2']:
                sc = torch.where(sc > 0, 2.0 ** torch.ceil(torch.log2(sc)), sc)
            sc = torch.where(top / E4M3_MAX < 2.0 ** -126, 1.0, sc)
            first = r // BLOCK if tile else r
            scale[first:first + sc.numel(), b] = sc
            each = sc.repeat_interleave(BLOCK)[:part.shape[0]] if tile else sc
            codes[r:r + 1024, b * BLOCK:(b + 1) * BLOCK] = _round_e4m3(part / each[:, None])
    return {'codes': codes, 'scale': scale}


def _exact_product(a, a_scale, b, b_scale):
    k, n = a.shape[1], b.shape[0]
    out = torch.zeros(a.shape[0], n, dtype=torch.float64, device=a.device)
    per_row = b_scale.double()[torch.arange(n, device=a.device) // BLOCK]
    for c in range(0, k, 8 * BLOCK):                                            # eight blocks at a time
        kb = torch.arange(c, min(k, c + 8 * BLOCK), device=a.device) // BLOCK
        out += (a[:, c:c + 8 * BLOCK].double() * a_scale.double()[:, kb]) @ (b[:, c:c + 8 * BLOCK].double() * per_row[:, kb]).t()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op == 'quant':
        return _exact_quant(case, s['x'])
    if op == 'gemm':
        out = _exact_product(s['a'], s['a_scale'], s['b'], s['b_scale'])
        return {'out': out if s['bias'] is None else out + s['bias'].double()}
    if op == 'grouped':
        at = s['offsets'].tolist()
        return {'out': torch.cat([_exact_product(s['a'][at[e]:at[e + 1]], s['a_scale'][at[e]:at[e + 1]], s['b'][e], s['b_scale'][e])
                                  for e in range(case['experts'])])}
    ids = s['ids'].tolist()
    by_expert = [[] for _ in range(case['experts'])]
    for t, chosen in enumerate(ids):
        for j, e in enumerate(chosen):
            if 0 <= e < case['experts']:
                by_expert[e].append((t, j))
    order = [place for group in by_expert for place in group]
    token = torch.tensor([t for t, _ in order], dtype=torch.long, device='cuda')
    slot = torch.tensor([j for _, j in order], dtype=torch.long, device='cuda')
    n, total = s['ids'].numel(), len(order)
    if op == 'permute':
        x = s['x'].detach().double()
        rows = torch.zeros(n, case['hidden'], dtype=torch.float64, device='cuda')
        rows[:total] = x[token]
        out = {'rows': rows}
        if case['dtype'] == 'fp8':
            out['row_scales'] = torch.zeros(n, s['scales'].shape[1], dtype=torch.float64, device='cuda')
            out['row_scales'][:total] = s['scales'].double()[token]
        if case['train']:
            out['grad_x'] = torch.zeros_like(x).index_add_(0, token, s['grad'][:total].double())
        return out
    rows, w = s['rows'].detach()[:total].double(), s['weights'].detach().double()
    y = torch.zeros(case['tokens'], case['hidden'], dtype=torch.float64, device='cuda')
    out = {'out': y.index_add_(0, token, rows * w[token, slot][:, None])}
    if case['train']:
        g = s['grad'].double()[token]
        out['grad_rows'] = torch.zeros(n, case['hidden'], dtype=torch.float64, device='cuda')
        out['grad_rows'][:total] = g * w[token, slot][:, None]
        out['grad_weights'] = torch.zeros_like(w)
        out['grad_weights'][token, slot] = (g * rows).sum(1)
    return out


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    op = case['op']
    if op == 'quant':
        rows, k = case['rows'], case['k']
        size = DTYPES[case['dtype']].itemsize * (2 if case['act'] == 'swiglu' else 1)
        scales = _blocks(rows) * _blocks(k) if case['block'] == 'tile' else rows * _blocks(k)
        return {'bytes': rows * k * (size + 1) + 4 * scales, 'flops': 0}
    if op == 'gemm':
        m, n, k = case['m'], case['n'], case['k']
        return {'bytes': m * k + n * k + 4 * (m + _blocks(n)) * _blocks(k) + 2 * m * n + (4 * n if case['bias'] else 0), 'flops': 2 * m * n * k}
    if op == 'grouped':
        rows, n, k, experts = case['tokens'] * case['topk'], case['n'], case['k'], case['experts']
        used = experts * (1 - (1 - 1 / experts) ** rows)                        # experts with a row, for even routing
        return {'bytes': int(rows * k + used * n * k + 4 * (rows + used * _blocks(n)) * _blocks(k) + 2 * rows * n), 'flops': 2 * rows * n * k}
    size = DTYPES[case['dtype']].itemsize
    tokens, hidden, n = case['tokens'], case['hidden'], case['tokens'] * case['topk']
    total = n * (1 - case['elsewhere'])
    token_bytes, all_bytes, row_bytes = tokens * hidden * size, n * hidden * size, int(total * hidden * size)
    ids = 8 * n + 4 * n + 4 * (case['experts'] + 1)
    if op == 'permute':
        if case['dtype'] == 'fp8':
            token_bytes, all_bytes = token_bytes + 4 * tokens * _blocks(hidden), all_bytes + 4 * n * _blocks(hidden)
        back = row_bytes + token_bytes if case['train'] else 0
        return {'bytes': token_bytes + all_bytes + ids + back, 'flops': int(total * hidden) if case['train'] else 0}
    forward = row_bytes + token_bytes + 4 * n + 4 * n
    back = token_bytes + row_bytes + all_bytes + 8 * n if case['train'] else 0
    return {'bytes': forward + back, 'flops': int(total * hidden) * (5 if case['train'] else 2)}
