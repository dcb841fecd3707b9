"""Routed experts of an FP8 checkpoint: tokens sorted by expert, the experts' products, and the weighted sum back.

``permute_tokens`` / ``unpermute_tokens`` are the dispatch and combine steps of ``DeepseekV3MoE.moe_infer``
(amct_pytorch/experimental/quantization/DeepSeekV3.2/cores/models/deepseek_v3_2/modeling_deepseek_v3_2.py:522-611),
with gradients, so that the calibration of the reference (cores/calibrator/dsv3_calib.py:60-186, which trains clip
factors through the expert layers) can run through them.  ``FP8RoutedExperts`` keeps the experts' weights in the
checkpoint's own format -- E4M3 codes and one fp32 scale for each 128 x 128 tile, what ``deploy.weight_dequant``
dequantizes -- and runs the two products of every expert on them.
"""
import torch
from torch.autograd import forward_ad as _forward_ad

from ....backend import ops as _ops
from ....deploy_op.fp8_block_linear import KeepsBufferTypes


class _Permute(torch.autograd.Function):
    """rows alone: the plan leaves through `plan_out`, because every further output costs the backward pass a tensor of zeros
    for its missing gradient (two launches here)."""

    @staticmethod
    def forward(ctx, x, expert_ids, num_experts, plan_out):
        rows, _, plan = _ops.moe_permute(x, expert_ids, num_experts)
        ctx.save_for_backward(plan.row_map)
        plan_out.append(plan)
        return rows

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_rows):
        (row_map,) = ctx.saved_tensors
        return _ops.moe_unpermute(grad_rows, _ops.MoePlan(row_map, None)), None, None, None


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, row_map, offsets):
        # the rows are read for the weights' gradient alone
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weights, row_map, offsets)
        return _ops.moe_unpermute(rows, _ops.MoePlan(row_map, offsets), weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        rows, weights, row_map, offsets = ctx.saved_tensors
        grad_rows, grad_weights = _ops.moe_unpermute_backward(
            grad_out, rows, _ops.MoePlan(row_map, offsets), weights, want_rows=ctx.needs_input_grad[0],
            want_weights=ctx.needs_input_grad[1])
        return grad_rows, grad_weights, None, None


def _refuse_forward_mode(name, *tensors):
    """A dual tensor need not require a gradient: past the autograd functions its tangent would be dropped in silence."""
    for t in tensors:
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f'{name} has no forward-mode derivative')


def permute_tokens(x, expert_ids, num_experts):
    """(rows, plan): rows[plan.row_map[t, j]] = x[t], sorted by expert; see ``ops.moe_permute``.  Differentiable in x
    (fp32 / fp16 / bf16), in reverse mode and once."""
    _refuse_forward_mode('permute_tokens', x)
    if not (torch.is_grad_enabled() and x.requires_grad):
        rows, _, plan = _ops.moe_permute(x, expert_ids, num_experts)
        return rows, plan
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f'no gradient for {x.dtype}')
    plan_out = []
    rows = _Permute.apply(x, expert_ids, num_experts, plan_out)
    return rows, plan_out[0]


def unpermute_tokens(rows, plan, weights=None):
    """out[t] = sum_j weights[t, j] * rows[plan.row_map[t, j]] for the plan of ``permute_tokens``; see
    ``ops.moe_unpermute``.  Differentiable in rows and weights, in reverse mode and once."""
    _refuse_forward_mode('unpermute_tokens', rows, weights)
    if not (torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad))):
        return _ops.moe_unpermute(rows, plan, weights)
    _ops.check_moe_offsets(plan)
    return _Unpermute.apply(rows, weights, plan.row_map, plan.offsets)


class FP8RoutedExperts(KeepsBufferTypes):
    """The routed experts of one layer on a checkpoint's FP8 weights: down(silu(gate(x)) * up(x)) of every chosen
    expert, weighted and summed (``moe_infer`` of the reference with its experts' Linears in FP8; inference only).

    Buffers: ``gate_up_weight`` float8_e4m3fn [E, 2 I, H] (gate rows, then up rows), ``gate_up_scale`` fp32
    [E, 2 I / 128, H / 128], ``down_weight`` [E, H, I], ``down_scale``.  Activations are quantized per token and 128
    channels ahead of both products.  ``first_expert``: number of the first expert held here; assignments to experts
    of other ranks add nothing.  ``pow2_scale``: activation scales are powers of two (checkpoints whose config says
    scale_fmt ue8m0)."""
    code_buffers = ('gate_up_weight', 'down_weight')

    def __init__(self, gate_up_weight, gate_up_scale, down_weight, down_scale, first_expert=0, pow2_scale=False):
        super().__init__()
        experts, width, hidden = gate_up_weight.shape if gate_up_weight.dim() == 3 else (0, 1, 0)
        if width % 256 or tuple(down_weight.shape) != (experts, hidden, width // 2):
            raise ValueError('gate_up_weight must be [E, 2 I, H] with I a multiple of 128, down_weight [E, H, I]')
        for name, codes, scale in (('gate_up', gate_up_weight, gate_up_scale), ('down', down_weight, down_scale)):
            tiles = (experts, -(-codes.shape[1] // 128), -(-codes.shape[2] // 128))
            if codes.dtype not in (torch.float8_e4m3fn, torch.uint8):
                raise ValueError(f'{name}_weight must hold E4M3 codes (float8_e4m3fn or uint8), not {codes.dtype}')
            if scale.dtype != torch.float32 or tuple(scale.shape) != tiles:
                raise ValueError(f'{name}_scale must be float32 with one value for each 128 x 128 tile, {tiles}')
        self.register_buffer('gate_up_weight', _ops.fp8_code_rows(gate_up_weight))
        self.register_buffer('gate_up_scale', gate_up_scale)
        self.register_buffer('down_weight', _ops.fp8_code_rows(down_weight))
        self.register_buffer('down_scale', down_scale)
        self.first_expert, self.pow2_scale = first_expert, pow2_scale

    @classmethod
    def from_checkpoint(cls, tensors, prefix, expert_numbers, first_expert=None, pow2_scale=False, device='cuda'):
        """From the checkpoint's tensors ``{prefix}.{e}.gate_proj.weight`` / ``.weight_scale_inv`` (and up_proj,
        down_proj) for the given expert numbers, which are consecutive.  ``first_expert`` is the first of them and need not be
        given."""
        expert_numbers = [int(e) for e in expert_numbers]
        if not expert_numbers or expert_numbers != list(range(expert_numbers[0], expert_numbers[0] + len(expert_numbers))):
            raise ValueError(f'expert_numbers must be consecutive numbers, at least one, not {expert_numbers}')
        if first_expert is None:
            first_expert = expert_numbers[0]
        elif first_expert != expert_numbers[0]:
            raise ValueError(f'first_expert is {first_expert}, the first of expert_numbers {expert_numbers[0]}')

        def stacked(*names):
            parts = [[tensors[f'{prefix}.{e}.{n}'].to(device) for n in names] for e in expert_numbers]
            codes = [[t.view(torch.uint8) if t.element_size() == 1 else t for t in p] for p in parts]
            return torch.stack([torch.cat(p) if len(p) > 1 else p[0] for p in codes])

        gate_up = stacked('gate_proj.weight', 'up_proj.weight').view(torch.float8_e4m3fn)
        down = stacked('down_proj.weight').view(torch.float8_e4m3fn)
        gate_up_scale = stacked('gate_proj.weight_scale_inv', 'up_proj.weight_scale_inv').float()
        return cls(gate_up, gate_up_scale, down, stacked('down_proj.weight_scale_inv').float(), first_expert, pow2_scale)

    @torch.no_grad()
    def moe_infer(self, x, topk_ids, topk_weight):
        """x [T, H], topk_ids [T, topk] (numbers among all experts), topk_weight [T, topk] -> [T, H] in x's dtype."""
        experts = self.gate_up_weight.shape[0]
        ids = topk_ids - self.first_expert if self.first_expert else topk_ids
        codes, scale = _ops.fp8_block_quant(x, pow2_scale=self.pow2_scale)
        rows, row_scale, plan = _ops.moe_permute(codes, ids, experts, scales=scale)
        h = _ops.gemm_fp8_block_grouped(rows, row_scale, plan.offsets, self.gate_up_weight, self.gate_up_scale, out_dtype=x.dtype)
        codes, scale = _ops.fp8_block_quant(h, act='swiglu', pow2_scale=self.pow2_scale)
        y = _ops.gemm_fp8_block_grouped(codes, scale, plan.offsets, self.down_weight, self.down_scale, out_dtype=x.dtype)
        return _ops.moe_unpermute(y, plan, topk_weight)

    def forward(self, x, topk_ids, topk_weight):
        return self.moe_infer(x, topk_ids, topk_weight)
