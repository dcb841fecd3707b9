import torch

from ..backend import ops


class KeepsBufferTypes(torch.nn.Module):
    """Module whose buffers change their device but never their type: ``.half()`` or ``.to(torch.bfloat16)`` of the model
    around it would turn codes into numbers and round the scales.  The ones named in ``code_buffers`` keep the layout that the
    products read, which copies (to another device, for instance) drop."""
    code_buffers = ()

    def _apply(self, fn, recurse=True):
        before = dict(self._buffers)
        super()._apply(fn, recurse)
        for name, old in before.items():
            new = self._buffers[name]
            if old is not None and new.dtype != old.dtype:
                self._buffers[name] = old.to(new.device)
        for name in self.code_buffers:
            self._buffers[name] = ops.fp8_code_rows(self._buffers[name])
        return self


class FP8BlockLinear(KeepsBufferTypes):
    """Linear on E4M3 codes with one fp32 scale for each block of 128: weights per 128 x 128 tile, activations per token
    and 128 channels at run time.

    Buffers, named and laid out as in the FP8 checkpoints that
    amct_pytorch/experimental/quantization/DeepSeekV3.2/deploy.py:48-90 reads, so that such a checkpoint's tensors load as
    they are: ``weight`` float8_e4m3fn [N, K], ``weight_scale_inv`` fp32 [ceil(N / 128), ceil(K / 128)] (what a code is
    multiplied by), ``bias`` fp32 [N] or None.  forward(): ``fp8_block_quant`` of the activations, then ``gemm_fp8_block``;
    output in the input's dtype.  Inference only, like every deploy module here.  ``pow2_scale``: activation scales are
    powers of two (checkpoints whose config says scale_fmt ue8m0).  The reference dequantizes these weights and has no
    Linear on them.
    """
    code_buffers = ('weight',)

    def __init__(self, quant_module):
        super().__init__()
        weight, scale = ops.fp8_block_quant(quant_module.weight.data, block='tile', pow2_scale=quant_module.pow2_scale)
        self._set(weight, scale, None if quant_module.bias is None else quant_module.bias.data, quant_module.pow2_scale)

    def _set(self, weight, scale, bias, pow2_scale):
        n, k = weight.shape
        if tuple(scale.shape) != (-(-n // 128), -(-k // 128)):
            raise ValueError(f'weight_scale_inv must have one value for each 128 x 128 tile of the weight {tuple(weight.shape)}')
        self.register_buffer('weight', ops.fp8_code_rows(weight.view(torch.float8_e4m3fn)))
        self.register_buffer('weight_scale_inv', scale.to(torch.float32).contiguous())
        self.register_buffer('bias', None if bias is None else bias.to(torch.float32))
        self.pow2_scale = pow2_scale

    @classmethod
    def from_checkpoint(cls, weight, weight_scale_inv, bias=None, pow2_scale=False):
        """The module for a checkpoint's own tensors: E4M3 codes (float8_e4m3fn or uint8) [N, K] and their tile scales."""
        module = cls.__new__(cls)
        torch.nn.Module.__init__(module)
        module._set(weight, weight_scale_inv, bias, pow2_scale)
        return module

    @torch.no_grad()
    def forward(self, x):
        x2 = x.reshape(-1, x.shape[-1])
        codes, scale = ops.fp8_block_quant(x2, pow2_scale=self.pow2_scale)
        out = ops.gemm_fp8_block(codes, scale, self.weight, self.weight_scale_inv, bias=self.bias, out_dtype=x.dtype)
        return out.reshape(*x.shape[:-1], self.weight.shape[0])
