"""CompressedLinear: a Linear whose parameters are the compressed form of its
weight; the dense weight is rebuilt on the GPU the first time it is needed.

Behaviour follows linear/compressed_linear.py:33-109 of the reference: a module
converted with `from_linear` carries exactly the parameters named by its
compressor's `compression_param_info` (plus the scales / zero points of its
scheme), is marked COMPRESSED, and turns FROZEN once its first forward call has
decompressed the weight.  Parameters live on the module's own device: there is
no offloading layer here.

With `keep_packed` (no counterpart in the reference) the module stays COMPRESSED: its weight
remains a quarter of the dense one's size, a forward call of few rows multiplies the packed
codes (`packed_linear`), and one of many rows decompresses the weight for that call.
"""
import warnings
from typing import Optional

import torch
from torch import Tensor
from torch.nn import Linear, Parameter
from torch.nn import functional as F

from compressed_tensors_amd import _lib
from compressed_tensors_amd.compressors.base import BaseCompressor
from compressed_tensors_amd.config import CompressionFormat, QuantizationStatus
from compressed_tensors_amd.linear.packed import packed_linear
from compressed_tensors_amd.quantization.initialize import initialize_module_for_quantization
from compressed_tensors_amd.quantization.quant_scheme import QuantizationScheme

__all__ = ["CompressedLinear"]


def _frozen(data: Tensor) -> Parameter:
    return Parameter(data, requires_grad=False)


# From here on decompressing first is faster.  Measured on one MI355X (us, packed against
# decompress and multiply): 4096 x 14336, 128 rows 37 : 100, 256 64 : 86, 384 110 : 102;
# 28672 x 4096, 128 rows 70 : 101, 192 100 : 110, 256 130 : 115.
_PACKED_ROWS = 192


class _PackedProduct(torch.autograd.Function):
    """packed_linear where nothing but the bias is differentiated"""

    @staticmethod
    def forward(input, weight_packed, weight_scale, weight_zero_point, bias):
        return packed_linear(input, weight_packed, weight_scale, weight_zero_point, bias)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, grad):
        return None, None, None, None, grad.reshape(-1, grad.shape[-1]).sum(0)


class CompressedLinear(Linear):
    #: multiply with the packed weight and never materialise it; set by `from_linear`
    keep_packed = False

    def __init__(self, *args, **kwargs) -> None:
        warnings.warn(
            "a CompressedLinear built by its constructor holds a dense weight and no "
            "compressor; convert an existing Linear with CompressedLinear.from_linear()",
            UserWarning,
            stacklevel=2,
        )
        super().__init__(*args, **kwargs)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, module: Linear, quantization_scheme: QuantizationScheme,
                    quantization_format: str, keep_packed: bool = False) -> "CompressedLinear":
        """Convert `module` in place (the same object is returned): its dense weight
        is replaced by uninitialised parameters with the compressed format's names,
        shapes and dtypes, ready to be filled from a compressed checkpoint.

        keep_packed: see the module's description; `pack-quantized` weights of 4 bits with
        groups of a multiple of 32 columns or one scale per row, no activation ordering."""
        if keep_packed:
            reason = why_not_kept_packed(module, quantization_scheme.weights, quantization_format)
            if reason is not None:
                raise NotImplementedError(reason)
        compressor = BaseCompressor.load_from_registry(quantization_format)
        dense_shape, device = module.weight.shape, module.weight.device

        module.__class__ = cls
        module.compressor = compressor
        initialize_module_for_quantization(module, quantization_scheme, force_zero_point=False)
        layout = compressor.compression_param_info(dense_shape, quantization_scheme.weights)
        module._swap_weight_for(layout, device)
        module.quantization_status = QuantizationStatus.COMPRESSED
        module.keep_packed = keep_packed
        return module

    def _swap_weight_for(self, layout, device) -> None:
        """drop the dense weight (and anything the compressed layout redefines), then
        register one empty parameter per entry of the layout"""
        for stale in {"weight", *layout}:
            if stale in self._parameters:
                del self._parameters[stale]
        for name, (shape, dtype) in layout.items():
            self.register_parameter(name, _frozen(torch.empty(shape, dtype=dtype, device=device)))

    def _materialise_weight(self) -> None:
        self.register_parameter("weight", _frozen(self.compressor.decompress_module(self)))
        self.quantization_status = QuantizationStatus.FROZEN

    def _forward_packed(self, input: Tensor) -> Tensor:
        zero_point = getattr(self, "weight_zero_point", None)
        if self.quantization_scheme.weights.symmetric:
            zero_point = None
        bias = self.bias
        # (what F.linear casts to inside autocast, and what it does not)
        cast = torch.is_autocast_enabled("cuda") and input.dtype is not torch.float64
        dtype = torch.get_autocast_dtype("cuda") if cast else input.dtype
        if (input.numel() <= _PACKED_ROWS * self.in_features and dtype in (torch.bfloat16, torch.float16)
                and not _lib.differentiated(input) and not _lib.has_tangent(bias)):
            if cast:
                input, bias = input.to(dtype), None if bias is None else bias.to(dtype)
            # (loading a checkpoint makes scales that require grad; here, too, they are constants)
            learns = bias is not None and bias.requires_grad and torch.is_grad_enabled()
            product = _PackedProduct.apply if learns else packed_linear
            return product(input, self.weight_packed, self.weight_scale.detach(), zero_point, bias)
        weight = self.compressor.decompress_weight(
            {"weight_packed": self.weight_packed, "weight_scale": self.weight_scale, "weight_zero_point": zero_point,
             "weight_shape": (self.out_features, self.in_features)}, self.quantization_scheme.weights)
        return F.linear(input, weight.to(input.dtype), self.bias)  # scales may be of another type

    def forward(self, input: Tensor) -> Tensor:
        if self.quantization_status == QuantizationStatus.COMPRESSED:
            if self.keep_packed:
                return self._forward_packed(input)
            self._materialise_weight()
        return F.linear(input, self.weight, self.bias)


def why_not_kept_packed(module: Linear, args, quantization_format: str) -> Optional[str]:
    """what keeps the product with packed weights from reading this one; None: nothing does"""
    if quantization_format != CompressionFormat.pack_quantized.value or args is None or args.num_bits != 4 or args.type != "int":
        return "keep_packed needs a pack-quantized 4-bit integer weight"
    if getattr(args, "actorder", None) is not None and str(getattr(args.actorder, "value", args.actorder)) == "group":
        return "keep_packed does not take weights with activation ordering"
    strategy = str(getattr(args.strategy, "value", args.strategy))
    if strategy == "group" and args.group_size % 32 == 0 and module.in_features % args.group_size == 0:
        return None
    if strategy != "channel":
        return (f"keep_packed needs one scale per row or groups of a multiple of 32 columns that divide "
                f"{module.in_features}, got {strategy} {args.group_size}")
    return None
