"""Products with a weight that stays packed: y = x @ W.T + b from the entries of a
`pack-quantized` 4-bit checkpoint, without the dense weight ever being written.

The reference decompresses the weight before its first product
(linear/compressed_linear.py:96-109); there is no counterpart of this call in it.
"""
from typing import Optional

import torch
from torch import Tensor

from compressed_tensors_amd import _lib

__all__ = ["packed_linear"]

_SCALES = (torch.bfloat16, torch.float16, torch.float32)


def packed_linear(x: Tensor, weight_packed: Tensor, weight_scale: Tensor,
                  weight_zero_point: Optional[Tensor] = None, bias: Optional[Tensor] = None) -> Tensor:
    """x [..., in_features] (bfloat16 or float16) times a packed 4-bit weight.

    weight_packed     int32 [out_features, ceil(in_features / 8)]
    weight_scale      [out_features, groups]: groups of a multiple of 32 columns each, or one
                      for the whole row
    weight_zero_point the packed zero points of an asymmetric scheme, int32
                      [ceil(out_features / 8), groups]; None for a symmetric one
    bias              [out_features] of x's type

    The result has x's type.  Sums are held in fp32, codes enter the product as the integers
    they are and nothing is rounded before the end, so it differs from
    `x @ decompress(weight).T`, whose weights are rounded to the scale's type first, by that
    rounding.  Forward only: a call that autograd would have to differentiate is refused
    (decompress the weight for it).
    """
    if x.ndim < 1 or weight_packed.ndim != 2 or weight_scale.ndim != 2:
        raise ValueError(f"expected x [..., in], weight_packed [out, words] and weight_scale [out, groups], got "
                         f"{tuple(x.shape)}, {tuple(weight_packed.shape)} and {tuple(weight_scale.shape)}")
    n, k = weight_packed.shape[0], x.shape[-1]
    groups = weight_scale.shape[1]
    if weight_packed.dtype is not torch.int32:
        raise ValueError(f"Expected {torch.int32} but got {weight_packed.dtype}, Aborting unpack.")
    if x.dtype is not torch.bfloat16 and x.dtype is not torch.float16:
        raise NotImplementedError(f"activations must be bfloat16 or float16, got {x.dtype}")
    if weight_scale.dtype not in _SCALES:
        raise NotImplementedError(f"scales of {weight_scale.dtype} are not supported")
    if k < 1 or weight_packed.shape[1] != (k + 7) // 8:
        raise ValueError(f"{k} columns need {(k + 7) // 8} words a row, weight_packed has {weight_packed.shape[1]}")
    if weight_scale.shape[0] != n or groups < 1 or k % groups:
        raise ValueError(f"scales {tuple(weight_scale.shape)} do not fit a [{n}, {k}] weight")
    if _lib.differentiated(x, weight_scale, bias):
        raise NotImplementedError("packed_linear has no backward and no forward-mode derivative: decompress the "
                                  "weight to differentiate, or call it under torch.no_grad() with plain tensors")
    if weight_zero_point is not None:
        if weight_zero_point.dtype is not torch.int32 or tuple(weight_zero_point.shape) != ((n + 7) // 8, groups):
            raise ValueError(f"expected packed zero points int32 [{(n + 7) // 8}, {groups}], got "
                             f"{weight_zero_point.dtype} {tuple(weight_zero_point.shape)}")
        weight_zero_point = weight_zero_point.contiguous()
    if bias is not None:
        if bias.dtype is not x.dtype or tuple(bias.shape) != (n,):
            raise ValueError(f"expected a bias {x.dtype} [{n}], got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    index = _lib.gpu_index(x, weight_packed, weight_scale, weight_zero_point, bias)
    if not _lib.is_current(index):
        with torch.cuda.device(index):
            return packed_linear(x, weight_packed, weight_scale, weight_zero_point, bias)
    if weight_scale.dtype is not x.dtype and weight_scale.dtype is not torch.float32:
        weight_scale = weight_scale.float()
    weight_packed, weight_scale = weight_packed.contiguous(), weight_scale.contiguous()
    rows = x if x.ndim == 2 else x.reshape(-1, k)
    m, (stride, inner) = rows.shape[0], rows.stride()
    if m > 16 and weight_packed.data_ptr() % 16:
        weight_packed = weight_packed.clone()
    # rows that start at 16-byte boundaries are read in place
    if inner != 1 or stride % 8 or rows.data_ptr() % 16 or (m > 1 and not k <= stride < 1 << 24):
        rows = x.new_empty((m, (k + 7) // 8 * 8))[:, :k].copy_(rows)
        stride = rows.stride(0)
    lib = _lib.load()
    out = x.new_empty((m, n) if x.ndim == 2 else (*x.shape[:-1], n))
    tmp_bytes = lib.ctmi_packed_linear_tmp_bytes(m, n, k, k // groups)
    tmp = torch.empty(tmp_bytes, dtype=torch.uint8, device=x.device) if tmp_bytes else None
    _lib.check(lib.ctmi_packed_linear(
        rows.data_ptr(), _lib.dtype_code(x.dtype), stride, weight_packed.data_ptr(), weight_scale.data_ptr(),
        _lib.dtype_code(weight_scale.dtype), _lib.ptr(weight_zero_point), _lib.ptr(bias), out.data_ptr(), m, n, k,
        k // groups, _lib.ptr(tmp), tmp_bytes, _lib.stream_of_index(index)))
    return out
