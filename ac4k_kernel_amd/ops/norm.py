"""`rms_norm`, the root-mean-square norm with the residual's addition in front and a quantizer behind it, and `dequantize`, the
inverse of `quantize`.  Neither has a counterpart in the reference, whose models norm and add in torch in front of
`quantize` (python/ac4k_kernel/ops/quant.py:73-242), the formats of which these keep.  Inference only, as every operator here."""
from __future__ import annotations

import torch

from .. import _rocm_ops
from .utils import align_up

_OUT_DTYPES = {"fp8e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def rms_norm(x, weight=None, eps=1e-6, residual=None, residual_out=None, precision=None, global_scale=None, out=None):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dim of x, with h = x, or h = x + residual rounded to x's type.

    x is bf16, fp16 or fp32 of any shape [.., K], K <= 65536; weight [K] (x's type or fp32; None: ones) and residual (x's type and shape).
    precision None returns y in x's type and shape (into `out`, which may be x).  Otherwise y goes, from 32 bits and without a
    rounding to x's type, into the format that `quantize(y.reshape(-1, K), 0, 1, precision=precision)` has, rows of all
    leading dims in order:
      "nvfp4"           (output [rows, align_up(K,64)/2] u8, sf [align_up(K,64)/64, align_up(rows,16), 4] e4m3, global_scale)
      "fp8e4m3"/"int8"  (output [rows, align_up(K,16)], sf [align_up(rows,16)] fp32)
    A positive 0-dim fp32 global_scale that is passed in is used as it is and saves finding the maximum over all rows.
    Rows whose largest |y| is under 2^-100 (nvfp4: tensors, and tensors of no rows) give zero codes and zero scales.
    A row with a NaN or an infinite element has NaN in it.  To nvfp4 it makes a global scale that is found NaN, and with it all rows; with a given
    one the other rows are as without it.
    With a residual, h is returned behind the rest; residual_out says where to (default a new tensor; x or residual themselves
    are allowed).
    """
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise RuntimeError("x must be a tensor of at least one dim")
    view = _rocm_ops._rows_view(x, "x")
    if view is None:
        x = x.contiguous()
        view = _rocm_ops._rows_view(x, "x")
    fresh = out is None
    if residual is not None:
        if not isinstance(residual, torch.Tensor):
            raise RuntimeError("residual must be a tensor")
        if not residual.is_contiguous() and _rocm_ops._rows_view(residual, "residual") is None:
            if residual_out is residual:
                raise RuntimeError("residual_out must have rows of contiguous elements, evenly apart")
            residual = residual.contiguous()
        if residual_out is None:
            residual_out = torch.empty_like(x, memory_format=torch.contiguous_format)
        else:
            fresh = False
    elif residual_out is not None:
        raise RuntimeError("residual_out without a residual")
    rows, k, _ = view
    sf, given = None, global_scale is not None
    if given and precision != "nvfp4":
        raise RuntimeError("only nvfp4 has a global scale")
    if precision is None:
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out is not None:
        raise RuntimeError("out is for unquantized results")
    elif precision == "nvfp4":
        out = x.new_empty((rows, align_up(k, 64) // 2), dtype=torch.uint8)
        sf = x.new_empty((align_up(k, 64) // 64, align_up(rows, 16), 4), dtype=torch.float8_e4m3fn)
        if not given:
            global_scale = x.new_empty((), dtype=torch.float32)
    elif precision in _OUT_DTYPES:
        out = x.new_empty((rows, align_up(k, 16)), dtype=_OUT_DTYPES[precision])
        sf = x.new_empty((align_up(rows, 16),), dtype=torch.float32)
    else:
        raise RuntimeError(f"precision must be None, nvfp4, fp8e4m3 or int8, not {precision}")
    _rocm_ops.rms_norm(out, sf, global_scale, given, x, weight, residual, residual_out, precision, float(eps), view, fresh)
    got = (out,) if precision is None else (out, sf, global_scale) if precision == "nvfp4" else (out, sf)
    if residual is not None:
        got += (residual_out,)
    return got if len(got) > 1 else got[0]


def dequantize(output, sf, global_scale=None, dtype=torch.bfloat16, cols=None, out=None):
    """The values that (output, sf[, global_scale]) of `quantize` without swizzle or of `rms_norm` stand for.

    output [.., R, W/2] u8 (nvfp4) or [.., R, W] e4m3 or int8; sf in the layout of `quantize`; global_scale, for nvfp4, 0-dim or
    one per leading plane.  Returns [.., R, cols] of dtype (bf16, fp16 or fp32), cols up to the padded width W, the
    default.  Each value is the product in fp32, rounded to dtype once.
    With `out`, contiguous [.., R, up to W] and apart from the operands, its type and columns count instead of dtype and cols.
    """
    return _rocm_ops.dequantize(out, output, sf, global_scale, dtype, cols)
