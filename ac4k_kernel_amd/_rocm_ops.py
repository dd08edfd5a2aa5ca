"""Tensor-level binding over the C ABI: the module the reference's package would import as
`ac4k_kernel._rocm_ops` (python/ac4k_kernel/__init__.py:39-48), with the function names and
positional arguments of `_cuda_ops` (lib/cuda_bindings.cc:64-85, include/ac4k_kernel/ops.h:27-48).

All functions write into caller-provided tensors, return None, enqueue on the current
torch stream and never synchronise.  Argument checks mirror the reference host launchers'
TORCH_CHECKs and raise RuntimeError.
"""
from __future__ import annotations

import torch

from . import _lib

_L = _lib.load()

__arch__ = _L.ac4k_arch().decode()
__arch_description__ = _L.ac4k_arch_description().decode()
__backend__ = _L.ac4k_backend().decode()
__version__ = _L.ac4k_version().decode()

_DTYPE_TAG = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _check(cond: bool, msg: str, *args) -> None:
    """RuntimeError(msg.format(*args)) unless cond; the message is only built on failure."""
    if not cond:
        raise RuntimeError(msg.format(*args) if args else msg)


def _check_tensor(t, dtype, name: str, suffix: str = "") -> None:
    # one combined test on the hot path; the individual messages are only built on failure
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype and t.is_contiguous():
        return
    name += suffix
    _check(isinstance(t, torch.Tensor), "{} must be a tensor", name)
    _check(t.is_cuda, "{} must be a CUDA tensor", name)
    _check(t.is_contiguous(), "{} must be contiguous", name)
    _check(t.dtype == dtype, "Inconsistency of Tensor type: {} must be {}", name, dtype)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # operands on a GPU: torch is initialised


def _stream() -> int:
    """hipStream_t of torch's current stream on the current device."""
    if _raw_stream is not None:
        return _raw_stream(_current_device())
    return torch.cuda.current_stream().cuda_stream


def _align_up(a: int, b: int) -> int:
    return (a + b - 1) // b * b


def _quant_geometry(inp: torch.Tensor, cross_dim: int, reduce_dim: int):
    """Checks shared by the three quantizers (quantize_nvfp4.cu:171-190,226-241)."""
    _check_tensor(inp, torch.bfloat16, "in")
    _check(2 <= inp.dim() <= 4, "in must be 2-4D")
    _check(0 <= cross_dim < inp.dim(), "cross_dim must be less than in.dim()")
    _check(0 <= reduce_dim < inp.dim(), "reduce_dim must be less than in.dim()")
    _check(cross_dim != reduce_dim, "cross_dim and reduce_dim must be different")
    if inp.dim() == 2:
        shape, stride = inp.shape, inp.stride()
        _check(shape[0] > 0 and shape[1] > 0, "in must not be empty")
        return [], (1, 1, shape[cross_dim], shape[reduce_dim], 0, 0, stride[cross_dim], stride[reduce_dim])
    shape, stride = list(inp.shape), list(inp.stride())
    lead = [i for i in range(inp.dim()) if i not in (cross_dim, reduce_dim)]
    lead_shape = [shape[i] for i in lead]
    ld = [(shape[i], stride[i]) for i in lead]
    while len(ld) < 2:
        ld.insert(0, (1, 0))
    (d0, s0), (d1, s1) = ld
    _check(inp.numel() > 0, "in must not be empty")
    return lead_shape, (d0, d1, shape[cross_dim], shape[reduce_dim], s0, s1, stride[cross_dim], stride[reduce_dim])


def global_scale(out: torch.Tensor, inp: torch.Tensor, max_scale: float) -> None:
    """out (0-dim fp32) = amax(|inp|) / max_scale  (python/ac4k_kernel/ops/quant.py:33-59)."""
    _check_tensor(inp, torch.bfloat16, "in")
    _check_tensor(out, torch.float32, "global_scale")
    _check(out.dim() == 0, "global_scale must be a scalar")
    _lib.check(_L.ac4k_global_scale_bf16(out.data_ptr(), inp.data_ptr(), inp.numel(), float(max_scale), _stream()))


def quantize_nvfp4(out, sf, inp, global_scale, cross_dim: int, reduce_dim: int, swizzle: bool) -> None:
    lead_shape, geom = _quant_geometry(inp, cross_dim, reduce_dim)
    R, K = geom[2], geom[3]
    _check_tensor(global_scale, torch.float32, "global_scale")
    _check(global_scale.dim() == 0, "global_scale must be a scalar")
    _check_tensor(out, torch.uint8, "out")
    _check(list(out.shape) == lead_shape + [R, _align_up(K, 64) // 2],
           "out must have shape [.., cross, align_up(reduce, 64) / 2]")
    _check_tensor(sf, torch.float8_e4m3fn, "sf")
    _check(list(sf.shape) == lead_shape + [_align_up(K, 64) // 64, _align_up(R, 16), 4], "meet invalid sf shape")
    _lib.check(_L.ac4k_quantize_nvfp4(out.data_ptr(), sf.data_ptr(), inp.data_ptr(), global_scale.data_ptr(),
                                      *geom, int(bool(swizzle)), _stream()))


def quantize_nvfp4_with_global_scale(out, sf, global_scale, inp, cross_dim: int, reduce_dim: int, swizzle: bool,
                                     max_scale: float) -> None:
    """global_scale (written) = amax(|inp|) / max_scale, then quantize_nvfp4 with it: the nvfp4 branch
    of the reference's Ac4kQuantizeOp.forward (quant.py:187-242) behind one C call."""
    lead_shape, geom = _quant_geometry(inp, cross_dim, reduce_dim)
    R, K = geom[2], geom[3]
    _check_tensor(global_scale, torch.float32, "global_scale")
    _check(global_scale.dim() == 0, "global_scale must be a scalar")
    _check_tensor(out, torch.uint8, "out")
    _check(list(out.shape) == lead_shape + [R, _align_up(K, 64) // 2],
           "out must have shape [.., cross, align_up(reduce, 64) / 2]")
    _check_tensor(sf, torch.float8_e4m3fn, "sf")
    _check(list(sf.shape) == lead_shape + [_align_up(K, 64) // 64, _align_up(R, 16), 4], "meet invalid sf shape")
    _quantize_nvfp4_bf16(out, sf, global_scale, inp, geom, swizzle, max_scale)


def quantize_nvfp4_new(inp, cross_dim: int, reduce_dim: int, swizzle: bool, max_scale: float):
    """The same into tensors made here, which need no checks: (out, sf, global_scale)."""
    lead_shape, geom = _quant_geometry(inp, cross_dim, reduce_dim)
    R, Kp = geom[2], (geom[3] + 63) // 64 * 64
    dev = inp.device
    out = torch.empty([*lead_shape, R, Kp // 2], dtype=torch.uint8, device=dev)
    sf = torch.empty([*lead_shape, Kp // 64, (R + 15) // 16 * 16, 4], dtype=torch.float8_e4m3fn, device=dev)
    global_scale = torch.empty((), dtype=torch.float32, device=dev)
    _quantize_nvfp4_bf16(out, sf, global_scale, inp, geom, swizzle, max_scale)
    return out, sf, global_scale


def _quantize_nvfp4_bf16(out, sf, global_scale, inp, geom, swizzle, max_scale) -> None:
    _lib.check(_L.ac4k_quantize_nvfp4_bf16(out.data_ptr(), sf.data_ptr(), global_scale.data_ptr(), inp.data_ptr(),
                                           *geom, int(bool(swizzle)), float(max_scale), _stream()))


def _quantize_rowwise(fn, out, out_dtype, sf, inp, scale_max, scale_dtype, cross_dim, reduce_dim, *extra):
    lead_shape, geom = _quant_geometry(inp, cross_dim, reduce_dim)
    R, K = geom[2], geom[3]
    _check_tensor(scale_max, scale_dtype, "scale_max")
    _check(scale_max.dim() == 0, "scale_max must be a scalar")
    _check_tensor(out, out_dtype, "out")
    _check(list(out.shape) == lead_shape + [R, _align_up(K, 16)], "out must have shape [.., cross, align_up(reduce, 16)]")
    _check_tensor(sf, torch.float32, "sf")
    _check(list(sf.shape) == lead_shape + [_align_up(R, 16)], "meet invalid sf shape")
    _lib.check(fn(out.data_ptr(), sf.data_ptr(), inp.data_ptr(), scale_max.data_ptr(), *geom, *extra, _stream()))


def quantize_fp8(out, sf, inp, scale_max, cross_dim: int, reduce_dim: int, swizzle: bool) -> None:
    _quantize_rowwise(_L.ac4k_quantize_fp8, out, torch.float8_e4m3fn, sf, inp, scale_max, torch.float32,
                      cross_dim, reduce_dim, int(bool(swizzle)))


def quantize_int8(out, sf, inp, scale_max, cross_dim: int, reduce_dim: int) -> None:
    _quantize_rowwise(_L.ac4k_quantize_int8, out, torch.int8, sf, inp, scale_max, torch.int32,
                      cross_dim, reduce_dim)


def _check_linear_operand(x, x_sf, x_gs, rows, name):
    # one pass over the attributes of a well-formed operand; what is wrong with another one is found out below
    if isinstance(x, torch.Tensor) and isinstance(x_sf, torch.Tensor) and isinstance(x_gs, torch.Tensor) and x.dim() == 2:
        K = x.size(1) * 2
        if (x.dtype is torch.uint8 and x.is_cuda and x.is_contiguous()
                and x_sf.dtype is torch.float8_e4m3fn and x_sf.is_cuda and x_sf.is_contiguous()
                and x_sf.shape == ((K + 63) // 64, (rows + 15) // 16 * 16, 4)
                and x_gs.dtype is torch.float32 and x_gs.is_cuda and x_gs.dim() == 0):
            return K
    _check(x.dim() == 2, "{} must be a 2d matrix", name)
    _check_tensor(x, torch.uint8, name)
    K = x.size(1) * 2
    _check(x_sf.dim() == 3, "scale_{} must be a 3d matrix", name)
    _check_tensor(x_sf, torch.float8_e4m3fn, "scale_", name)
    _check(x_sf.shape == ((K + 63) // 64, _align_up(rows, 16), 4), "scale_{} has an invalid shape", name)
    _check_tensor(x_gs, torch.float32, "global_scale_", name)
    _check(x_gs.dim() == 0, "{}_global_scale must be a scalar", name)
    return K


def _bias_args(bias, N):
    if bias is None:
        return None, 0
    _check(bias.dtype in _DTYPE_TAG, "bias must be bfloat16, half or float")
    _check(bias.is_cuda and bias.is_contiguous(), "bias must be contiguous")
    _check(bias.dim() == 2, "bias must be a 2d matrix")
    _check(bias.size(0) == 1, "bias shape[0] must be 1")
    _check(bias.size(1) == N, "bias shape[1] must be {}", N)
    return bias.data_ptr(), _DTYPE_TAG[bias.dtype]


def _check_output(D):
    if isinstance(D, torch.Tensor) and D.dim() == 2 and D.is_cuda and D.is_contiguous():
        tag = _DTYPE_TAG.get(D.dtype)
        if tag is not None:
            return D.size(0), D.size(1), tag
    _check(isinstance(D, torch.Tensor) and D.dim() == 2, "d must be a 2d matrix")
    _check(D.dtype in _DTYPE_TAG, "d must be bfloat16, half or float")
    _check(False, "d must be contiguous")


def linear_nvfp4(D, A, A_sf, A_global_scale, B, B_sf, B_global_scale, bias=None) -> None:
    """Checks of linear_nvfp4.cu:759-805.  Shapes for which the library asks for scratch (too few output
    tiles for the GPU, long K) get a workspace tensor and the split-K kernels; everything else goes to
    the reference-shaped entry point, which allocates nothing and picks its kernel by shape."""
    M, N, tag = _check_output(D)
    if A.dim() != 2 or A.size(0) != M:
        _check(False, "A size(0) must be {}", M)
    K = _check_linear_operand(A, A_sf, A_global_scale, M, "a")
    if K % 16 != 0:
        _check(False, "A size(1)*2 must be multiple of 16 but see {}", K)
    if B.dim() != 2 or B.size(1) * 2 != K:
        _check(False, "B size(1) must equal A size(1)")
    if B.size(0) != N:
        _check(False, "B size(0) must be {}", N)
    _check_linear_operand(B, B_sf, B_global_scale, N, "b")
    bias_ptr, bias_tag = (None, 0) if bias is None else _bias_args(bias, N)
    if M == 0 or N == 0:
        return
    nbytes = _L.ac4k_linear_nvfp4_scratch_bytes(M, N, K)
    if nbytes > 0:
        ws = D.new_empty((nbytes,), dtype=torch.uint8)
        _lib.check(_L.ac4k_linear_nvfp4_workspace(D.data_ptr(), tag, A.data_ptr(), A_sf.data_ptr(),
                                                  A_global_scale.data_ptr(), B.data_ptr(), B_sf.data_ptr(),
                                                  B_global_scale.data_ptr(), bias_ptr, bias_tag, M, N, K,
                                                  ws.data_ptr(), nbytes, _stream()))
        return
    _lib.check(_L.ac4k_linear_nvfp4(D.data_ptr(), tag, A.data_ptr(), A_sf.data_ptr(),
                                    A_global_scale.data_ptr(), B.data_ptr(), B_sf.data_ptr(),
                                    B_global_scale.data_ptr(), bias_ptr, bias_tag, M, N, K, _stream()))


_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def linear_nvfp4_epilogue(D, A, A_sf, A_global_scale, B, B_sf, B_global_scale, bias=None, activation=None, residual=None, fresh=False) -> None:
    """linear_nvfp4 with D = act(product + bias) + residual, rounded once.  fresh: D is a new tensor that overlaps nothing."""
    M, N, tag = _check_output(D)
    number = _ACTIVATIONS.get(activation) if activation is None or isinstance(activation, str) else None
    if number is None:
        _check(False, "activation must be one of {}", list(_ACTIVATIONS))
    operands = (A, A_sf, A_global_scale, B, B_sf, B_global_scale)
    dev = _current_device()
    for t in operands:
        if not isinstance(t, torch.Tensor) or t.get_device() != dev:
            _check(t is not None, "operands must be tensors, not NoneType")
            _same_device(t)
    if not fresh or bias is not None or residual is not None:
        _same_device(D, bias, residual)
    _check(A.dim() == 2 and A.size(0) == M, "A size(0) must be {}", M)
    K = _check_linear_operand(A, A_sf, A_global_scale, M, "a")
    if K % 16 != 0:
        _check(False, "A size(1)*2 must be multiple of 16 but see {}", K)
    _check(B.dim() == 2 and B.size(1) * 2 == K, "B size(1) must equal A size(1)")
    _check(B.size(0) == N, "B size(0) must be {}", N)
    _check_linear_operand(B, B_sf, B_global_scale, N, "b")
    bias_ptr, bias_tag = (None, 0) if bias is None else _bias_args(bias, N)
    residual_ptr, residual_step = None, 0
    if residual is not None:
        if _check_float(residual, "residual") != tag or residual.shape != (M, N):
            _check(False, "residual must have the type of the output and be [{}, {}]", M, N)
        if N:
            v = _rows_view(residual, "residual")
            _check(v is not None, "residual must have rows of contiguous elements, evenly apart")
            residual_ptr, residual_step = residual.data_ptr(), v[2]
        _check(fresh or _same_rows(D, residual) or not _may_overlap(D, residual), "out may be residual itself, but not overlap it otherwise")
    if M == 0 or N == 0:
        return
    if not fresh:  # all contiguous
        first = D.data_ptr()
        end = first + M * N * D.element_size()
        for t in (*operands, bias):
            if t is not None and t.data_ptr() < end and first < t.data_ptr() + t.nbytes:
                _check(False, "out must not overlap an operand")
    nbytes = _L.ac4k_linear_nvfp4_scratch_bytes(M, N, K)
    ws = D.new_empty((nbytes,), dtype=torch.uint8) if nbytes > 0 else None
    _lib.check(_L.ac4k_linear_nvfp4_epilogue(D.data_ptr(), tag, A.data_ptr(), A_sf.data_ptr(), A_global_scale.data_ptr(), B.data_ptr(), B_sf.data_ptr(),
                                             B_global_scale.data_ptr(), bias_ptr, bias_tag, number, residual_ptr, residual_step, M, N, K,
                                             None if ws is None else ws.data_ptr(), nbytes, _stream()))


def prepack_weight_nvfp4(B, B_sf) -> torch.Tensor:
    """Weight image of B [N, K/2] / B_sf [K/64, align_up(N,16), 4] for linear_nvfp4_prepacked: a uint8
    tensor of ac4k_prepack_weight_nvfp4_bytes(N, K) bytes.  K must be a multiple of 128."""
    _check(B.dim() == 2, "b must be a 2d matrix")
    _check_tensor(B, torch.uint8, "b")
    N, K = B.size(0), B.size(1) * 2
    _check(B_sf.dim() == 3, "scale_b must be a 3d matrix")
    _check_tensor(B_sf, torch.float8_e4m3fn, "scale_", "b")
    _check(B_sf.shape == ((K + 63) // 64, _align_up(N, 16), 4), "scale_b has an invalid shape")
    nbytes = _L.ac4k_prepack_weight_nvfp4_bytes(N, K)
    _check(nbytes > 0, "no weight image for N = {}, K = {}: K must be a multiple of 128", N, K)
    image = torch.empty((nbytes,), dtype=torch.uint8, device=B.device)
    _lib.check(_L.ac4k_prepack_weight_nvfp4(image.data_ptr(), B.data_ptr(), B_sf.data_ptr(), N, K, _stream()))
    return image


def linear_nvfp4_prepacked(D, A, A_sf, A_global_scale, W_image, B_global_scale, bias=None) -> None:
    """linear_nvfp4 on a weight image made by prepack_weight_nvfp4 (N = D.size(1), K = 2 * A.size(1))."""
    M, N, tag = _check_output(D)
    _check(A.dim() == 2 and A.size(0) == M, "A size(0) must be {}", M)
    K = _check_linear_operand(A, A_sf, A_global_scale, M, "a")
    _check_tensor(W_image, torch.uint8, "w_image")
    _check(N > 0 and W_image.numel() == _L.ac4k_prepack_weight_nvfp4_bytes(N, K) and W_image.numel() > 0,
           "w_image is not the weight image of a [{}, {}] weight", N, K)
    _check_tensor(B_global_scale, torch.float32, "global_scale_", "b")
    _check(B_global_scale.dim() == 0, "b_global_scale must be a scalar")
    bias_ptr, bias_tag = _bias_args(bias, N)
    if M == 0:
        return
    nbytes = _L.ac4k_linear_nvfp4_prepacked_workspace_bytes(M, N, K)
    ws = D.new_empty((nbytes,), dtype=torch.uint8) if nbytes > 0 else None
    _lib.check(_L.ac4k_linear_nvfp4_prepacked(D.data_ptr(), tag, A.data_ptr(), A_sf.data_ptr(),
                                              A_global_scale.data_ptr(), W_image.data_ptr(),
                                              B_global_scale.data_ptr(), bias_ptr, bias_tag, M, N, K,
                                              None if ws is None else ws.data_ptr(), nbytes, _stream()))


def linear_nvfp4_fused(D, X, X_q, X_sf, X_global_scale, B, B_sf, B_global_scale, bias=None) -> None:
    """quantize(X, 0, 1) + linear_nvfp4 for a bf16 activation X [M, K], 1 <= M <= 32;
    X_q / X_sf / X_global_scale receive the quantized activation."""
    M, N, tag = _check_output(D)
    K = _check_fused_activation(X, M)
    _check_tensor(X_q, torch.uint8, "x_q")
    _check(list(X_q.shape) == [M, K // 2], "x_q must be [M, K/2]")
    _check_linear_operand(X_q, X_sf, X_global_scale, M, "x")
    _check(B.dim() == 2 and B.size(0) == N and B.size(1) == K // 2, "weight must be [N, K/2]")
    _check_linear_operand(B, B_sf, B_global_scale, N, "b")
    bias_ptr, bias_tag = _bias_args(bias, N)
    if K % 256 != 0:  # the C entry point takes whole stages of the kernels it began with: the composition itself, same kernels
        quantize_nvfp4_with_global_scale(X_q, X_sf, X_global_scale, X, 0, 1, False, 2688.0)
        linear_nvfp4(D, X_q, X_sf, X_global_scale, B, B_sf, B_global_scale, bias)
        return
    nbytes = _L.ac4k_linear_nvfp4_workspace_bytes(M, N, K)  # 0: one K range per tile, no scratch
    ws = D.new_empty((nbytes,), dtype=torch.uint8) if nbytes > 0 else None
    _lib.check(_L.ac4k_linear_nvfp4_fused_bf16(D.data_ptr(), tag, X.data_ptr(), X_q.data_ptr(),
                                               X_sf.data_ptr(), X_global_scale.data_ptr(), B.data_ptr(),
                                               B_sf.data_ptr(), B_global_scale.data_ptr(), bias_ptr, bias_tag,
                                               M, N, K, None if ws is None else ws.data_ptr(), nbytes, _stream()))


def _check_fused_activation(X, M):
    _check_tensor(X, torch.bfloat16, "x")
    _check(X.dim() == 2 and X.size(0) == M, "x must be [{}, K]", M)
    _check(1 <= M <= 32, "the fused linear takes 1 <= M <= 32")
    K = X.size(1)
    _check(K % 64 == 0, "K must be a multiple of 64")
    return K


def linear_nvfp4_fused_scratch(D, X, B, B_sf, B_global_scale, bias=None) -> bool:
    """linear_nvfp4_fused for a caller who does not ask for the quantized activation: it and the workspace are one allocation.
    False, with nothing done, for a K that runs as the composition."""
    M, N, tag = _check_output(D)
    K = _check_fused_activation(X, M)
    if K == 0 or K % 256 != 0:
        return False
    _check(B.dim() == 2 and B.size(0) == N and B.size(1) == K // 2, "weight must be [N, K/2]")
    _check_linear_operand(B, B_sf, B_global_scale, N, "b")
    bias_ptr, bias_tag = (None, 0) if bias is None else _bias_args(bias, N)
    nbytes = _L.ac4k_linear_nvfp4_workspace_bytes(M, N, K)  # 0: one K range per tile, no scratch
    q_bytes, sf_bytes = _align_up(M * K // 2, 256), K // 64 * _align_up(M, 16) * 4  # (a multiple of 256: K % 256 == 0)
    ws_bytes = _align_up(nbytes, 256)
    ws = D.new_empty((ws_bytes + q_bytes + sf_bytes + 4,), dtype=torch.uint8)
    at = ws.data_ptr()
    q = at + ws_bytes
    _lib.check(_L.ac4k_linear_nvfp4_fused_bf16(D.data_ptr(), tag, X.data_ptr(), q, q + q_bytes, q + q_bytes + sf_bytes, B.data_ptr(),
                                               B_sf.data_ptr(), B_global_scale.data_ptr(), bias_ptr, bias_tag,
                                               M, N, K, at if nbytes > 0 else None, nbytes, _stream()))
    return True


def _check_attention_operand(x, x_sf, x_gs, B, H, rows, width, name):
    """One packed operand of mha_nvfp4_fwd: x [B,H,rows,width/2], x_sf [B,H,ceil(width/64),align_up(rows,16),4]
    (mha_nvfp4.cu:917-1003)."""
    _check_tensor(x, torch.uint8, name)
    _check(x.dim() == 4 and list(x.shape) == [B, H, rows, width // 2], "{} must be [{}, {}, {}, {}]", name, B, H, rows, width // 2)
    _check_tensor(x_sf, torch.float8_e4m3fn, name + "_sf")
    _check(x_sf.dim() == 5, "{}_sf must be a 5D tensor", name)
    _check(list(x_sf.shape) == [B, H, (width + 63) // 64, _align_up(rows, 16), 4], "Meet invalid {}_sf size", name)
    _check_tensor(x_gs, torch.float32, name + "_global_scale")
    _check(x_gs.dim() == 0, "{}_global_scale must be a float tensor", name)


def mha_nvfp4_fwd(o, q, q_sf, q_global_scale, k, k_sf, k_global_scale, v, v_sf, v_global_scale, sm_scale: float) -> None:
    """Checks of mha_nvfp4.cu:917-1012.  o may be a permuted view (the reference's caller passes one): only its
    shape [B,H,Nq,Dv], dtype and device are checked."""
    _check(isinstance(q, torch.Tensor) and q.dim() == 4, "Q must be a 4D tensor")
    B, H, Nq = q.size(0), q.size(1), q.size(2)
    Dqk = q.size(3) * 2
    _check(Dqk % 16 == 0, "Dqk must be multiple of 16")
    _check(Dqk <= 128, "Dqk must be less than 128")
    _check(isinstance(k, torch.Tensor) and k.dim() == 4, "K must be a 4D tensor")
    _check(k.size(0) == B, "K must have the same batch size as Q")
    _check(k.size(1) == H, "K must have the same head number as Q")
    _check(k.size(3) == q.size(3), "K must have the same dim as Q")
    Nkv = k.size(2)
    _check(isinstance(v, torch.Tensor) and v.dim() == 4, "V must be a 4D tensor")
    Dv = v.size(2)
    _check(Dv <= 128, "Dv must be less than 128")
    _check(v.size(3) * 2 == _align_up(Nkv, 64), "V must have the same sequence length as K")
    _check_attention_operand(q, q_sf, q_global_scale, B, H, Nq, Dqk, "q")
    _check_attention_operand(k, k_sf, k_global_scale, B, H, Nkv, Dqk, "k")
    _check_attention_operand(v, v_sf, v_global_scale, B, H, Dv, _align_up(Nkv, 64), "v")
    _check(isinstance(o, torch.Tensor) and o.is_cuda, "O must be a CUDA tensor")
    _check(o.dtype == torch.bfloat16, "O must be a bfloat16 tensor")
    _check(o.dim() == 4 and list(o.shape) == [B, H, Nq, Dv], "O must be [{}, {}, {}, {}]", B, H, Nq, Dv)
    if B == 0 or H == 0 or Nq == 0:
        return
    _check(Nkv > 0, "K must not be empty")
    _lib.check(_L.ac4k_mha_nvfp4_fwd(o.data_ptr(), *o.stride(), q.data_ptr(), q_sf.data_ptr(), q_global_scale.data_ptr(),
                                     k.data_ptr(), k_sf.data_ptr(), k_global_scale.data_ptr(), v.data_ptr(), v_sf.data_ptr(),
                                     v_global_scale.data_ptr(), B, H, Nq, Nkv, Dqk, Dv, float(sm_scale), _stream()))


def mha_int8_x_fp8_fwd(o, q, q_sf, q_quantize_block_size: int, k, k_sf, k_quantize_block_size: int, v, v_sf,
                       sm_scale: float) -> None:
    """Checks of mha_int8_x_fp8.cu:982-1044.  o may be a permuted view: only its shape [B,H,Nq,Dv], dtype and
    device are checked."""
    _check_tensor(q, torch.int8, "Q")
    _check(q.dim() == 4, "Q must be a 4D tensor")
    B, H, Nq, Dqk = q.size(0), q.size(1), q.size(2), q.size(3)
    _check(Dqk % 16 == 0, "Dqk must be multiple of 16")
    _check(Dqk <= 128, "Dqk must be less than 128")
    _check_tensor(q_sf, torch.float32, "Q_SF")
    _check(q_sf.dim() == 3, "Q_SF must be a 3D tensor")
    _check(list(q_sf.shape) == [B, H, -(-Nq // q_quantize_block_size)], "Meet invalid Q_SF size")
    _check_tensor(k, torch.int8, "K")
    _check(k.dim() == 4, "K must be a 4D tensor")
    _check(k.size(0) == B, "K must have the same batch size as Q")
    _check(k.size(1) == H, "K must have the same head number as Q")
    _check(k.size(3) == Dqk, "K must have the same dim as Q")
    Nkv = k.size(2)
    _check_tensor(k_sf, torch.float32, "K_SF")
    _check(k_sf.dim() == 3, "K_SF must be a 3D tensor")
    _check(list(k_sf.shape) == [B, H, -(-Nkv // k_quantize_block_size)], "Meet invalid K_SF size")
    _check_tensor(v, torch.float8_e4m3fn, "V")
    _check(v.dim() == 4, "V must be a 4D tensor")
    _check(v.size(0) == B, "V must have the same batch size as Q")
    _check(v.size(1) == H, "V must have the same head number as Q")
    Dv = v.size(2)
    _check(v.size(3) == _align_up(Nkv, 16), "Meet invalid v size(3) with {}=={}", v.size(3), _align_up(Nkv, 16))
    _check(Dv <= 128, "Dv must be less than 128")
    _check_tensor(v_sf, torch.float32, "V_SF")
    _check(v_sf.dim() == 3 and list(v_sf.shape) == [B, H, _align_up(Dv, 16)], "Meet invalid v_sf size")
    _check(isinstance(o, torch.Tensor) and o.is_cuda, "O must be a CUDA tensor")
    _check(o.dtype == torch.bfloat16, "O must be a bfloat16 tensor")
    _check(o.dim() == 4 and list(o.shape) == [B, H, Nq, Dv], "O must be [{}, {}, {}, {}]", B, H, Nq, Dv)
    if B == 0 or H == 0 or Nq == 0:
        return
    _check(Nkv > 0, "K must not be empty")
    _lib.check(_L.ac4k_mha_int8_x_fp8_fwd(o.data_ptr(), *o.stride(), q.data_ptr(), q_sf.data_ptr(), int(q_quantize_block_size),
                                          k.data_ptr(), k_sf.data_ptr(), int(k_quantize_block_size), v.data_ptr(),
                                          v_sf.data_ptr(), B, H, Nq, Nkv, Dqk, Dv, float(sm_scale), _stream()))


def _attention(entry, workspace_bytes, o, q, k, v, scale: float, sm_scale: float, bnhd: bool) -> bool:
    try:
        if bnhd:
            (B, Nq, H, Dqk), (k_B, Nkv, k_H, k_D), (v_B, v_N, v_H, Dv), (o_B, o_N, o_H, o_D) = q.shape, k.shape, v.shape, o.shape
        else:
            (B, H, Nq, Dqk), (k_B, k_H, Nkv, k_D), (v_B, v_H, v_N, Dv), (o_B, o_H, o_N, o_D) = q.shape, k.shape, v.shape, o.shape
    except ValueError:  # not 4D
        return False
    dev, bf16 = q.get_device(), torch.bfloat16  # -1 on the CPU
    if not (B == k_B == v_B == o_B and H == k_H == v_H == o_H and Nkv == v_N and Nq == o_N and Dqk == k_D and Dv == o_D
            and dev >= 0 and dev == k.get_device() == v.get_device() == o.get_device()
            and q.dtype is bf16 and k.dtype is bf16 and v.dtype is bf16 and o.dtype is bf16):
        return False
    if bnhd:
        (q_b, q_n, q_h, q_d), (k_b, k_n, k_h, k_d), (v_b, v_n, v_h, v_d), (o_b, o_n, o_h, o_d) = q.stride(), k.stride(), v.stride(), o.stride()
    else:
        (q_b, q_h, q_n, q_d), (k_b, k_h, k_n, k_d), (v_b, v_h, v_n, v_d), (o_b, o_h, o_n, o_d) = q.stride(), k.stride(), v.stride(), o.stride()
    if q_d != 1 or k_d != 1 or v_d != 1:
        return False
    nbytes = workspace_bytes(B, H, Nq, Nkv, Dqk, Dv)
    if nbytes < 0:
        return False
    ws = q.new_empty((nbytes,), dtype=torch.uint8)
    _lib.check(entry(o.data_ptr(), o_b, o_h, o_n, o_d, q.data_ptr(), q_b, q_h, q_n, k.data_ptr(), k_b, k_h, k_n, v.data_ptr(), v_b, v_h, v_n,
                     B, H, Nq, Nkv, Dqk, Dv, scale, sm_scale, ws.data_ptr(), nbytes, _stream()))
    return True


def attention_int8_x_fp8(o, q, k, v, v_scale_max: float, sm_scale: float, bnhd: bool = False) -> bool:
    """The whole `_int8_x_fp8_attention` (python/ac4k_kernel/ops/attention.py:137-190) behind one C call on bf16 q, k, v
    of [B,H,N,D], or of [B,N,H,D] with `bnhd` (any batch, head and token strides).  False, with nothing done, for operands this call does not
    take - odd shapes, other dtypes and the ones an operator-by-operator call rejects with its own message."""
    return _attention(_L.ac4k_attention_int8_x_fp8_bf16, _L.ac4k_attention_int8_x_fp8_workspace_bytes, o, q, k, v, v_scale_max, sm_scale, bnhd)


def attention_nvfp4(o, q, k, v, sm_scale: float, bnhd: bool = False) -> bool:
    """The same for `_nvfp4_attention` (python/ac4k_kernel/ops/attention.py:100-133) on dense q, k, v."""
    return _attention(_L.ac4k_attention_nvfp4_bf16, _L.ac4k_attention_nvfp4_workspace_bytes, o, q, k, v, 2688.0, sm_scale, bnhd)


def quantize_int8_token_block(y, scale, x_bhnd, block: int) -> None:
    """y int8 [B,H,N,align_up(D,16)], scale fp32 [B,H,ceil(N/block)] <- x bf16 viewed as [B,H,N,D] (any batch, head and
    token strides, head dim contiguous): the per-token-block quantizer of python/ac4k_kernel/ops/attention.py:18-99."""
    _check(isinstance(x_bhnd, torch.Tensor) and x_bhnd.is_cuda and x_bhnd.dtype == torch.bfloat16, "x must be a CUDA bfloat16 tensor")
    _check(x_bhnd.dim() == 4 and x_bhnd.stride(3) == 1, "x must be 4D with a contiguous head dim")
    B, H, N, D = x_bhnd.shape
    _check_tensor(y, torch.int8, "y")
    _check(list(y.shape) == [B, H, N, _align_up(D, 16)], "Meet invalid y size")
    _check_tensor(scale, torch.float32, "scale")
    _check(list(scale.shape) == [B, H, -(-N // block)], "Meet invalid scale size")
    if x_bhnd.numel() == 0:
        return
    _lib.check(_L.ac4k_quantize_int8_token_block_bf16(y.data_ptr(), scale.data_ptr(), x_bhnd.data_ptr(), B, H, N, D,
                                                      x_bhnd.stride(0), x_bhnd.stride(1), x_bhnd.stride(2), int(block), _stream()))


_PRECISIONS = {None: 0, "fp8e4m3": 1, "int8": 2, "nvfp4": 3}
_EIGHT_BITS = {torch.float8_e4m3fn: 1, torch.int8: 2}


def _check_float(t, name: str) -> int:
    if isinstance(t, torch.Tensor) and t.is_cuda:
        tag = _DTYPE_TAG.get(t.dtype)
        if tag is not None:
            return tag
    _check(isinstance(t, torch.Tensor), "{} must be a tensor", name)
    _check(t.is_cuda, "{} must be a CUDA tensor", name)
    _check(t.dtype in _DTYPE_TAG, "{} must be bfloat16, half or float", name)
    return _DTYPE_TAG[t.dtype]


def _same_device(*tensors) -> None:
    """Kernels run on the current device and its stream: every operand has to be there."""
    dev = _current_device()
    for t in tensors:
        if t is not None and not (isinstance(t, torch.Tensor) and t.get_device() == dev):
            _check(isinstance(t, torch.Tensor), "operands must be tensors, not {}", type(t).__name__)
            _check(False, "operands must be on the current device, {}: got one on {}", dev, t.device)


def _rows_view(t, name: str):
    """t [.., K] as rows: (rows, K, elements between rows) of the tensor itself, or None if no single row stride describes it."""
    shape, stride = t.shape, t.stride()
    if not shape or shape[-1] < 1:
        _check(False, "{} must have a last dim of at least one element", name)
    if t.is_contiguous():
        return t.numel() // shape[-1], shape[-1], shape[-1]
    rows, step = 1, 0
    if shape[-1] > 1 and stride[-1] != 1:
        return None
    for n, s in zip(reversed(shape[:-1]), reversed(stride[:-1])):
        if n == 1:
            continue
        if rows > 1 and s != step * rows:
            return None
        if rows == 1:
            step = s
        rows *= n
    return rows, shape[-1], step


def _may_overlap(a, b) -> bool:
    """Whether two tensors can share memory: not if one ends before the other begins, nor if, of every length of some stride, each has a part
    of its own (columns of the rows of one buffer, heads of one projection)."""
    if not (a.numel() and b.numel()):
        return False
    a0, b0, size_a, size_b = a.data_ptr(), b.data_ptr(), a.element_size(), b.element_size()
    if a0 <= b0:
        if a0 + size_a * (1 + sum([(n - 1) * s for n, s in zip(a.shape, a.stride())])) <= b0:
            return False
    elif b0 + size_b * (1 + sum([(n - 1) * s for n, s in zip(b.shape, b.stride())])) <= a0:
        return False
    dims_a = [(s * size_a, n) for s, n in zip(a.stride(), a.shape) if n > 1]
    dims_b = [(s * size_b, n) for s, n in zip(b.stride(), b.shape) if n > 1]
    steps = {s for s, _ in dims_a + dims_b}
    for step in steps:
        if step and not any(s > step and s % step for s in steps):
            # the longer strides are whole steps: every element is inside [0, part) of the place of the first one, in steps
            part_a = size_a + sum((n - 1) * s for s, n in dims_a if s < step)
            part_b = size_b + sum((n - 1) * s for s, n in dims_b if s < step)
            away = (b0 - a0) % step
            if part_a <= away and away + part_b <= step:
                return False
    return True


def _places_of_their_own(t) -> bool:
    """Whether no two elements of t share memory, as far as strides in rising order say."""
    reach = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < reach:
            return False
        reach = s * n
    return True


def _same_rows(a, b) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride()


def rms_norm(out, sf, global_scale, given_scale: bool, x, weight, residual, residual_out, precision, eps: float, view=None, fresh=False) -> None:
    """out (and sf, global_scale) <- norm of the rows of x, or of x + residual, which residual_out receives.  view: _rows_view(x), where the
    caller has it; fresh: out, sf and residual_out are new dense tensors of the right shapes and overlap nothing."""
    tag = _check_float(x, "x")
    view = view or _rows_view(x, "x")
    _check(view is not None, "x must have rows of contiguous elements, evenly apart")
    rows, K, x_step = view
    number = _PRECISIONS.get(precision)
    if number is None:
        _check(False, "precision must be one of {}", list(_PRECISIONS))
    if global_scale is not None:
        _check_tensor(global_scale, torch.float32, "global_scale")
        _check(global_scale.dim() == 0, "global_scale must be a scalar")
    dev = _current_device()
    if x.get_device() != dev or not fresh or global_scale is not None:
        _same_device(x, residual_out, out, sf, global_scale)
    weight_ptr, weight_tag = None, tag
    if weight is not None:
        weight_tag = _check_float(weight, "weight")
        if (weight_tag != tag and weight_tag != 2) or weight.get_device() != dev:
            _check(weight.get_device() == dev, "weight must be on the current device")
            _check(False, "weight must have the type of x or be float")
        if weight.shape != (K,) or not weight.is_contiguous():
            _check(False, "weight must be contiguous of [{}]", K)
        weight_ptr = weight.data_ptr()
    if (residual is None) != (residual_out is None):
        _check(False, "a residual comes with residual_out, and the other way round")
    residual_ptr = sum_ptr = None
    residual_step = sum_step = 0
    if residual is not None:
        if _check_float(residual, "residual") != tag or residual.shape != x.shape or residual.get_device() != dev:
            _check(residual.get_device() == dev, "residual must be on the current device")
            _check(False, "residual must have the type and shape of x")
        v = _rows_view(residual, "residual")
        if v is None:
            _check(False, "residual must have rows of contiguous elements, evenly apart")
        residual_ptr, residual_step, sum_ptr, sum_step = residual.data_ptr(), v[2], residual_out.data_ptr(), K
        if not fresh:
            _check(_check_float(residual_out, "residual_out") == tag and residual_out.shape == x.shape, "residual_out must have the type and shape of x")
            v = _rows_view(residual_out, "residual_out")
            _check(v is not None and (rows <= 1 or v[2] >= K), "residual_out must have rows of contiguous elements, evenly apart")
            sum_step = v[2]
            for t in (x, residual):
                _check(_same_rows(t, residual_out) or not _may_overlap(t, residual_out),
                       "residual_out may be x or residual itself, but not overlap them otherwise")
            for t in (weight, global_scale):
                _check(t is None or not _may_overlap(t, residual_out), "residual_out must not overlap weight or global_scale")
    out_step = K
    if not fresh:
        if precision is None:
            _check(_check_float(out, "out") == tag and out.shape == x.shape, "out must have the type and shape of x")
            v = _rows_view(out, "out")
            _check(v is not None and (rows <= 1 or v[2] >= K), "out must have rows of contiguous elements, evenly apart")
            out_step = v[2]
            _check(_same_rows(out, x) or not _may_overlap(out, x), "out may be x itself, but not overlap it otherwise")
            for t in (residual, residual_out, weight):
                _check(t is None or not _may_overlap(out, t), "out must not overlap residual, residual_out or weight")
        else:
            nvfp4 = precision == "nvfp4"
            _check_tensor(out, torch.uint8 if nvfp4 else torch.float8_e4m3fn if precision == "fp8e4m3" else torch.int8, "out")
            _check(list(out.shape) == [rows, _align_up(K, 64) // 2 if nvfp4 else _align_up(K, 16)], "meet invalid out shape")
            _check_tensor(sf, torch.float8_e4m3fn if nvfp4 else torch.float32, "sf")
            _check(list(sf.shape) == ([_align_up(K, 64) // 64, _align_up(rows, 16), 4] if nvfp4 else [_align_up(rows, 16)]), "meet invalid sf shape")
    if rows == 0:
        if global_scale is not None and not given_scale:
            global_scale.zero_()  # that of a tensor of zeros
        return
    ws_ptr, nbytes = None, 0
    if number == 3 and not given_scale:
        nbytes = _L.ac4k_rms_norm_workspace_bytes(rows, K, tag, number, 0)
        if nbytes > 0:
            ws = x.new_empty((nbytes,), dtype=torch.uint8)
            ws_ptr = ws.data_ptr()
    _lib.check(_L.ac4k_rms_norm(out.data_ptr(), out_step, None if sf is None else sf.data_ptr(),
                                None if global_scale is None else global_scale.data_ptr(), int(given_scale), x.data_ptr(), x_step,
                                residual_ptr, residual_step, sum_ptr, sum_step, weight_ptr, weight_tag, rows, K, tag, number, eps, ws_ptr, nbytes,
                                _stream()))


def dequantize(out, q, sf, global_scale=None, dtype=None, cols=None):
    """out [.., R, cols] (None: a new tensor of dtype) <- the values of q, sf (and global_scale, for nvfp4) as `quantize` returns them
    without swizzle; returns out."""
    if not isinstance(q, torch.Tensor) or q.dim() < 2:
        _check(False, "q must have at least two dims")
    kind = q.dtype
    nvfp4 = kind is torch.uint8
    number = 3 if nvfp4 else _EIGHT_BITS.get(kind)
    if number is None:
        _check(False, "q must be uint8 (nvfp4), float8_e4m3fn or int8")
    _check_tensor(q, kind, "q")
    _check_tensor(sf, torch.float8_e4m3fn if nvfp4 else torch.float32, "sf")
    dev = _current_device()
    if q.get_device() != dev or sf.get_device() != dev:
        _same_device(q, sf)
    *lead, R, W = q.shape
    planes, gs_step, gs_ptr = 1, 0, None
    for n in lead:
        planes *= n
    if nvfp4:
        W *= 2
        if W % 64 != 0 or sf.shape != (*lead, W // 64, (R + 15) // 16 * 16, 4):
            _check(W % 64 == 0, "rows of q must be whole pieces of 64 elements")
            _check(False, "meet invalid sf shape")
        _check_tensor(global_scale, torch.float32, "global_scale")
        if global_scale.get_device() != dev:
            _same_device(global_scale)
        if global_scale.dim() != 0:
            _check(list(global_scale.shape) == lead, "global_scale must be a scalar or have the leading dims of q")
            gs_step = 1
        gs_ptr = global_scale.data_ptr()
    else:
        if W % 16 != 0 or sf.shape != (*lead, (R + 15) // 16 * 16):
            _check(W % 16 == 0, "rows of q must be whole pieces of 16 elements")
            _check(False, "meet invalid sf shape")
        if global_scale is not None:
            _check(False, "only nvfp4 has a global scale")
    if out is None:
        cols = W if cols is None else cols
        tag = _DTYPE_TAG.get(dtype)
        if tag is None or not 0 <= cols <= W:
            _check(tag is not None, "out must be bfloat16, half or float")
            _check(False, "out must be contiguous of [.., {}, up to {}]", R, W)
        out = q.new_empty((*lead, R, cols), dtype=dtype)
    else:
        tag = _check_float(out, "out")
        _same_device(out)
        *out_lead, cols = out.shape
        _check(out.is_contiguous() and out_lead == [*lead, R] and cols <= W, "out must be contiguous of [.., {}, up to {}]", R, W)
        _check(not any(_may_overlap(out, t) for t in (q, sf, global_scale) if t is not None), "out must not overlap the quantized operands")
    if planes and R and cols:
        _lib.check(_L.ac4k_dequantize(out.data_ptr(), tag, q.data_ptr(), sf.data_ptr(), gs_ptr, gs_step, planes, R, W, cols, number, _stream()))
    return out


_ROPE_SECTIONS = {}


def _rope_sections(sections, pairs: int):
    """The C array of a tuple of sections, checked against the table; kept by its values."""
    got = _ROPE_SECTIONS.get((sections, pairs))
    if got is None:
        _check(1 <= len(sections) <= 8 and sum(sections) == pairs and min(sections) >= 0, "sections must be 1 to 8 counts of pairs, {} in all", pairs)
        if len(_ROPE_SECTIONS) > 64:
            _ROPE_SECTIONS.clear()
        got = _ROPE_SECTIONS[sections, pairs] = (_lib._i64 * len(sections))(*sections)
    return got


_RopePair = _lib.RopeTensor * 2
_POSITIONS = {torch.int32, torch.int64}


def rope(outs, xs, table, sections, positions, grid, bnhd: bool, interleaved: bool, inverse: bool):
    """outs (None: new dense tensors) <- xs, one or two tensors, turned by the angles of their tokens' positions; returns outs."""
    count = len(xs)
    if count > 2 or count < 1 or (outs is not None and len(outs) != count):
        _check(False, "rope takes one or two tensors, and as many outputs")
    x = xs[0]
    tag = _check_float(x, "x")
    dev = _current_device()
    _check_tensor(table, torch.float32, "table")
    if x.dim() != 4 or table.dim() != 3:
        _check(False, "x must be a 4D tensor, table [length, pairs, 2]")
    B, N, N2, D = x.shape
    length, pairs, two = table.shape
    if not bnhd:
        N = N2
    if two != 2 or length < 1 or pairs < 1 or 2 * pairs > D:
        _check(two == 2 and length >= 1 and pairs >= 1, "table must be [length, pairs, 2]")
        _check(False, "{} pairs do not fit a head of {}", pairs, D)
    section_arg, axes = _rope_sections(sections, pairs), len(sections)
    if x.get_device() != dev or table.get_device() != dev:
        _same_device(x, table)
    args, used = _RopePair(), 0
    made, spans = [], []  # spans: first and end address of the caller's outputs
    for i, t in enumerate(xs):
        if i:
            if t.get_device() != dev or t.dtype is not x.dtype or t.dim() != 4 or t.shape[0] != B or t.shape[1 if bnhd else 2] != N or t.shape[3] != D:
                _same_device(t)
                _check(_check_float(t, "x") == tag, "all tensors must have one type")
                _check(False, "all tensors must have the same batch, tokens and head dim")
        t_b, t_n, t_h, t_d = t.stride()
        if t_d != 1:
            _check(False, "heads must be contiguous")
        if outs is None:
            o = torch.empty_like(t, memory_format=torch.contiguous_format)
            made.append(o)
        else:
            o = outs[i]
            _same_device(o)
            _check(_check_float(o, "out") == tag, "all tensors must have one type")
            _check(o.shape == t.shape, "out must have the shape of x")
            _check(o.stride(3) == 1 and _places_of_their_own(o), "heads of out must be contiguous, and apart from each other")
            _check(_same_rows(t, o) or not _may_overlap(t, o), "out may be x itself, but not overlap it otherwise")
        if t.numel() == 0:
            continue
        o_b, o_n, o_h, _ = o.stride()
        if outs is not None:
            first = o.data_ptr()
            last = sum([(n - 1) * s for n, s in zip(o.shape, (o_b, o_n, o_h, 1))])
            spans.append((first, first + (1 + last) * (4 if tag == 2 else 2)))
        args[used] = ((t.data_ptr(), o.data_ptr(), t_b, t_n, t_h, o_b, o_n, o_h, t.shape[2]) if bnhd else
                      (t.data_ptr(), o.data_ptr(), t_b, t_h, t_n, o_b, o_h, o_n, t.shape[1]))
        used += 1
    if count == 2 and outs is not None:
        _check(not any(_may_overlap(o, t) for o, t in ((outs[0], xs[1]), (outs[1], xs[0]), (outs[0], outs[1]))),
               "the two tensors must not overlap each other")
    pos_ptr, pos_bytes, pos_strides, grid_arg = None, 0, (0, 0, 0), None
    if positions is not None:
        if grid is not None or positions.dtype not in _POSITIONS or positions.shape != (axes, B, N) or positions.get_device() != dev:
            _same_device(positions)
            _check(grid is None, "positions or a grid, one of them")
            _check(positions.is_cuda and positions.dtype in _POSITIONS, "positions must be a CUDA tensor of int32 or int64")
            _check(False, "positions must be [{}, {}, {}]", axes, B, N)
        pos_ptr, pos_bytes, pos_strides = positions.data_ptr(), positions.element_size(), positions.stride()
    else:
        _check(grid is not None and len(grid) == axes and min(grid) >= 1, "grid must have one size of at least 1 for each axis")
        _check(max(grid) <= length, "the table has {} positions, the grid {}", length, max(grid))
        grid_arg = (_lib._i64 * axes)(*grid)
    for first, end in spans:
        at = table.data_ptr()
        if at < end and first < at + length * pairs * 8:
            _check(False, "out must not overlap the table")
        if pos_ptr is not None and pos_ptr < end:
            last = sum([(n - 1) * s for n, s in zip(positions.shape, pos_strides)])
            _check(first >= pos_ptr + (1 + last) * pos_bytes, "out must not overlap the positions")
    if used:
        _lib.check(_L.ac4k_rope(args, used, tag, B, N, D, table.data_ptr(), length, pairs, section_arg, axes, pos_ptr, pos_bytes, *pos_strides,
                                grid_arg, interleaved, inverse, _stream()))
    return outs or tuple(made)


def linear_grouped_nvfp4(D, A, A_sf, A_global_scale, B, B_sf, B_global_scale, offsets, rows=None, bias=None, whole=False) -> None:
    """D[i] = linear of row rows[i] (row i without rows) of A on the weight of the expert whose range of offsets holds i; rows that no range holds stay
    as they are, or become zero (whole)."""
    M, N, tag = _check_output(D)
    _check(isinstance(A, torch.Tensor) and A.dim() == 2, "a must be a 2d matrix")
    T = A.size(0)
    K = _check_linear_operand(A, A_sf, A_global_scale, T, "a")
    _check(K >= 64 and K % 64 == 0, "K must be a multiple of 64 but see {}", K)
    _check(isinstance(B, torch.Tensor) and B.dim() == 3, "b must be [experts, N, K/2]")
    E = B.size(0)
    _check(B.size(1) == N, "b size(1) must be {}", N)
    _check(B.size(2) * 2 == K, "b size(2) must equal a size(1)")
    _check_tensor(B, torch.uint8, "b")
    _check_tensor(B_sf, torch.float8_e4m3fn, "scale_b")
    _check(B_sf.shape == (E, K // 64, _align_up(N, 16), 4), "scale_b has an invalid shape")
    _check_tensor(B_global_scale, torch.float32, "global_scale_b")
    _check(B_global_scale.dim() == 0 or list(B_global_scale.shape) == [E], "b_global_scale must be a scalar or one per expert")
    _check_tensor(offsets, torch.int32, "offsets")
    _check(list(offsets.shape) == [E + 1], "offsets must be [{}]", E + 1)
    if rows is None:
        _check(T == M, "A size(0) must be {}", M)
    else:
        _check_tensor(rows, torch.int32, "rows")
        _check(list(rows.shape) == [M], "rows must be [{}]", M)
    bias_ptr, bias_tag = None, 0
    if bias is not None:
        bias_tag = _check_float(bias, "bias")
        _check(bias.is_contiguous() and list(bias.shape) == [E, N], "bias must be contiguous of [{}, {}]", E, N)
        bias_ptr = bias.data_ptr()
    _same_device(D, A, A_sf, A_global_scale, B, B_sf, B_global_scale, offsets, rows, bias)
    if M == 0 or N == 0 or E == 0:
        if whole:
            D.zero_()
        return
    _check(T > 0, "rows of an empty a")
    if not whole:  # (otherwise D is new memory)
        first = D.data_ptr()
        end = first + M * N * D.element_size()
        for t in (A, A_sf, A_global_scale, B, B_sf, B_global_scale, offsets, rows, bias):  # all contiguous
            if t is not None and t.data_ptr() < end and first < t.data_ptr() + t.nbytes:
                _check(False, "out must not overlap an operand")
    nbytes = _L.ac4k_linear_grouped_nvfp4_workspace_bytes(T, M, N, K, E, int(rows is not None))
    ws = D.new_empty((nbytes,), dtype=torch.uint8) if nbytes > 0 else None
    call = _L.ac4k_linear_grouped_nvfp4_whole if whole else _L.ac4k_linear_grouped_nvfp4
    _lib.check(call(D.data_ptr(), tag, A.data_ptr(), A_sf.data_ptr(), A_global_scale.data_ptr(), T, None if rows is None else rows.data_ptr(),
                    B.data_ptr(), B_sf.data_ptr(), B_global_scale.data_ptr(), int(B_global_scale.dim() > 0), bias_ptr, bias_tag, offsets.data_ptr(),
                    M, N, K, E, None if ws is None else ws.data_ptr(), nbytes, _stream()))


_SCORING = {"softmax": 0, "sigmoid": 1}


def route_experts(logits, k: int, bias, scoring, groups: int, top_groups: int, best: int, renormalize: bool, scale: float, view=None):
    """The k experts of each row of logits: new tensors weights, experts [.., k], offsets [E + 1], rows [T * k] and places [.., k].  view:
    _rows_view(logits), where the caller has it."""
    tag = _check_float(logits, "logits")
    view = view or _rows_view(logits, "logits")
    if view is None:
        _check(False, "logits must have rows of contiguous elements, evenly apart")
    T, E, stride = view
    number = _SCORING.get(scoring)
    if number is None:
        _check(False, "scoring must be one of {}", list(_SCORING))
    if E > 1024 or not 1 <= groups <= 64 or E % groups or not 1 <= top_groups <= groups or not 1 <= best <= 2 or not 1 <= k <= min(64, E // groups * top_groups):
        _check(E <= 1024, "at most 1024 experts, got {}", E)
        _check(1 <= groups <= 64 and E % groups == 0, "groups must be 1 to 64 and divide the {} experts, got {}", E, groups)
        _check(1 <= top_groups <= groups and 1 <= best <= 2, "top_groups must be 1 to {} and group_best 1 or 2, got {} and {}", groups, top_groups, best)
        _check(False, "top_k must be 1 to 64 and at most the {} experts of the groups taken, got {}", E // groups * top_groups, k)
    bias_ptr = None
    if bias is not None:
        _check_tensor(bias, torch.float32, "bias")
        if bias.shape != (E,):
            _check(False, "bias must be [{}]", E)
        bias_ptr = bias.data_ptr()
        _same_device(bias)
    if logits.get_device() != _current_device():
        _same_device(logits)
    new = logits.new_empty
    experts = new((*logits.shape[:-1], k), dtype=torch.int32)
    places, weights = torch.empty_like(experts), torch.empty_like(experts, dtype=torch.float32)
    offsets, rows = new((E + 1,), dtype=torch.int32), new((T * k,), dtype=torch.int32)
    if T == 0:
        offsets.zero_()
        return weights, experts, offsets, rows, places
    nbytes = _L.ac4k_route_experts_workspace_bytes(T, E, k, groups, top_groups) if T > 64 else 0
    ws_ptr = None
    if nbytes > 0:
        ws = new((nbytes,), dtype=torch.uint8)
        ws_ptr = ws.data_ptr()
    _lib.check(_L.ac4k_route_experts(weights.data_ptr(), experts.data_ptr(), offsets.data_ptr(), rows.data_ptr(), places.data_ptr(), logits.data_ptr(), tag,
                                     stride, bias_ptr, T, E, k, number, groups, top_groups, best, bool(renormalize), scale, ws_ptr, nbytes, _stream()))
    return weights, experts, offsets, rows, places


def combine_experts(out, y, weights, places, residual=None):
    """out [.., N] (None: a new tensor) <- residual + the rows of y [M, N] that places [.., k] name, times weights; returns out."""
    tag = _check_float(y, "y")
    if y.dim() != 2:
        _check(False, "y must be a 2d matrix")
    view = _rows_view(y, "y")
    if view is None:
        _check(False, "y must have rows of contiguous elements, evenly apart")
    M, N, y_step = view
    _check_tensor(weights, torch.float32, "weights")
    _check_tensor(places, torch.int32, "places")
    if not places.shape or places.shape[-1] < 1 or weights.shape != places.shape:
        _check(places.dim() >= 1 and places.shape[-1] >= 1, "places must be [.., k]")
        _check(False, "weights must have the shape of places")
    *lead, k = places.shape
    T = places.numel() // k
    dev = _current_device()
    if y.get_device() != dev or weights.get_device() != dev or places.get_device() != dev or residual is not None or out is not None:
        _same_device(y, weights, places, residual, out)
    residual_ptr, residual_step, out_step = None, 0, N
    if residual is not None:
        if residual.dtype is not y.dtype or residual.shape != (*lead, N):
            _check(False, "residual must have the type of y and shape {}", [*lead, N])
        v = _rows_view(residual, "residual")
        if v is None:
            _check(False, "residual must have rows of contiguous elements, evenly apart")
        residual_ptr, residual_step = residual.data_ptr(), v[2]
    if out is None:
        out = y.new_empty((*lead, N))
    else:
        _check(_check_float(out, "out") == tag and list(out.shape) == [*lead, N], "out must have the type of y and shape {}", [*lead, N])
        v = _rows_view(out, "out")
        _check(v is not None and (T <= 1 or v[2] >= N), "out must have rows of contiguous elements, evenly apart")
        out_step = v[2]
        _check(not any(_may_overlap(out, t) for t in (y, weights, places)), "out must not overlap y, weights or places")
        _check(residual is None or _same_rows(out, residual) or not _may_overlap(out, residual), "out may be residual itself, but not overlap it otherwise")
    if T:
        _lib.check(_L.ac4k_combine_experts(out.data_ptr(), out_step, y.data_ptr(), y_step, weights.data_ptr(), places.data_ptr(), residual_ptr, residual_step,
                                           T, k, M, N, tag, _stream()))
    return out


_KINDS = {"rms": 0, "layer": 1}
_NO_VECTOR = (None, 0, 0, None)


def _vector_type(t, name: str, x, dev, before):
    """The type of one of a block's vectors, which is x's or fp32 and that of those before it."""
    if not isinstance(t, torch.Tensor) or t.get_device() != dev or t.dtype is not before and (before is not None or t.dtype is not x.dtype and t.dtype is not torch.float32):
        _check_float(t, name)
        _same_device(t)
        _check(t.dtype in (x.dtype, torch.float32), "{} must have the type of x or be float", name)
        _check(False, "weight, post_weight, gate, scale and shift must have one type")
    return t.dtype


def _norm_vector(t, name: str, shape):
    """(address, elements between vectors, rows that share one; 0: all) of one of a block's vectors, [K] or with leading dims that are those of x or,
    from some dim on, 1; and the tensor that holds it, a copy where no single stride describes it."""
    t_shape, K = t.shape, shape[-1]
    if t_shape[-1] != K:
        _check(False, "{} must have a last dim of {}", name, K)
    if len(t_shape) == 1:
        if t.stride(0) != 1 and K > 1:
            t = t.contiguous()
        return t.data_ptr(), 0, 0, t
    same = len(t_shape) - 1
    if len(t_shape) == len(shape):
        rows, count = 1, 1
        while same and t_shape[same - 1] == 1:
            same -= 1
            rows *= shape[same]
        for n in t_shape[:same]:
            count *= n
        if count == 1 or t_shape[:same] == shape[:same]:
            view = _rows_view(t, name)
            if view is None:
                t = t.contiguous()
                view = _rows_view(t, name)
            if t_shape[:same] == shape[:same]:
                return t.data_ptr(), view[2], 0 if count == 1 else rows, t
    _check(False, "{} must be [{}], or have the leading dims of x or 1 from some dim on, not {}", name, K, list(t_shape))


def block_norm(out, sf, global_scale, given_scale: bool, x, residual, residual_out, weight, post_weight, gate, scale, shift, kind, residual_scale: float,
               precision, eps: float, view=None, fresh=False) -> None:
    """out (and sf, global_scale) <- norm and modulation of the rows of x, or of residual_scale * residual + gate * (norm of x * post_weight), which residual_out
    receives.  view: _rows_view(x), where the caller has it; fresh: out, sf and residual_out are new dense tensors of the right shapes and overlap nothing."""
    tag = _check_float(x, "x")
    view = view or _rows_view(x, "x")
    _check(view is not None, "x must have rows of contiguous elements, evenly apart")
    rows, K, x_step = view
    number, kind_number = _PRECISIONS.get(precision), _KINDS.get(kind)
    if number is None or kind_number is None:
        _check(number is not None, "precision must be one of {}", list(_PRECISIONS))
        _check(False, "kind must be one of {}", list(_KINDS))
    if global_scale is not None:
        _check_tensor(global_scale, torch.float32, "global_scale")
        _check(global_scale.dim() == 0, "global_scale must be a scalar")
    dev = _current_device()
    if x.get_device() != dev or not fresh or global_scale is not None:
        _same_device(x, residual_out, out, sf, global_scale)
    if (residual is None) != (residual_out is None):
        _check(False, "a residual comes with residual_out, and the other way round")
    vector_type, shape, weight_ptr, post_ptr = None, x.shape, None, None
    gate_at = scale_at = shift_at = _NO_VECTOR
    if weight is not None:
        vector_type = _vector_type(weight, "weight", x, dev, None)
        if weight.shape != (K,) or not weight.is_contiguous():
            _check(False, "weight must be contiguous of [{}]", K)
        weight_ptr = weight.data_ptr()
    if post_weight is not None:
        vector_type = _vector_type(post_weight, "post_weight", x, dev, vector_type)
        if post_weight.shape != (K,) or not post_weight.is_contiguous():
            _check(False, "post_weight must be contiguous of [{}]", K)
        post_ptr = post_weight.data_ptr()
    if gate is not None:
        vector_type = _vector_type(gate, "gate", x, dev, vector_type)
        gate_at = _norm_vector(gate, "gate", shape)
    if scale is not None:
        vector_type = _vector_type(scale, "scale", x, dev, vector_type)
        scale_at = _norm_vector(scale, "scale", shape)
    if shift is not None:
        vector_type = _vector_type(shift, "shift", x, dev, vector_type)
        shift_at = _norm_vector(shift, "shift", shape)
    residual_ptr = sum_ptr = None
    residual_step = sum_step = 0
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.dtype is not x.dtype or residual.shape != shape or residual.get_device() != dev:
            _check_float(residual, "residual")
            _same_device(residual)
            _check(False, "residual must have the type and shape of x")
        v = _rows_view(residual, "residual")
        if v is None:
            _check(False, "residual must have rows of contiguous elements, evenly apart")
        residual_ptr, residual_step, sum_ptr, sum_step = residual.data_ptr(), v[2], residual_out.data_ptr(), K
        if not fresh:
            _check(_check_float(residual_out, "residual_out") == tag and residual_out.shape == shape, "residual_out must have the type and shape of x")
            v = _rows_view(residual_out, "residual_out")
            _check(v is not None and (rows <= 1 or v[2] >= K), "residual_out must have rows of contiguous elements, evenly apart")
            sum_step = v[2]
            for t in (x, residual):
                _check(_same_rows(t, residual_out) or not _may_overlap(t, residual_out),
                       "residual_out may be x or residual itself, but not overlap them otherwise")
            for t in (weight, post_weight, gate, scale, shift, global_scale):
                _check(t is None or not _may_overlap(t, residual_out), "residual_out must not overlap a vector or global_scale")
    elif gate is not None or post_weight is not None:
        _check(False, "a gate or a post_weight comes with a residual")
    out_step = K
    if not fresh:
        if precision is None:
            _check(_check_float(out, "out") == tag and out.shape == shape, "out must have the type and shape of x")
            v = _rows_view(out, "out")
            _check(v is not None and (rows <= 1 or v[2] >= K), "out must have rows of contiguous elements, evenly apart")
            out_step = v[2]
            _check(_same_rows(out, x) or not _may_overlap(out, x), "out may be x itself, but not overlap it otherwise")
            for t in (residual, residual_out, weight, post_weight, gate, scale, shift):
                _check(t is None or not _may_overlap(out, t), "out must not overlap residual, residual_out or a vector")
        else:
            nvfp4 = precision == "nvfp4"
            _check_tensor(out, torch.uint8 if nvfp4 else torch.float8_e4m3fn if precision == "fp8e4m3" else torch.int8, "out")
            _check(list(out.shape) == [rows, _align_up(K, 64) // 2 if nvfp4 else _align_up(K, 16)], "meet invalid out shape")
            _check_tensor(sf, torch.float8_e4m3fn if nvfp4 else torch.float32, "sf")
            _check(list(sf.shape) == ([_align_up(K, 64) // 64, _align_up(rows, 16), 4] if nvfp4 else [_align_up(rows, 16)]), "meet invalid sf shape")
    if rows == 0:
        if global_scale is not None and not given_scale:
            global_scale.zero_()  # that of a tensor of zeros
        return
    ws_ptr, nbytes = None, 0
    if number == 3 and not given_scale:
        nbytes = _L.ac4k_block_norm_workspace_bytes(rows, K, tag, number, 0)
        if nbytes > 0:
            ws = x.new_empty((nbytes,), dtype=torch.uint8)
            ws_ptr = ws.data_ptr()
    _lib.check(_L.ac4k_block_norm(out.data_ptr(), out_step, None if sf is None else sf.data_ptr(), None if global_scale is None else global_scale.data_ptr(),
                                  int(given_scale), x.data_ptr(), x_step, residual_ptr, residual_step, sum_ptr, sum_step, weight_ptr, post_ptr, *gate_at[:3],
                                  *scale_at[:3], *shift_at[:3], 2 if vector_type is torch.float32 else tag, rows, K, tag, number, kind_number, residual_scale, eps,
                                  ws_ptr, nbytes, _stream()))
