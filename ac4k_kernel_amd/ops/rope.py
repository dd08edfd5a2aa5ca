"""`rope`: rotary positions with several axes (text, images, video).  The reference's `rope3d` (python/ac4k_kernel/ops/rope_3d.py,
lib/cuda/sm120/rope3d.cu:23-129) turns pairs by three axes in 64 bits; here tables are made from angles in 64 bits and
the rotation is in fp32."""
from __future__ import annotations

import torch

from .. import _rocm_ops


def rope_table(sections, length, theta=10000.0, shared=False, device="cuda"):
    """Table for `rope`: fp32 [length, sum(sections), 2], cosine and sine of position * frequency, angles in 64 bits.

    sections: pairs of each axis.  The n pairs of an axis have the frequencies theta^(-j/n), j = 0 .. n-1; with shared=True the
    pairs of all axes have one series, theta^(-j/pairs).
    """
    sections = (sections,) if isinstance(sections, int) else tuple(sections)
    counts = (sum(sections),) if shared else sections
    if sum(sections) < 1 or min(sections) < 0 or length < 1:
        raise RuntimeError("a table needs pairs and positions")
    exponent = torch.cat([torch.arange(n, dtype=torch.float64, device=device) / n for n in counts if n > 0])
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * torch.pow(float(theta), -exponent)
    return torch.stack((angle.cos(), angle.sin()), dim=-1).to(torch.float32)


def rope(x, table, positions=None, grid=None, sections=None, layout="BNHD", interleaved=True, inverse=False, out=None):
    """x, or two tensors (q, k) in one call, with the pairs of every head turned by the angles of their token.

    x [B, N, H, D] (layout "BNHD") or [B, H, N, D] ("BHND"), bf16, fp16 or fp32, D contiguous, any other strides; the tensors of a pair may
    differ in H.  table fp32 [length, pairs, 2] of (cos, sin), see `rope_table`; the first 2 * pairs elements of a head are turned, in pairs
    (2j, 2j+1), or (j, j + pairs) with interleaved=False, the others copied.  sections: pairs of each axis, in order (default: one axis).
    Where the tokens are: positions, int32 or int64 [axes, B, N], [B, N] for one axis, or [axes, 1, N] / [N] for all batches alike; or grid, the sizes
    of the axes, whose places the tokens take in row-major order; default: token n is at n.  A token with a negative position, or behind
    the last place of the grid, stays as it is; a position the table does not have gives NaN.
    inverse turns back: the gradient of the rotation.  out may be x itself.  Returns a tensor, or a tuple for a pair.
    """
    if layout not in ("BNHD", "BHND"):
        raise RuntimeError(f"Unsupported layout: {layout}")
    single = isinstance(x, torch.Tensor)
    xs = (x,) if single else tuple(x)
    for t in xs:
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise RuntimeError("rope takes one or two 4D tensors")
        if t.stride(3) != 1:
            xs = tuple([u.contiguous() if u.stride(3) != 1 else u for u in xs])
    if not xs or not isinstance(table, torch.Tensor) or table.dim() != 3:
        raise RuntimeError("rope takes one or two 4D tensors and a table of [length, pairs, 2]")
    outs = None if out is None else (out,) if single else tuple(out)
    sections = (table.shape[1],) if sections is None else (sections,) if isinstance(sections, int) else tuple(sections)
    bnhd = layout == "BNHD"
    if positions is None:
        tokens = xs[0].shape[1 if bnhd else 2]
        if grid is None:
            if len(sections) != 1:
                raise RuntimeError("several axes need positions or a grid")
            grid = (tokens,)
        grid = tuple([int(g) for g in grid]) if tokens else (1,) * len(sections)
    elif isinstance(positions, torch.Tensor):
        while positions.dim() < 3:
            positions = positions.unsqueeze(0)
        if positions.shape[1] == 1 != xs[0].shape[0]:
            positions = positions.expand(-1, xs[0].shape[0], -1)
    else:
        raise RuntimeError("positions must be a CUDA tensor of int32 or int64")
    outs = _rocm_ops.rope(outs, xs, table, sections, positions, grid, bnhd, interleaved, inverse)
    return outs[0] if single else outs
