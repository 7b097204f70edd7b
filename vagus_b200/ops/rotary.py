"""Rotary positions for queries and keys in one launch.

``t = position * inv_freq[i]`` rotates channel pair i of the first
``R = 2 len(inv_freq)`` channels of a head by t and multiplies it by ``scale``;
the other channels pass through.  Pairs are channels (2i, 2i+1) in the
``"interleaved"`` layout and (i, i + R/2) in the ``"half"`` layout.  Angles are
formed in 64 bits, so positions in the millions keep their precision.  CUDA runs
``rotary.cu`` for fp32, fp16 and bf16; the backward is the same kernel with the
angles negated.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from ._core import native

LAYOUTS = ("interleaved", "half")
_KERNEL_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _positions(positions, B, L, device):
    """(B, L) int64 positions from an offset, (L,) or (B, L)."""
    if isinstance(positions, int):
        positions = positions + torch.arange(L, device=device)
    return positions.expand(B, L).to(torch.int64)


def rotary_ref(x, positions, inv_freq, layout: str = "interleaved", scale: float = 1.0):
    """The plain form for one tensor (B, L, H, D)."""
    B, L = x.shape[0], x.shape[1]
    ang = _positions(positions, B, L, x.device)[..., None].double() * inv_freq.double()
    up = torch.promote_types(x.dtype, torch.float32)
    cos, sin = (torch.cos(ang) * scale).to(up)[:, :, None], (torch.sin(ang) * scale).to(up)[:, :, None]
    R = 2 * inv_freq.shape[0]
    h = x[..., :R].to(up)
    if layout == "interleaved":
        a, b = h[..., 0::2], h[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = h[..., :R // 2], h[..., R // 2:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y.to(x.dtype), x[..., R:]), -1)


class _Rotary(torch.autograd.Function):
    """q and, unless it is None, k.  The backward applies this function with the
    angles negated and a tangent is rotated like its primal, so derivatives of
    either mode can be taken again."""

    @staticmethod
    def forward(ctx, q, k, pos, offset, inv, interleaved, scale, sign):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(pos, inv)
        ctx.save_for_forward(pos, inv)
        ctx.meta = (offset, interleaved, scale, sign)
        ctx.shapes = (q.shape, None if k is None else k.shape)
        return native().rotary(q, k, pos, offset, inv, interleaved, scale, sign)

    @staticmethod
    def jvp(ctx, tq, tk, tpos, toffset, tinv, *_):
        if tinv is not None:
            raise NotImplementedError("rotary: no derivative with respect to inv_freq on the GPU")
        pos, inv = ctx.saved_tensors
        offset, interleaved, scale, sign = ctx.meta
        of_q, of_k = ctx.shapes
        tq = tk.new_zeros(of_q) if tq is None else tq
        tk = tq.new_zeros(of_k) if tk is None and of_k is not None else tk
        return _run(tq, tk, pos, offset, inv, interleaved, scale, sign)

    @staticmethod
    def backward(ctx, dq, dk):
        pos, inv = ctx.saved_tensors
        offset, interleaved, scale, sign = ctx.meta
        if dq is None and dk is None:
            return (None,) * 8
        if dq is None:
            gk, gq = _run(dk, None, pos, offset, inv, interleaved, scale, -sign)
        else:
            gq, gk = _run(dq, dk, pos, offset, inv, interleaved, scale, -sign)
        return gq, gk, None, None, None, None, None, None


def _run(q, k, *args):
    """The kernel, through the function above where a derivative of either mode may be
    taken (inside a dual level any tensor may carry a tangent)."""
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) \
            or forward_ad._current_level >= 0:
        return _Rotary.apply(q, k, *args)
    return native().rotary(q, k, *args)


def _check(q, k, positions, inv_freq):
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
        raise ValueError("rotary: q (B, L, H, D) and k (B, L, Hk, D)")
    if k is not None and (k.dtype != q.dtype or k.device != q.device):
        raise ValueError("rotary: q and k must share dtype and device")
    B, L, D = q.shape[0], q.shape[1], q.shape[3]
    if inv_freq.dim() != 1 or not inv_freq.is_floating_point() or not 1 <= inv_freq.shape[0] <= D // 2 \
            or inv_freq.device != q.device:
        raise ValueError(f"rotary: inv_freq (R/2,) on q's device with 2 <= R <= {D}")
    if isinstance(positions, torch.Tensor):
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
            raise ValueError("rotary: positions must be int32 or int64 on q's device")
        if tuple(positions.shape) not in ((L,), (B, L)):
            raise ValueError(f"rotary: positions of shape ({L},) or ({B}, {L}), got {tuple(positions.shape)}")


def rotary(q, k, positions, inv_freq, layout: str = "interleaved", scale: float = 1.0):
    """Rotate ``q`` (B, L, H, D) and ``k`` (B, L, Hk, D); returns both.  ``k`` may
    be None: the result is then the rotated ``q`` alone.

    ``positions``: an int (token l sits at positions + l), or an int32 / int64
    tensor (L,) or (B, L).  ``inv_freq``: (R/2,) angle per step of position,
    float64 (other float types are converted), R <= D.  Derivatives of both modes
    are taken with respect to q and k."""
    if layout not in LAYOUTS:
        raise ValueError(f"rotary layout must be one of {LAYOUTS}, got {layout!r}")
    if isinstance(positions, int):
        pos, offset = None, positions
    elif isinstance(positions, torch.Tensor):
        pos, offset = positions, 0
    else:
        raise ValueError("rotary: positions must be an int or a tensor")
    if not q.is_cuda or q.dtype not in _KERNEL_TYPES:
        _check(q, k, positions, inv_freq)
        y = rotary_ref(q, positions, inv_freq, layout, scale)
        return y if k is None else (y, rotary_ref(k, positions, inv_freq, layout, scale))
    # on the GPU the binding checks the arguments (the same conditions)
    out = _run(q, k, pos, offset, inv_freq, layout == "interleaved", scale, 1.0)
    return out[0] if k is None else out
