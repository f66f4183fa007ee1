"""Per-head RMS norm of queries and keys with the position rotation in the same pass (``csrc/kernels/qk_rope.hip``)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import native


def rotary_table(positions: int, dim: int, base: float = 10000.0, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """Cosines and sines ``[positions, dim / 2]`` (fp32) of the angles ``position * base ** (-2 i / dim)``.  The angles are
    formed in 64 bits: in 32 the angle of a position in the tens of thousands has lost all but three digits."""
    if positions < 1 or dim < 2 or dim % 2:
        raise ValueError(f"positions must be positive and dim even (got {positions}, {dim})")
    rates = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rates
    return angles.cos().float(), angles.sin().float()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, *, rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                 positions: Optional[torch.Tensor] = None, interleaved: bool = False,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``R(position) (x / sqrt(mean(x^2) + eps) * weight)`` for every head of ``q`` and ``k``; differentiable in both and in
    the weights.

    ``q``, ``k``: fp16 or bf16 ``[B, S, heads, dim]`` or ``[T, heads, dim]``, ``dim`` a multiple of 8 up to 256; they may
    differ in the number of heads.  Views into a fused projection are read in place (unit inner stride, other strides
    multiples of 8 elements, 16-byte aligned - anything else, here and below, is copied first).

    ``q_weight``, ``k_weight``: ``[dim]``, fp32 or of q's dtype, shared by the heads of a side; without them there is no norm.

    ``rope``: cosines and sines, fp32 ``[positions, rotated / 2]`` (:func:`rotary_table`); without it there is no rotation.
    The first ``rotated`` elements of every head are turned in pairs ``(i, i + rotated / 2)`` - ``rotated`` a multiple of
    16 - or, ``interleaved``, in neighbouring pairs - a multiple of 8.  ``positions``: int64, one per token; an index
    outside the table is clamped into it.  By default a token's position is its place in the sequence ``S`` (or ``T``).

    Returns contiguous tensors of the shapes and dtype of q and k.  All arithmetic is fp32, rounded once at the end; the
    weight gradients are summed in fp32 in a fixed order.  Forward-mode differentiation, a second derivative and traces are
    refused.
    """
    if rope is None and positions is not None:
        raise ValueError("positions mean something only with rope")
    cos, sin = rope if rope is not None else (None, None)
    for name, t in (("cos", cos), ("sin", sin)):
        if t is not None and t.requires_grad:
            raise ValueError(f"{name} is a table of constants: no gradient is formed for it")
    yq, yk = native().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, interleaved, eps)
    return yq, yk


def qk_norm_rope_reference(x: torch.Tensor, weight=None, *, rope=None, positions=None, interleaved=False, eps=1e-6):
    """One side of :func:`qk_norm_rope` in plain differentiable torch operations (the fp32 oracle path)."""
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight
    if rope is None:
        return x
    cos, sin = (t.to(x.dtype) for t in rope)
    if positions is None:
        positions = torch.arange(x.shape[-3], device=x.device)
    positions = positions.clamp(0, cos.shape[0] - 1)
    cos, sin = cos[positions].unsqueeze(-2), sin[positions].unsqueeze(-2)
    n = 2 * cos.shape[-1]
    turned, rest = x[..., :n], x[..., n:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)
