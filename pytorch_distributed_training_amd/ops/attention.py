"""Softmax attention with a learned relative position bias (gfx950 kernels, ``csrc/kernels/rel_attention.hip``)."""
from __future__ import annotations

import functools
import math
from typing import Optional, Tuple

import torch

from . import native

MAX_BUCKETS = 128
MAX_DISTANCE = 512
MASK_DTYPES = (torch.bool, torch.uint8, torch.int32)  # read in place; other whole numbers are compared with 0 first


@functools.lru_cache(maxsize=None)
def bucket_steps(num_buckets: int, max_distance: int) -> Tuple[int, ...]:
    """First distance of every logarithmic bucket of one side.

    Half of the buckets serve keys at or before the query, half the keys behind it.  Of the ``half`` buckets of a side the
    first ``exact = half // 2`` hold one distance each; logarithmic bucket ``j`` starts at the smallest distance ``d`` with
    ``(d / exact) ** m >= (max_distance / exact) ** j``, ``m = half - exact`` - compared in whole numbers, so a distance
    that lies exactly on a border belongs to the bucket above it - and the last bucket takes everything further away.
    """
    if num_buckets < 4 or num_buckets % 2 or num_buckets > MAX_BUCKETS:
        raise ValueError(f"num_buckets must be even, from 4 to {MAX_BUCKETS} (got {num_buckets})")
    half = num_buckets // 2
    exact = half // 2
    if not exact < max_distance <= MAX_DISTANCE:
        raise ValueError(f"max_distance must be above num_buckets // 4 = {exact} and at most {MAX_DISTANCE} (got {max_distance})")
    m, steps, d = half - exact, [], exact
    for j in range(m):
        while d ** m * exact ** j < max_distance ** j * exact ** m:
            d += 1
        steps.append(d)
    return tuple(steps)


def relative_bucket(distance: torch.Tensor, num_buckets: int, max_distance: int) -> torch.Tensor:
    """Bucket of every ``key position - query position`` (the rule of :func:`bucket_steps`), in plain torch operations."""
    steps = bucket_steps(num_buckets, max_distance)
    half = num_buckets // 2
    exact = half // 2
    far = distance.abs()
    log = torch.bucketize(far, torch.tensor(steps, device=distance.device), right=True) - 1 + exact
    return torch.where(far < exact, far, log) + half * (distance > 0).to(far.dtype)


def mask_bits(key_mask: torch.Tensor) -> torch.Tensor:
    """A key mask ``[B, S]`` as the kernels read it: one bit per key, int64 ``[B, ceil(S / 64)]``."""
    if key_mask.dtype not in MASK_DTYPES:
        key_mask = key_mask.ne(0)
    return native().rel_mask_bits(key_mask)


def relative_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                       max_distance: int = 128, key_mask: Optional[torch.Tensor] = None,
                       cu_seqlens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None,
                       scale: Optional[float] = None, dropout_p: float = 0.0, rng=None, site: int = 0) -> torch.Tensor:
    """``softmax(scale q k^T + bias[bucket(j - i)]) v`` per head, both directions attended; differentiable in q, k, v, bias.

    ``q``, ``k``, ``v``: fp16 or bf16 ``[B, S, heads, dim]`` of one shape, ``dim`` a multiple of 8 up to 128, any ``S``; views
    into a fused projection are read in place (unit inner stride, other strides multiples of 8 elements, 16-byte aligned -
    anything else is copied first).  With ``cu_seqlens`` (int32 ``[B + 1]`` on the GPU, ascending from 0) they are the packed rows
    ``[T, heads, dim]`` of sequences of different lengths instead, ``max_seqlen`` the longest of them; rows from
    ``cu_seqlens[-1]`` on belong to no sequence, their outputs and gradients are zero.  So are those of rows beyond
    ``max_seqlen`` in a sequence that is longer after all: the sequence is cut there.  Memory for row statistics and the number of
    workgroups grow with the number of sequences times ``max_seqlen``.

    ``bias``: ``[buckets, heads]``, fp32 or of q's dtype; ``None`` leaves it out.  ``max_distance`` (at most 512): where the
    last bucket of each side begins at the latest, see :func:`bucket_steps`.

    ``key_mask``: ``[B, S]`` bool or integer, non-zero = attended, holes allowed; a key that is not attended takes no part
    whatever its row holds (infinities and NaN included) and gets zero gradients.  A query without any attended key has a
    zero output and no gradient.  An additive float mask is refused.

    ``scale`` (``1 / sqrt(dim)`` by default): not zero, of a size from 2^-64 to 2^64.

    ``dropout_p`` (at most 0.99) with ``rng`` (an :class:`~.fused.RngKey`) and ``site``: dropout on the probabilities with the framework's
    counter-based masks.

    Forward and backward may be captured into a graph; masks and ``cu_seqlens`` are then read at every replay (``max_seqlen`` and
    the shapes are those of the capture).  As with any operator, let no eager autograd graph of the same leaves live meanwhile:
    their gradients would be accumulated on its stream, outside the capture.

    Forward-mode differentiation, a second derivative and traces are refused.

    Returns a contiguous tensor of q's shape and dtype.  Probabilities and their gradients are rounded to q's dtype as
    operands of the matrix products (in fp16 by a power of two above their size, so that small gradients of the output keep
    their digits); scores, softmax statistics and all sums are fp32.  The gradient of ``bias`` is summed in
    fp32 in a fixed order, so it is the same in every run.
    """
    if torch._C._is_tracing():  # (sizes are tensors there, and bucket_steps() would keep them)
        raise RuntimeError("relative_attention cannot be traced: a trace would hold its empty output tensor")
    if q.dim() not in (3, 4) or (q.dim() == 3) != (cu_seqlens is not None):
        raise ValueError("q, k, v must be [B, S, heads, dim], or packed [T, heads, dim] with cu_seqlens")
    if cu_seqlens is not None:
        if key_mask is not None:
            raise ValueError("packed rows take no key mask: leave the masked keys out of the rows")
        if max_seqlen is None:
            raise ValueError("packed rows need max_seqlen, the longest sequence")
    elif key_mask is not None:
        if tuple(key_mask.shape) != tuple(q.shape[:2]):
            raise ValueError(f"key_mask must be [B, S] = {tuple(q.shape[:2])}, got {tuple(key_mask.shape)}")
        if key_mask.is_floating_point() or key_mask.is_complex():
            raise ValueError("key_mask holds truth values (non-zero = attended), not additive scores")
        if key_mask.dtype not in MASK_DTYPES:
            key_mask = key_mask.ne(0)
    steps: Tuple[int, ...] = ()
    if bias is not None:
        if bias.dim() != 2:
            raise ValueError("bias must be [buckets, heads]")
        steps = bucket_steps(bias.shape[0], max_distance)
        if not bias.is_contiguous():
            bias = bias.contiguous()
    else:
        max_distance = 0
    if not 0.0 <= dropout_p <= 0.99:
        raise ValueError(f"dropout_p must be from 0 to 0.99 (got {dropout_p})")
    if dropout_p > 0.0 and rng is None:
        raise ValueError("dropout needs rng, the key of the forward pass")
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if not 2.0 ** -64 <= abs(scale) <= 2.0 ** 64:  # (fp32 holds the scale, its reciprocal and their products with the scores)
        raise ValueError(f"the size of scale must be from 2^-64 to 2^64 (got {scale})")
    state, micro, sids = (rng.state, rng.counter, rng.sample_ids) if dropout_p > 0.0 else (None, 0, None)
    return native().relative_attention(q, k, v, bias, max_distance, steps, key_mask, cu_seqlens, int(max_seqlen or 0), scale, state,
                                       dropout_p, micro, site, sids)


def relative_attention_reference(q, k, v, bias=None, *, max_distance=128, key_mask=None, scale=None, dropout_p=0.0, training=False):
    """The padded form of :func:`relative_attention` in plain differentiable torch operations (the fp32 oracle path)."""
    n = q.shape[1]
    scores = torch.einsum("bihd,bjhd->bhij", q, k) * (1.0 / math.sqrt(q.shape[-1]) if scale is None else scale)
    if bias is not None:
        place = torch.arange(n, device=q.device)
        scores = scores + bias[relative_bucket(place[None, :] - place[:, None], bias.shape[0], max_distance)].permute(2, 0, 1)
    if key_mask is not None:
        dead = key_mask.eq(0)[:, None, None, :]
        scores = scores.masked_fill(dead, torch.finfo(scores.dtype).min)
    probs = torch.softmax(scores, dim=-1)
    if key_mask is not None:
        probs = probs.masked_fill(dead, 0.0)
    probs = torch.nn.functional.dropout(probs, dropout_p, training)
    return torch.einsum("bhij,bjhd->bihd", probs, v)
