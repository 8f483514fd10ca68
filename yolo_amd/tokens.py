"""Token operators over feature maps: layer norm, attention and a learned relative position bias, with their gradients.

A map's NHWC pixels are its tokens: a (B, H, W, C) activation is ``(B, H*W, heads, C // heads)`` here without a copy, also as
a channel slice of a wider buffer.  Tensors live on the GPU; attention takes bfloat16, layer norm bfloat16 or float32 rows.
Gradients flow through ``torch.autograd`` (once: the gradients carry no graph of their own; forward-mode tangents and
``torch.jit.trace`` are refused); all arithmetic happens inside
libyolo_amd.so, on torch's current stream of the tensors' device, and equal inputs give equal bits.  Results and scratch are
torch allocations of each call, so calls on different streams, or captured into different graphs, share nothing.  A training
step that is captured into a graph takes its forward and backward pass together; no eager result of the same leaves may be
alive meanwhile (autograd would tie the captured stream to the default one; where these operators' backward passes meet
that, they raise before it breaks the capture).
``engine.Program`` records the forward passes into a layer program.
"""
from typing import List, Optional

import torch

from . import lib as _lib                     # loads libyolo_amd.so, which the binding below links against
from . import _torch_ops as _ops              # no fallback: a missing binding is an import error (python -m yolo_amd.build)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5
               ) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (at most 16384 channels).

    x: (..., C) bfloat16 or float32, evenly spaced rows (also a channel slice); weight, bias: (C,) of one type, bfloat16 or
    float32, or None.  Statistics and the sums of the weight's gradient are float32 whatever the types."""
    return _ops.layer_norm(x, weight, bias, eps)


def axis_buckets(n: int, buckets: int, max_distance: int) -> List[int]:
    """Bucket of each signed distance -(n - 1) .. n - 1 along one axis.  Half of the ``buckets`` go to positive distances; of
    a half, the first half hold one distance each and the others grow by a constant factor up to ``max_distance``, the last
    one holding all that is farther.  Decided by whole-number comparisons, so a border falls on one side everywhere."""
    if n < 1:
        raise _lib.YamdError(f"an axis has at least one position, got {n}")
    if buckets < 4 or buckets % 4:
        raise _lib.YamdError(f"buckets must be a positive multiple of 4, got {buckets}")
    half, near = buckets // 2, buckets // 4
    if max_distance <= near:
        raise _lib.YamdError(f"max_distance must be above {near} for {buckets} buckets, got {max_distance}")
    steps = half - near
    # first distance of bucket near + t: the smallest m with (m / near)^steps >= (max_distance / near)^t
    first, m = [], near
    for t in range(steps):
        while m < n and m ** steps * near ** t < near ** steps * max_distance ** t:      # (n: beyond the axis)
            m += 1
        first.append(m)
    mag = []
    t = 0
    for m in range(n):
        while t + 1 < steps and m >= first[t + 1]:
            t += 1
        mag.append(m if m < near else near + t)
    return [mag[-d] for d in range(-(n - 1), 0)] + [mag[0]] + [half + mag[d] for d in range(1, n)]


class RelativePosition:
    """Which row of a learned table each distance between two positions of an ``h x w`` map reads.

    Along each axis a distance (query minus key) falls into one of ``buckets`` buckets (``axis_buckets``); a table for a map
    has ``buckets**2`` rows (vertical bucket times ``buckets`` plus horizontal bucket), one for a sequence (``h == 1``) has
    ``buckets``.  Built once per map size and kept beside the table."""

    def __init__(self, h: int, w: int, buckets: int, max_distance: int, device="cuda"):
        if h < 1 or w < 1 or h * w > 1 << 24:
            raise _lib.YamdError(f"bad map {h} x {w}")
        if h > 1 and w > 760:
            raise _lib.YamdError(f"a map of several rows is at most 760 wide, got {h} x {w}")
        self.h, self.w, self.buckets, self.max_distance = int(h), int(w), int(buckets), int(max_distance)
        if buckets ** (2 if h > 1 else 1) > 1 << 20:
            raise _lib.YamdError(f"more than 2^20 rows in the table of {buckets} buckets")
        of = torch.tensor(axis_buckets(w, buckets, max_distance), dtype=torch.int64)
        self.rows = buckets
        if h > 1:
            by = torch.tensor(axis_buckets(h, buckets, max_distance), dtype=torch.int64)
            of = (by[:, None] * buckets + of[None, :]).reshape(-1)
            self.rows = buckets * buckets
        self.distances = of.numel()
        start = torch.zeros(self.rows + 1, dtype=torch.int64)
        start[1:] = torch.cumsum(torch.bincount(of, minlength=self.rows), 0)
        # bucket of each distance, and the distances in order of bucket with each bucket's first place (for the gradient)
        self.bucket_of = of.to(torch.int32).to(device)
        self.order = torch.argsort(of, stable=True).to(torch.int32).to(device)
        self.start = start.to(torch.int32).to(device)


def relative_bias(table: torch.Tensor, position: RelativePosition) -> torch.Tensor:
    """The bias of every distance, (heads, position.distances) float32, from a learned ``(position.rows, heads)`` table
    (bfloat16 or float32).  ``attention`` reads it by distance; a program that serves fixed weights computes it once."""
    return _ops.relative_bias(table, position.bucket_of, position.order, position.start)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None, key_mask: Optional[torch.Tensor] = None,
              bias: Optional[torch.Tensor] = None, position: Optional[RelativePosition] = None) -> torch.Tensor:
    """``softmax(scale * q k^T + bias) v`` per image and head: (B, Lq, heads, d) bfloat16.

    q: (B, Lq, heads, d); k, v: (B, Lk, kv_heads, d), heads a multiple of kv_heads (consecutive heads share keys); bfloat16,
    d a multiple of 8 up to 128, channels contiguous and rows at multiples of 16 bytes (copy a broadcast tensor first).  scale: 1/sqrt(d) by default.  key_mask: (B, Lk) bool, False = not attended (what
    k and v hold there does not matter); a query left without keys gets zeros and no gradient.  bias: (heads,
    position.distances) float32, see ``relative_bias``, for self-attention over the h x w map (or sequence) of ``position``;
    values below -1e5 (-inf, the type's lowest value, ...) mask, and a query with only such scores is left without keys
    (with a bias, the largest score of a query that has keys must lie above -1e5).
    Scores, statistics and sums are float32 (scores should stay below 1e6 in size: beyond, their rounding reaches the
    probabilities, and from 5e8 on a result may be NaN or zeros); probabilities are rounded to bfloat16 for the products with v and do, and score
    gradients for the products with q and k."""
    if (bias is None) != (position is None):
        raise _lib.YamdError("bias and position go together")
    if position is None:
        return _ops.attention(q, k, v, scale, key_mask, None, 0, 0)
    return _ops.attention(q, k, v, scale, key_mask, bias, position.h, position.w)
