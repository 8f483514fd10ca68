"""Token operators over feature maps: layer norm, attention and a learned relative position bias, with their gradients.

A map's NHWC pixels are its tokens: a (B, H, W, C) activation is ``(B, H*W, heads, C // heads)`` here without a copy, also as
a channel slice of a wider buffer.  Tensors live on the GPU; attention takes bfloat16, layer norm bfloat16 or float32 rows.
Gradients flow through ``torch.autograd``; all arithmetic happens inside libyolo_amd.so, on torch's current stream of the
tensors' device, and equal inputs give equal bits.  ``engine.Program`` records the forward passes into a layer program.
"""
import contextlib
import ctypes
import math
from typing import List, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import lib as _lib

LIB = _lib.LIB
_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_byref = ctypes.byref


def _on(device: torch.device):
    """Makes ``device`` the current one for a library call (kernels are launched on the current device)."""
    return contextlib.nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return int(torch.cuda.current_stream(device).cuda_stream)


def _require(t: torch.Tensor, name: str, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise _lib.YamdError(f"{name} must live on the GPU: yolo_amd has no CPU path")
    if device is not None and t.device != device:
        raise _lib.YamdError(f"{name} is on {t.device}, expected {device}")


def _wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- layer norm ---------------------------------------------------------------------------------------------------------
def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """(..., C) as evenly spaced rows (N, C), without a copy."""
    c = t.shape[-1]
    try:
        r = t.view(-1, c) if t.numel() else t.reshape(0, c)
    except RuntimeError:
        raise _lib.YamdError(f"{name}: rows must be evenly spaced, got shape {tuple(t.shape)} strides {t.stride()}") from None
    if c > 1 and t.numel() and r.stride(1) != 1:
        raise _lib.YamdError(f"{name}: channels must be contiguous, got strides {t.stride()}")
    return r


def _param(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _norm_forward(x, weight, bias, eps, stats: bool):
    rows = _rows(x, "x")
    n, c = rows.shape
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    ms = torch.empty((2, n), dtype=torch.float32, device=dev) if stats else None
    p = weight if weight is not None else bias
    with _on(dev):
        _lib.check(LIB.yamd_layer_norm(rows.data_ptr(), rows.stride(0) if n > 1 else c, _param(weight), _param(bias),
                                       _DTYPES[p.dtype] if p is not None else 0, eps, y.data_ptr(), c,
                                       ms[0].data_ptr() if stats else None, ms[1].data_ptr() if stats else None, n, c,
                                       _DTYPES[x.dtype], _stream(dev)), "layer_norm")
    return y, ms


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, ms = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, ms)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, ms = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        rows = _rows(x, "x")
        n, c = rows.shape
        dev = x.device
        dys = dy.contiguous()
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_x else None
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        ws = None
        if want_w or want_b:
            ws = torch.empty(LIB.yamd_layer_norm_backward_workspace_bytes(n, c), dtype=torch.uint8, device=dev)
        p = weight if weight is not None else bias
        with _on(dev):
            _lib.check(LIB.yamd_layer_norm_backward(dys.data_ptr(), c, rows.data_ptr(), rows.stride(0) if n > 1 else c, _param(weight),
                                                    _DTYPES[p.dtype] if p is not None else 0, ms[0].data_ptr(), ms[1].data_ptr(),
                                                    _param(dx), c, _param(dw), _param(db), n, c, _DTYPES[x.dtype], _param(ws),
                                                    0 if ws is None else ws.numel(), _stream(dev)), "layer_norm_backward")
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5
               ) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (at most 16384 channels).

    x: (..., C) bfloat16 or float32, evenly spaced rows (also a channel slice); weight, bias: (C,) of one type, bfloat16 or
    float32, or None.  Statistics and the sums of the weight's gradient are float32 whatever the types."""
    _require(x, "x")
    if x.dtype not in _DTYPES:
        raise _lib.YamdError(f"x must be bfloat16 or float32, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 16384:
        raise _lib.YamdError(f"x must have 1 to 16384 channels, got shape {tuple(x.shape)}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        _require(t, name, x.device)
        if t.dtype not in _DTYPES or t.shape != x.shape[-1:] or not t.is_contiguous():
            raise _lib.YamdError(f"{name} must be contiguous ({x.shape[-1]},) bfloat16 or float32, got {tuple(t.shape)} {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise _lib.YamdError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0:
        raise _lib.YamdError(f"eps must not be negative, got {eps}")
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


# ---- relative position bias -----------------------------------------------------------------------------------------------
def axis_buckets(n: int, buckets: int, max_distance: int) -> List[int]:
    """Bucket of each signed distance -(n - 1) .. n - 1 along one axis.  Half of the ``buckets`` go to positive distances; of
    a half, the first half hold one distance each and the others grow by a constant factor up to ``max_distance``, the last
    one holding all that is farther.  Decided by whole-number comparisons, so a border falls on one side everywhere."""
    if buckets < 4 or buckets % 4:
        raise _lib.YamdError(f"buckets must be a positive multiple of 4, got {buckets}")
    half, near = buckets // 2, buckets // 4
    if max_distance <= near:
        raise _lib.YamdError(f"max_distance must be above {near} for {buckets} buckets, got {max_distance}")
    steps = half - near
    # first distance of bucket near + t: the smallest m with (m / near)^steps >= (max_distance / near)^t
    first, m = [], near
    for t in range(steps):
        while m ** steps * near ** t < near ** steps * max_distance ** t:
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
        if h > 1 and w > 768:
            raise _lib.YamdError(f"a map of several rows is at most 768 wide, got {h} x {w}")
        self.h, self.w, self.buckets, self.max_distance = int(h), int(w), int(buckets), int(max_distance)
        bx = torch.tensor(axis_buckets(w, buckets, max_distance), dtype=torch.int64)
        if h == 1:
            of, self.rows = bx, buckets
        else:
            by = torch.tensor(axis_buckets(h, buckets, max_distance), dtype=torch.int64)
            of, self.rows = (by[:, None] * buckets + bx[None, :]).reshape(-1), buckets * buckets
        self.distances = of.numel()
        start = torch.zeros(self.rows + 1, dtype=torch.int64)
        start[1:] = torch.cumsum(torch.bincount(of, minlength=self.rows), 0)
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device = dev
        self.bucket_of = of.to(torch.int32).to(dev)
        self.order = torch.argsort(of, stable=True).to(torch.int32).to(dev)
        self.start = start.to(torch.int32).to(dev)


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, position):
        ctx.position, ctx.dtype = position, table.dtype
        return _bias_forward(table, position)

    @staticmethod
    @once_differentiable
    def backward(ctx, dbias):
        pos = ctx.position
        d = dbias.contiguous()
        heads = d.shape[0]
        dtable = torch.empty((pos.rows, heads), dtype=ctx.dtype, device=d.device)
        with _on(d.device):
            _lib.check(LIB.yamd_relative_bias_backward(d.data_ptr(), pos.order.data_ptr(), pos.start.data_ptr(), pos.distances, heads,
                                                       pos.rows, dtable.data_ptr(), _DTYPES[ctx.dtype], _stream(d.device)),
                       "relative_bias_backward")
        return dtable, None


def _bias_forward(table, position):
    heads = table.shape[1]
    bias = torch.empty((heads, position.distances), dtype=torch.float32, device=table.device)
    with _on(table.device):
        _lib.check(LIB.yamd_relative_bias(table.data_ptr(), _DTYPES[table.dtype], position.bucket_of.data_ptr(), position.distances,
                                          heads, position.rows, bias.data_ptr(), _stream(table.device)), "relative_bias")
    return bias


def relative_bias(table: torch.Tensor, position: RelativePosition) -> torch.Tensor:
    """The bias of every distance, (heads, position.distances) float32, from a learned ``(position.rows, heads)`` table
    (bfloat16 or float32).  ``attention`` reads it by distance; a program that serves fixed weights computes it once."""
    _require(table, "table", position.device)
    if table.dtype not in _DTYPES or table.dim() != 2 or table.shape[0] != position.rows or not 1 <= table.shape[1] <= 65535 \
            or not table.is_contiguous():
        raise _lib.YamdError(f"table must be contiguous ({position.rows}, heads) bfloat16 or float32, got {tuple(table.shape)} {table.dtype}")
    if _wants_grad(table):
        return _RelativeBias.apply(table, position)
    return _bias_forward(table, position)


# ---- attention ----------------------------------------------------------------------------------------------------------
def _tokens(t: torch.Tensor) -> "_lib.Tokens":
    # (a stride of a dimension of one element is never used; torch leaves any value there)
    return _lib.Tokens(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _desc(q, k, scale, position) -> "_lib.AttentionDesc":
    h, w = (0, 0) if position is None else (position.h, position.w)
    return _lib.AttentionDesc(q.shape[0], q.shape[2], k.shape[2], q.shape[3], q.shape[1], k.shape[1], h, w, scale)


def _attention_forward(q, k, v, scale, mask, bias, position, stats: bool):
    dev = q.device
    b, lq, heads, _ = q.shape
    lse = torch.empty((b, heads, lq), dtype=torch.float32, device=dev) if stats else None
    if q.numel() == 0 or k.numel() == 0:             # no query, or no key: rows left without keys are zero
        if lse is not None:
            lse.fill_(-math.inf)
        return torch.zeros(q.shape, dtype=q.dtype, device=dev), lse
    o = torch.empty(q.shape, dtype=q.dtype, device=dev)
    d = _desc(q, k, scale, position)
    nbytes = LIB.yamd_attention_workspace_bytes(_byref(d), int(bias is not None))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _on(dev):
        _lib.check(LIB.yamd_attention(_byref(d), _byref(_tokens(q)), _byref(_tokens(k)), _byref(_tokens(v)), _param(mask),
                                      0 if mask is None else mask.stride(0), _param(bias), _byref(_tokens(o)), _param(lse), _param(ws),
                                      nbytes, _stream(dev)), "attention")
    return o, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, mask, scale, position):
        o, lse = _attention_forward(q, k, v, scale, mask, bias, position, True)
        ctx.save_for_backward(q, k, v, bias, mask, o, lse)
        ctx.scale, ctx.position = scale, position
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, bias, mask, o, lse = ctx.saved_tensors
        dev = q.device
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
        dbias = None if bias is None else torch.empty_like(bias)
        if q.numel() == 0 or k.numel() == 0:
            for t in (dq, dk, dv, dbias):
                if t is not None:
                    t.zero_()
            return dq, dk, dv, dbias, None, None, None
        do = do.contiguous()
        d = _desc(q, k, ctx.scale, ctx.position)
        nbytes = LIB.yamd_attention_backward_workspace_bytes(_byref(d), int(bias is not None))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        with _on(dev):
            _lib.check(LIB.yamd_attention_backward(_byref(d), _byref(_tokens(q)), _byref(_tokens(k)), _byref(_tokens(v)), _param(mask),
                                                   0 if mask is None else mask.stride(0), _param(bias), _byref(_tokens(o)),
                                                   lse.data_ptr(), _byref(_tokens(do)), _byref(_tokens(dq)), _byref(_tokens(dk)),
                                                   _byref(_tokens(dv)), _param(dbias), ws.data_ptr(), nbytes, _stream(dev)),
                       "attention_backward")
        return dq, dk, dv, dbias, None, None, None


def _check_tokens(t: torch.Tensor, name: str, device, shape: Tuple[int, ...]) -> None:
    _require(t, name, device)
    if t.dtype != torch.bfloat16:
        raise _lib.YamdError(f"{name} must be bfloat16, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise _lib.YamdError(f"{name} must be {shape}, got {tuple(t.shape)}")
    if t.numel() == 0:
        return
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(n > 1 and (s % 8 or s < 8) for n, s in zip(shape[:3], t.stride()[:3])):
        raise _lib.YamdError(f"{name}: channels must be contiguous and tokens, heads and images start at multiples of 16 bytes "
                             f"(strides {t.stride()})")


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None, key_mask: Optional[torch.Tensor] = None,
              bias: Optional[torch.Tensor] = None, position: Optional[RelativePosition] = None) -> torch.Tensor:
    """``softmax(scale * q k^T + bias) v`` per image and head: (B, Lq, heads, d) bfloat16.

    q: (B, Lq, heads, d); k, v: (B, Lk, kv_heads, d), heads a multiple of kv_heads (consecutive heads share keys); bfloat16,
    d a multiple of 8 up to 128.  scale: positive, 1/sqrt(d) by default.  key_mask: (B, Lk) bool, False = not attended (what
    k and v hold there does not matter); a query left without keys gets zeros and no gradient.  bias: (heads,
    position.distances) float32, see ``relative_bias``, for self-attention over the h x w map (or sequence) of ``position``.
    Scores, statistics and sums are float32; probabilities are rounded to bfloat16 for the products with v and do, and score
    gradients for the products with q and k."""
    _require(q, "q")
    if q.dim() != 4 or not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise _lib.YamdError("q must be (batch, tokens, heads, channels) and k, v (batch, tokens, kv_heads, channels)")
    b, lq, heads, d = q.shape
    lk, kv_heads = k.shape[1], k.shape[2]
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise _lib.YamdError(f"{heads} heads do not share {kv_heads} key heads evenly")
    if not 8 <= d <= 128 or d % 8:
        raise _lib.YamdError(f"channels per head must be a multiple of 8 up to 128, got {d}")
    _check_tokens(q, "q", q.device, (b, lq, heads, d))
    _check_tokens(k, "k", q.device, (b, lk, kv_heads, d))
    _check_tokens(v, "v", q.device, (b, lk, kv_heads, d))
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise _lib.YamdError(f"scale must be positive and finite, got {scale}")
    if key_mask is not None:
        _require(key_mask, "key_mask", q.device)
        if key_mask.dtype != torch.bool or tuple(key_mask.shape) != (b, lk) or (lk > 1 and key_mask.stride(1) != 1) \
                or (b > 1 and lk > 0 and key_mask.stride(0) < lk):
            raise _lib.YamdError(f"key_mask must be bool {(b, lk)} with contiguous rows, got {tuple(key_mask.shape)} {key_mask.dtype}")
    if (bias is None) != (position is None):
        raise _lib.YamdError("bias and position go together")
    if bias is not None:
        _require(bias, "bias", q.device)
        if not lq == lk == position.h * position.w:
            raise _lib.YamdError(f"a position bias needs Lq == Lk == {position.h} * {position.w}, got {lq} and {lk}")
        if bias.dtype != torch.float32 or tuple(bias.shape) != (heads, position.distances) or not bias.is_contiguous():
            raise _lib.YamdError(f"bias must be contiguous float32 {(heads, position.distances)}, got {tuple(bias.shape)} {bias.dtype}")
    if _wants_grad(q, k, v, bias):
        return _Attention.apply(q, k, v, bias, key_mask, scale, position)
    return _attention_forward(q, k, v, scale, key_mask, bias, position, False)[0]
