"""GPU tests of the token operators against plain 64-bit implementations.

Tolerances are elementwise bounds derived from the roundings that the kernels make, computed beside the reference in 64 bits:
bf16 rounds by at most U = 2^-8 of the value (half a step).  Attention rounds the probabilities P for P v and P^T do, the
score gradients dS for dS k and dS^T q, and the results; D = rowsum(do o) inherits the error of o.  Float32 parts (scores,
statistics, sums) get RHO, a bound of a probability's relative error that is computed from the scores' sizes."""
import ctypes
import math

import pytest
import torch

from yolo_amd import lib as L
from yolo_amd import tokens
from yolo_amd.engine import Program

pytestmark = pytest.mark.gpu

U = torch.finfo(torch.bfloat16).eps / 2
F = torch.finfo(torch.float32).eps / 2


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _within(name, got, want, tol):
    got = got.detach().double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
    assert over <= 0, f"{name}: beyond its bound by {over} (largest value {want.abs().max().item()})"


# ---- layer norm -----------------------------------------------------------------------------------------------------------
def _norm_case(dev, x, w, b, eps, dy, dtype_round):
    """(y, dx, dw, db) in 64 bits and their bounds.  K: float32 operations in a row of sums: a thread adds at most 16 terms,
    six exchange steps and sixteen waves follow, and the two passes over the row use both statistics."""
    K = 64
    xd, dyd = x.detach().double(), dy.double()
    wd = torch.ones(x.shape[-1], dtype=torch.float64, device=dev) if w is None else w.detach().double()
    bd = torch.zeros_like(wd) if b is None else b.detach().double()
    mu = xd.mean(1, keepdim=True)
    var = ((xd - mu) ** 2).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (xd - mu) * r
    big = xd.abs().amax(1, keepdim=True)
    e_xh = K * F * (xh.abs() + r * big)                                # error of xh: of the mean (relative to the row), of r
    y = xh * wd + bd
    t_y = dtype_round * y.abs() + e_xh * wd.abs() + 4 * F * (y.abs() + bd.abs()) + 1e-30
    g = dyd * wd
    m0, m1 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - m0 - xh * m1)
    e_m1 = (g.abs() * e_xh).mean(1, keepdim=True) + K * F * (g * xh).abs().mean(1, keepdim=True)
    t_dx = dtype_round * dx.abs() + K * F * r * (g.abs() + g.abs().mean(1, keepdim=True) + (xh * m1).abs()) \
        + r * (e_xh * m1.abs() + xh.abs() * e_m1) * 1.01 + 1e-30
    rows = K + x.shape[0] / 16                                         # the longest chain of row additions
    dw, db = (dyd * xh).sum(0), dyd.sum(0)
    t_dw = (dyd.abs() * e_xh).sum(0) + rows * F * (dyd * xh).abs().sum(0) + 1e-30
    t_db = rows * F * dyd.abs().sum(0) + 1e-30
    return (y, dx, dw, db), (t_y, t_dx, t_dw, t_db)


@pytest.mark.parametrize("rows,c", [(1, 1), (1, 8), (3, 7), (17, 16), (64, 64), (65, 128), (33, 129), (400, 171), (50, 256), (50, 257), (9, 512),
                                    (9, 520), (31, 1000), (5, 1024), (5, 1025), (7, 2048), (3, 3000), (2, 4096), (3, 4100), (2, 8192),
                                    (2, 16383), (3, 16384), (5000, 96), (20011, 40)])
@pytest.mark.parametrize("dtype,pdtype", [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
def test_layer_norm(gpu_device, rows, c, dtype, pdtype):
    g = _gen(gpu_device, rows * 31 + c)
    n = lambda *s: torch.randn(*s, generator=g, device=gpu_device)
    x = (n(rows, c) * 2 + 3 * n(rows, 1)).to(dtype).requires_grad_()
    w, b = (1 + 0.3 * n(c)).to(pdtype).requires_grad_(), n(c).to(pdtype).requires_grad_()
    dy = n(rows, c).to(dtype)
    y = tokens.layer_norm(x, w, b, 1e-3)
    got = (y,) + torch.autograd.grad(y, (x, w, b), dy)
    assert [t.dtype for t in got] == [dtype, dtype, pdtype, pdtype]
    u = U if dtype == torch.bfloat16 else F
    up = U if pdtype == torch.bfloat16 else F
    want, tol = _norm_case(gpu_device, x, w, b, 1e-3, dy, u)
    for name, a, r, t in zip(("y", "dx", "dw", "db"), got, want, tol):
        _within(name, a, r, t + (up * (r.abs() + t) if name in ("dw", "db") else u * t))
    with torch.no_grad():
        assert torch.equal(tokens.layer_norm(x, w, b, 1e-3), y)        # the same kernel with and without statistics


def test_layer_norm_without_parameters_and_partial_gradients(gpu_device):
    g = _gen(gpu_device, 5)
    x = torch.randn(37, 96, generator=g, device=gpu_device)
    w, b = torch.randn(96, generator=g, device=gpu_device), torch.randn(96, generator=g, device=gpu_device)
    dy = torch.randn(37, 96, generator=g, device=gpu_device)
    for use_w, use_b in [(False, False), (True, False), (False, True), (True, True)]:
        ww, bb = (w if use_w else None), (b if use_b else None)
        want, tol = _norm_case(gpu_device, x, ww, bb, 1e-5, dy, F)
        _within("y", tokens.layer_norm(x, ww, bb), want[0], tol[0])
        for wants in [(True, False, False), (False, True, False), (False, False, True), (True, True, True)]:
            leaves = [t if t is None else t.clone().requires_grad_(q) for t, q in zip((x, ww, bb), wants)]
            asked = [k for k, t in enumerate(leaves) if t is not None and t.requires_grad]
            if not asked:
                continue
            y = tokens.layer_norm(*leaves)
            for k, got in zip(asked, torch.autograd.grad(y, [leaves[k] for k in asked], dy)):
                _within("xwb"[k], got, want[k + 1], tol[k + 1] * 1.01)


def test_layer_norm_views_and_shapes(gpu_device):
    g = _gen(gpu_device, 6)
    wide = torch.randn(2, 5, 6, 96, generator=g, device=gpu_device).bfloat16()
    w, b = torch.randn(40, generator=g, device=gpu_device), torch.randn(40, generator=g, device=gpu_device)
    for view in (wide[..., 16:56], wide[..., 3:43], wide[:, :, :, 40:80]):
        y = tokens.layer_norm(view, w, b)
        assert y.shape == view.shape and y.is_contiguous()
        # (slices that start off a 16-byte boundary are added up in another order: held to the bound, not to the bits)
        want, tol = _norm_case(gpu_device, view.reshape(-1, 40), w, b, 1e-5, view.reshape(-1, 40), U)
        _within("y", y.view(-1, 40), want[0], tol[0] * (1 + U))
    assert tokens.layer_norm(wide[:0, ..., :40], w, b).shape == (0, 5, 6, 40)
    one = torch.randn(40, generator=g, device=gpu_device)
    assert tokens.layer_norm(one, w, b).shape == (40,)
    e = torch.empty(0, 40, device=gpu_device, requires_grad=True)
    wg = w.clone().requires_grad_()
    de, dw = torch.autograd.grad(tokens.layer_norm(e, wg, b), (e, wg), torch.empty(0, 40, device=gpu_device))
    assert de.shape == (0, 40) and torch.equal(dw, torch.zeros_like(dw))


def test_layer_norm_refuses(gpu_device):
    x = torch.zeros(4, 6, 8, device=gpu_device)
    w = torch.ones(8, device=gpu_device)
    for bad in (x.permute(1, 0, 2), x.transpose(1, 2)[..., ::1].transpose(0, 1), x[..., ::2], x.half(), x.expand(3, 4, 6, 8)):
        with pytest.raises(L.YamdError):
            tokens.layer_norm(bad)
    for kw in (dict(weight=w[:7]), dict(weight=w.half()), dict(weight=w, bias=w.bfloat16()), dict(weight=w.cpu()),
               dict(weight=torch.ones(16, device=gpu_device)[::2]), dict(eps=-1.0)):
        with pytest.raises(L.YamdError):
            tokens.layer_norm(x, **kw)
    with pytest.raises(L.YamdError):
        tokens.layer_norm(torch.zeros(2, 16385, device=gpu_device))
    y = tokens.layer_norm(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(y.sum(), [y.grad_fn.next_functions[0][0].variable], create_graph=True)


def test_layer_norm_nan_and_constant_rows(gpu_device):
    x = torch.randn(6, 64, device=gpu_device).bfloat16()
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    x[3] = 2.5
    y = tokens.layer_norm(x, eps=1e-5)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    assert torch.equal(y[3], torch.zeros_like(y[3]))
    keep = torch.tensor([0, 4, 5], device=gpu_device)
    assert torch.equal(y[keep], tokens.layer_norm(x[keep], eps=1e-5))


def test_layer_norm_squares_that_overflow(gpu_device):
    """A variance beyond float32 is infinite, and the row then comes out as its bias."""
    x = torch.zeros(3, 96, device=gpu_device)
    x[1, 5], x[2, 7] = 1e25, -3e15
    b = torch.linspace(-1, 1, 96, device=gpu_device)
    y = tokens.layer_norm(x, None, b)
    assert torch.equal(y[0], b) and torch.equal(y[1], b)
    want, tol = _norm_case(gpu_device, x[2:], None, b, 1e-5, torch.zeros_like(x[2:]), F)
    _within("y", y[2:], want[0], tol[0])


def test_layer_norm_without_rows(gpu_device):
    for params in (False, True):
        x = torch.zeros(0, 40, device=gpu_device, dtype=torch.bfloat16, requires_grad=True)
        w = torch.ones(40, device=gpu_device, requires_grad=True) if params else None
        y = tokens.layer_norm(x, w, w)
        assert torch.autograd.grad(y, x, torch.zeros_like(y), retain_graph=True)[0].shape == (0, 40)
        if params:
            assert torch.equal(torch.autograd.grad(y, w, torch.zeros_like(y))[0], torch.zeros(40, device=gpu_device))


def test_layer_norm_rows_beyond_32_bits(gpu_device):
    """Rows 2^30 elements apart: the third starts beyond 2^31."""
    big = torch.empty(2 * (1 << 30) + 64, dtype=torch.bfloat16, device=gpu_device)
    x = torch.as_strided(big, (3, 64), (1 << 30, 1))
    x.copy_(torch.randn(3, 64, device=gpu_device))
    assert torch.equal(tokens.layer_norm(x), tokens.layer_norm(x.contiguous()))


# ---- attention ------------------------------------------------------------------------------------------------------------
def _index(h, w, dev):
    t = torch.arange(h * w, device=dev)
    a = t + t // w * (w - 1)
    return a[:, None] - a[None, :] + a[-1]


def _reference(q, k, v, scale, mask=None, bias=None, hw=None, do=None):
    """Results in 64 bits and their bounds: dicts over o, dq, dk, dv (and dbias by distance)."""
    d = q.shape[-1]
    group = q.shape[2] // k.shape[2]
    Q, K, V = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    if mask is not None:                       # what masked places hold does not matter
        K, V = (torch.where(mask[:, None, :, None], t, 0.0) for t in (K, V))
    K, V = (t.repeat_interleave(group, 1) for t in (K, V))
    s = scale * Q @ K.transpose(2, 3)
    size = scale * Q.abs() @ K.abs().transpose(2, 3)
    if bias is not None:
        idx = _index(*hw, q.device)
        full = bias.detach().double()[:, idx]
        full = torch.where(full < -1e5, -math.inf, full)
        s = s + full
        size = size + torch.where(full == -math.inf, 0.0, full.abs())
    if mask is not None:
        s = s.masked_fill(~mask[:, None, None, :], -math.inf)
    m = s.amax(3, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(s - m)
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    # relative error of a probability from float32: of the exponent (scores are sums of d terms, then a few operations on
    # numbers as large as scores and statistics), of the exponential and of the sums
    rho = 2 * F * ((d + 16) * size.max().item() + 8 * m.abs().max().item() + 4 * math.log(s.shape[3] + 1) + 64)
    sat = 1e-12
    o, a = p @ V, p @ V.abs()
    t_o = U * o.abs() + (1 + U) * ((U + rho) * a) + sat
    back = lambda t: t.transpose(1, 2)
    want, tol = {"o": back(o)}, {"o": back(t_o)}
    if do is None:
        return want, tol
    G = torch.where(total > 0, do.detach().double().transpose(1, 2), 0.0)
    dp = G @ V.transpose(2, 3)
    D = (G * o).sum(3, keepdim=True)
    ds = p * (dp - D)
    # D takes over the error of o: 2^-16 of the probabilities with a bias or few keys; beyond, they are rounded
    near = p * (G.abs() @ V.abs().transpose(2, 3) + (G.abs() * a).sum(3, keepdim=True))     # what dS is a difference of
    e_D = (G.abs() * ((U + rho) * a if bias is None and s.shape[3] > 256 else (U * U + rho) * a)).sum(3, keepdim=True)
    e_ds = p * e_D + (rho + 2 * (d + 8) * F) * near
    t_ds = U * (ds.abs() + e_ds) + e_ds
    fold = lambda t: t.reshape(t.shape[0], k.shape[2], group, *t.shape[2:]).sum(2)
    dq, dk, dv = scale * ds @ K, scale * fold(ds.transpose(2, 3) @ Q), fold(p.transpose(2, 3) @ G)
    t_dq = scale * t_ds @ K.abs()
    t_dk = scale * fold(t_ds.transpose(2, 3) @ Q.abs())
    t_dv = fold(((U + rho) * p).transpose(2, 3) @ G.abs())
    for n, x, t in (("dq", dq, t_dq), ("dk", dk, t_dk), ("dv", dv, t_dv)):
        want[n], tol[n] = back(x), back(U * (x.abs() + t) + 1.01 * t + sat)
    if bias is not None:
        flat = idx.reshape(-1)
        sums = lambda t: torch.zeros(t.shape[1], bias.shape[1], dtype=torch.float64, device=q.device).index_add_(
            1, flat, t.sum(0).reshape(t.shape[1], -1))
        want["dbias"] = sums(ds)
        tol["dbias"] = sums(e_ds) + 4096 * F * sums(ds.abs()) + sat    # (4096: the longest chain of additions)
    return want, tol


def _inputs(dev, seed, b, lq, lk, heads, kv, d):
    g = _gen(dev, seed)
    n = lambda *s: torch.randn(*s, generator=g, device=dev).bfloat16()
    return [(1.5 * n(b, lq, heads, d).float()).bfloat16().requires_grad_(), n(b, lk, kv, d).requires_grad_(), n(b, lk, kv, d).requires_grad_()], \
        n(b, lq, heads, d), g


def _check(dev, q, k, v, do, scale=None, mask=None, table=None, pos=None):
    scale_ = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    bias = None if pos is None else tokens.relative_bias(table, pos)
    kw = {} if pos is None else dict(bias=bias, position=pos)
    o = tokens.attention(q, k, v, scale, mask, **kw)
    leaves = [q, k, v] + ([bias] if pos is not None else [])
    grads = torch.autograd.grad(o, leaves, do, retain_graph=True)
    want, tol = _reference(q, k, v, scale_, mask, bias, None if pos is None else (pos.h, pos.w), do)
    for n, got in zip(("dq", "dk", "dv", "dbias"), grads):
        _within(n, got, want[n], tol[n])
    _within("o", o, want["o"], tol["o"])
    again = torch.autograd.grad(o, leaves, do)
    for n, x, y in zip(("dq", "dk", "dv", "dbias"), grads, again):
        assert torch.equal(x, y), f"{n}: two runs differ"
    with torch.no_grad():
        served = tokens.attention(q, k, v, scale, mask, **kw)
    _within("o (served)", served, want["o"], tol["o"])
    return want, tol, grads


@pytest.mark.parametrize("b,lq,lk,heads,kv,d", [
    (1, 1, 1, 1, 1, 8), (1, 1, 64, 2, 1, 16), (2, 31, 33, 2, 2, 24), (1, 32, 64, 1, 1, 64), (2, 65, 63, 4, 2, 40), (1, 127, 129, 2, 2, 128),
    (1, 129, 128, 3, 1, 96), (3, 128, 200, 2, 1, 72), (2, 300, 1000, 4, 4, 32), (1, 257, 511, 8, 2, 104), (1, 700, 20, 4, 2, 64),
    (1, 5, 3000, 6, 3, 56), (8, 1, 700, 8, 2, 64), (1, 64, 2100, 8, 8, 120), (2, 640, 640, 2, 2, 88), (1, 40, 4000, 16, 1, 128)])
def test_attention(gpu_device, b, lq, lk, heads, kv, d):
    (q, k, v), do, _ = _inputs(gpu_device, lq + lk, b, lq, lk, heads, kv, d)
    _check(gpu_device, q, k, v, do)


@pytest.mark.parametrize("kind", ["random", "prefix", "one", "empty", "sparse"])
@pytest.mark.parametrize("lq,lk,heads,kv,d", [(70, 130, 4, 2, 64), (1, 2500, 8, 2, 32), (200, 333, 2, 2, 128), (33, 64, 2, 1, 40)])
def test_attention_masks_with_garbage_behind(gpu_device, kind, lq, lk, heads, kv, d):
    (q, k, v), do, g = _inputs(gpu_device, lq * lk, 3, lq, lk, heads, kv, d)
    mask = torch.rand(3, lk, generator=g, device=gpu_device) < 0.6
    if kind == "prefix":
        mask = torch.arange(lk, device=gpu_device)[None] < torch.tensor([[lk], [lk // 2], [1]], device=gpu_device)
    elif kind == "one":
        mask = torch.arange(lk, device=gpu_device)[None] == torch.tensor([[lk - 1], [0], [lk // 2]], device=gpu_device)
    elif kind == "empty":
        mask[1] = False
    elif kind == "sparse":
        mask = torch.rand(3, lk, generator=g, device=gpu_device) < 0.02
    clean, _, _ = _check(gpu_device, q, k, v, do, mask=mask)
    # NaN and infinities in masked places change nothing, not even a bit
    with torch.no_grad():
        dirty = [t.clone() for t in (k, v)]
        dirty[0][~mask] = math.nan
        dirty[1][~mask] = math.inf
    ref = torch.autograd.grad(tokens.attention(q, k, v, None, mask), (q, k, v), do)
    kd, vd = (t.requires_grad_() for t in dirty)
    o = tokens.attention(q, kd, vd, None, mask)
    assert torch.equal(o, tokens.attention(q, k, v, None, mask))
    for x, y in zip(torch.autograd.grad(o, (q, kd, vd), do), ref):
        assert torch.equal(x, y)
    assert not ref[1][~mask].any() and not ref[2][~mask].any()
    if kind == "empty":
        assert not o[1].any() and not ref[0][1].any()


def test_attention_empty_rows_ignore_queries_and_gradients(gpu_device):
    (q, k, v), do, _ = _inputs(gpu_device, 11, 2, 40, 90, 2, 2, 64)
    mask = torch.ones(2, 90, dtype=torch.bool, device=gpu_device)
    mask[1] = False
    with torch.no_grad():
        q[1], do[1] = math.nan, math.nan
    o = tokens.attention(q, k, v, None, mask)
    grads = torch.autograd.grad(o, (q, k, v), do)
    assert not o[1].any() and all(torch.isfinite(t).all() for t in grads) and not any(t[1].any() for t in grads)


@pytest.mark.parametrize("b,h,w,heads,d,buckets", [(1, 1, 1, 1, 32, 8), (2, 1, 77, 2, 64, 32), (1, 1, 400, 2, 40, 8), (2, 5, 7, 2, 16, 8),
                                                   (2, 20, 20, 2, 32, 16), (1, 11, 13, 3, 64, 8), (1, 3, 100, 2, 96, 8), (1, 40, 12, 2, 128, 16),
                                                   (1, 19, 19, 2, 128, 8), (3, 2, 150, 1, 64, 8), (1, 300, 2, 1, 64, 8), (1, 2, 420, 1, 32, 8),
                                                   (1, 130, 1, 2, 64, 8)])
@pytest.mark.parametrize("tdtype", [torch.float32, torch.bfloat16])
def test_attention_with_learned_bias(gpu_device, b, h, w, heads, d, buckets, tdtype):
    (q, k, v), do, g = _inputs(gpu_device, h * w + d, b, h * w, h * w, heads, heads, d)
    pos = tokens.RelativePosition(h, w, buckets, 64, gpu_device)
    table = torch.randn(pos.rows, heads, generator=g, device=gpu_device).to(tdtype).requires_grad_()
    bias = tokens.relative_bias(table, pos)
    assert torch.equal(bias, table.detach().float()[pos.bucket_of.long()].t())
    want, tol, grads = _check(gpu_device, q, k, v, do, table=table, pos=pos)
    # the table's gradient: sums over each bucket's distances
    dt, = torch.autograd.grad(bias, (table,), grads[3])
    one = torch.zeros(pos.rows, pos.distances, dtype=torch.float64, device=gpu_device)
    one[pos.bucket_of.long(), torch.arange(pos.distances, device=gpu_device)] = 1
    dwant, dtol = one @ want["dbias"].t(), one @ (tol["dbias"] + 64 * F * want["dbias"].abs()).t()
    assert dt.dtype == tdtype
    _within("dtable", dt, dwant, dtol + (U if tdtype == torch.bfloat16 else F) * (dwant.abs() + dtol))


@pytest.mark.parametrize("lq,lk,heads,d", [(1600, 1600, 20, 32), (130, 1500, 129, 64), (1664, 70, 20, 128), (100, 2000, 257, 96)])
def test_attention_cuts_the_last_items_only(gpu_device, lq, lk, heads, d):
    """A little more than 256 tiles of rows: 256 walk their keys (queries) whole, the others in parts."""
    (q, k, v), do, g = _inputs(gpu_device, lq + lk, 1, lq, lk, heads, heads, d)
    mask = torch.rand(1, lk, generator=g, device=gpu_device) < 0.9
    mask[0, lk // 3:lk // 2] = False
    _check(gpu_device, q, k, v, do, mask=mask)


@pytest.mark.parametrize("b,h,w,heads,d", [(1, 40, 40, 20, 32), (2, 1, 1000, 17, 64), (3, 25, 30, 15, 128)])
def test_biased_attention_cuts_the_last_items_only(gpu_device, b, h, w, heads, d):
    (q, k, v), do, g = _inputs(gpu_device, h * w + d, b, h * w, h * w, heads, heads, d)
    pos = tokens.RelativePosition(h, w, 16, 64, gpu_device)
    table = torch.randn(pos.rows, heads, generator=g, device=gpu_device).requires_grad_()
    _check(gpu_device, q, k, v, do, table=table, pos=pos)


def test_bias_that_masks(gpu_device):
    """-inf, the lowest value and usual large negative values in the bias mask; rows that have nothing else get zeros."""
    h, w, heads = 4, 40, 2
    (q, k, v), do, g = _inputs(gpu_device, 3, 1, h * w, h * w, heads, heads, 64)
    pos = tokens.RelativePosition(h, w, 8, 16, gpu_device)
    for low in (-math.inf, torch.finfo(torch.float32).min, -1e9, -1e20):
        table = torch.randn(pos.rows, heads, generator=g, device=gpu_device)
        table[::2, 0] = low                    # head 0: every other bucket
        table[:, 1] = low                      # head 1: everything
        o = tokens.attention(q, k, v, bias=tokens.relative_bias(table, pos), position=pos)
        assert torch.isfinite(o).all() and not o[:, :, 1].any()
        t = table.clone().requires_grad_()
        b = tokens.relative_bias(t, pos)
        got = torch.autograd.grad(tokens.attention(q, k, v, bias=b, position=pos), (q, k, v, b), do)
        want, tol = _reference(q, k, v, 0.125, None, b, (h, w), do)
        for n, x in zip(("dq", "dk", "dv", "dbias"), got):
            _within(n, x, want[n], tol[n])
        assert not got[0][:, :, 1].any() and not got[3][1].any()


def test_bias_with_mask_and_without_gradient(gpu_device):
    h, w, heads = 9, 12, 2
    (q, k, v), do, g = _inputs(gpu_device, 4, 2, h * w, h * w, heads, heads, 64)
    pos = tokens.RelativePosition(h, w, 8, 16, gpu_device)
    table = torch.randn(pos.rows, heads, generator=g, device=gpu_device).requires_grad_()
    mask = torch.rand(2, h * w, generator=g, device=gpu_device) < 0.5
    mask[1, :] = False
    mask[1, 5] = True
    _check(gpu_device, q, k, v, do, mask=mask, table=table, pos=pos)
    frozen = tokens.relative_bias(table.detach(), pos)
    got = torch.autograd.grad(tokens.attention(q, k, v, None, mask, frozen, pos), (q, k, v), do)
    want, tol = _reference(q, k, v, 0.125, mask, frozen, (h, w), do)
    loose = _reference(q, k, v, 0.125, mask, None, None, do)[1]        # (without its gradient o reaches D rounded)
    for n, x in zip(("dq", "dk", "dv"), got):
        _within(n, x, want[n], tol[n] + loose[n])


def test_gradients_against_differences(gpu_device):
    """Directional differences in 64 bits of the reference's own forward, against the kernels' gradients."""
    h, w = 4, 6
    (q, k, v), do, g = _inputs(gpu_device, 8, 1, h * w, h * w, 2, 2, 16)
    pos = tokens.RelativePosition(h, w, 8, 16, gpu_device)
    table = torch.randn(pos.rows, 2, generator=g, device=gpu_device).requires_grad_()
    o = tokens.attention(q, k, v, bias=tokens.relative_bias(table, pos), position=pos)
    grads = torch.autograd.grad(o, (q, k, v, table), do)
    idx = _index(h, w, gpu_device)

    def loss(q_, k_, v_, t_):
        s = 0.25 * torch.einsum("bihd,bjhd->bhij", q_, k_) + t_[pos.bucket_of.long()].t()[:, idx]
        return (torch.einsum("bhij,bjhd->bihd", torch.softmax(s, 3), v_) * do.double()).sum()

    at = [t.detach().double() for t in (q, k, v, table)]
    for n in range(4):
        for _ in range(3):
            way = torch.randn(at[n].shape, generator=g, device=gpu_device, dtype=torch.float64)
            e = 1e-6
            up, down = ([t + e * s * way if i == n else t for i, t in enumerate(at)] for s in (1, -1))
            diff = (loss(*up) - loss(*down)) / (2 * e)
            got = (grads[n].double() * way).sum()
            # every element of a gradient is off by about three roundings of its own size at most in norm
            assert abs(got - diff) <= 3 * U * grads[n].double().norm() * way.norm() + 1e-6


def test_attention_layouts(gpu_device):
    """Slices of one buffer, heads before tokens, padded rows: the same bits as contiguous tensors; dense gradients."""
    b, n, heads, d = 2, 100, 3, 40
    g = _gen(gpu_device, 2)
    qkv = torch.randn(b, n, 3, heads, d, generator=g, device=gpu_device).bfloat16()
    q, k, v = qkv.unbind(2)
    ref = tokens.attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(tokens.attention(q, k, v), ref)
    turned = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v)]       # (B, heads, N, d) in memory
    assert torch.equal(tokens.attention(*turned), ref)
    wide = torch.full((b, n, heads, 64), math.nan, dtype=torch.bfloat16, device=gpu_device)
    padded = wide[..., 8:48]
    padded.copy_(k)
    assert torch.equal(tokens.attention(q, padded, v), ref)
    leaf = qkv.clone().requires_grad_()
    do = torch.randn(b, n, heads, d, generator=g, device=gpu_device).bfloat16()
    got, = torch.autograd.grad(tokens.attention(*leaf.unbind(2)), (leaf,), do)
    parts = [t.contiguous().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(tokens.attention(*parts), parts, do)
    assert torch.equal(got, torch.stack(want, 2))
    # a gradient that is broadcast (its strides are zero) and one in another layout
    o = tokens.attention(*parts)
    assert torch.equal(torch.autograd.grad(o.float().sum(), parts, retain_graph=True)[0], torch.autograd.grad(o, parts, torch.ones_like(o), retain_graph=True)[0])
    do_t = do.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(torch.autograd.grad(o, parts, do_t)[2], want[2])


def test_attention_gradient_from_a_longer_vector(gpu_device):
    """The gradient of a result that was joined to something else starts anywhere."""
    leaves, do, _ = _inputs(gpu_device, 77, 1, 33, 65, 2, 1, 32)
    want = torch.autograd.grad(tokens.attention(*leaves), leaves, do)
    flat = torch.cat([torch.zeros(3, device=gpu_device, dtype=torch.bfloat16), do.flatten()])
    joined = flat[3:].view(do.shape)
    assert joined.data_ptr() % 16 and joined.is_contiguous()
    got = torch.autograd.grad(tokens.attention(*leaves), leaves, joined)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("lq,lk,d", [(300, 2, 64), (100, 3, 32), (64, 20, 128), (33, 700, 96)])
def test_gradients_of_peaked_rows(gpu_device, lq, lk, d):
    """Rows whose probability lies on few keys, where dS is a small difference: relative to all of dq and dk the gradients stay
    within twice the root mean square of two roundings to bf16 (of dS and of the result; the fourth row adds that of P)."""
    (q, k, v), do, _ = _inputs(gpu_device, lq + lk, 2, lq, lk, 2, 2, d)
    scale = 1 / math.sqrt(d) if lk < 100 else 0.6
    _check(gpu_device, q, k, v, do, scale=scale)
    want, _ = _reference(q, k, v, scale, do=do)
    grads = torch.autograd.grad(tokens.attention(q, k, v, scale), (q, k), do)
    for n, g in zip(("dq", "dk"), grads):
        off = ((g.double() - want[n]).norm() / want[n].norm()).item()
        assert off <= 2 * math.sqrt(2) * U / math.sqrt(3), (n, off)


def test_attention_broadcast_batch_is_refused(gpu_device):
    q = torch.randn(2, 8, 1, 16, device=gpu_device).bfloat16()
    k = torch.randn(1, 8, 1, 16, device=gpu_device).bfloat16().expand(2, 8, 1, 16)
    with pytest.raises(L.YamdError):
        tokens.attention(q, k, k)


def test_attention_refuses(gpu_device):
    q = torch.zeros(2, 16, 4, 32, device=gpu_device, dtype=torch.bfloat16)
    k = torch.zeros(2, 20, 2, 32, device=gpu_device, dtype=torch.bfloat16)
    m = torch.ones(2, 20, dtype=torch.bool, device=gpu_device)
    tokens.attention(q, k, k, 0.1, m)
    pos = tokens.RelativePosition(4, 4, 8, 16, gpu_device)
    bias = torch.zeros(4, pos.distances, device=gpu_device)
    same = q[:, :, :2]
    bad = [dict(q=q.float()), dict(q=q.half()), dict(k=k[:, :, :1].expand(2, 20, 3, 32)), dict(v=k[:, :19]), dict(q=q[..., :12]),
           dict(q=q[..., 4:28]), dict(k=k.cpu()), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(mask=m[:, :19]),
           dict(mask=m.float()), dict(mask=m.t().contiguous().t()), dict(mask=m[:1].expand(2, 20)), dict(q=q[0]),
           dict(bias=bias, position=pos), dict(k=q, v=q, bias=bias[:3], position=pos), dict(k=q, v=q, bias=bias.double(), position=pos),
           dict(k=same, v=same, bias=bias[:, :-1], position=pos)]
    for kw in bad:
        a = dict(q=q, k=k, v=kw.get("k", k), scale=None, mask=None, bias=None, position=None)
        a.update(kw)
        with pytest.raises(L.YamdError):
            tokens.attention(a["q"], a["k"], a["v"], a["scale"], a["mask"], a["bias"], a["position"])
    with pytest.raises(L.YamdError):
        tokens.relative_bias(torch.zeros(pos.rows - 1, 4, device=gpu_device), pos)
    with pytest.raises(L.YamdError):
        tokens.relative_bias(torch.zeros(pos.rows, 4, device=gpu_device).half(), pos)


def test_attention_nothing(gpu_device):
    mk = lambda *s: torch.randn(*s, device=gpu_device).bfloat16().requires_grad_()
    for lq, lk, b in [(0, 5, 2), (5, 0, 2), (0, 0, 1), (4, 4, 0)]:
        q, k, v = mk(b, lq, 2, 16), mk(b, lk, 2, 16), mk(b, lk, 2, 16)
        o = tokens.attention(q, k, v)
        assert o.shape == q.shape and not o.any()
        for t, g in zip((q, k, v), torch.autograd.grad(o, (q, k, v), torch.ones_like(o))):
            assert g.shape == t.shape and not g.any()


def test_attention_keys_beyond_32_bits(gpu_device):
    """Keys 2^23 elements apart: from the 256th on they lie beyond 2^31 elements."""
    n, st = 300, 1 << 23
    big = torch.empty((n - 1) * st + 64, dtype=torch.bfloat16, device=gpu_device)
    k = torch.as_strided(big, (1, n, 1, 64), (8, st, 8, 1))
    g = _gen(gpu_device, 1)
    k.copy_(torch.randn(1, n, 1, 64, generator=g, device=gpu_device))
    q, v = (torch.randn(1, n, 1, 64, generator=g, device=gpu_device).bfloat16() for _ in range(2))
    assert torch.equal(tokens.attention(q, k, v), tokens.attention(q, k.contiguous(), v))
    assert torch.equal(tokens.attention(k, v, q), tokens.attention(k.contiguous(), v, q))
    ql, kl, vl = (t.detach().clone().requires_grad_() if t is not k else k.detach().requires_grad_() for t in (q, k, v))
    do = torch.randn(1, n, 1, 64, generator=g, device=gpu_device).bfloat16()
    got = torch.autograd.grad(tokens.attention(ql, kl, vl), (ql, kl, vl), do)
    dense = [t.detach().contiguous().requires_grad_() for t in (ql, kl, vl)]
    for x, y in zip(got, torch.autograd.grad(tokens.attention(*dense), dense, do)):
        assert torch.equal(x, y)


def test_extreme_scores(gpu_device):
    """Scores up to +-1e4: one key takes all; large equal scores; an infinite query gives NaN in its own row only."""
    d = 64
    g = _gen(gpu_device, 9)
    q = torch.randn(1, 70, 1, d, generator=g, device=gpu_device).bfloat16()
    k, v = (torch.randn(1, 90, 1, d, generator=g, device=gpu_device).bfloat16() for _ in range(2))
    q200, k200 = q * 200, k * 200              # (rounded to bf16: the operator's inputs)
    o = tokens.attention(q200, k200, v, 1 / 8)
    s = q200.double()[0, :, 0] @ k200.double()[0, :, 0].t() / 8
    top = s.topk(2, 1)
    sure = (top.values[:, 0] - top.values[:, 1]) > 30          # the others together weigh below 90 exp(-30)
    assert sure.sum() > 50
    # the weight of that key is 1 but for the rounding of its exponent, one float32 step of the score (in units of log 2: times
    # 1.4427, and ln 2 turns it back), which reaches the result because the weight is then rounded to bf16 and its sum is not
    picked = v[0, top.indices[:, 0], 0].double()
    tol = (2 * U + U * U + 2 * F * top.values[:, :1].abs()) * picked.abs()
    _within("o", o[0, :, 0][sure], picked[sure], tol[sure] + 1e-9)
    q2 = q.clone()
    q2[0, 3] = math.inf
    o2 = tokens.attention(q2, k, v)
    assert torch.isnan(o2[0, 3]).all()
    keep = torch.arange(70, device=gpu_device) != 3
    assert torch.equal(o2[0, keep], tokens.attention(q, k, v)[0, keep])


def test_output_slices_are_all_that_is_written(gpu_device):
    """Through the C ABI: o as a channel slice of a wider buffer; its other channels, rows and images stay as they were."""
    b, n, heads, d = 2, 70, 2, 32
    g = _gen(gpu_device, 4)
    q, k, v = (torch.randn(b, n, heads, d, generator=g, device=gpu_device).bfloat16() for _ in range(3))
    wide = torch.full((b + 1, n + 3, 3 * heads * d), 7.0, dtype=torch.bfloat16, device=gpu_device)
    out = wide[:b, :n, heads * d:2 * heads * d].unflatten(2, (heads, d))
    lse = torch.full((b * heads * n + 64,), 7.0, device=gpu_device)
    tk = lambda t: L.Tokens(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))
    desc = L.AttentionDesc(b, heads, heads, d, n, n, 0, 0, 0.2)
    r = ctypes.byref
    L.check(L.LIB.yamd_attention(r(desc), r(tk(q)), r(tk(k)), r(tk(v)), None, 0, None, r(tk(out)), None, lse.data_ptr(), None, 0,
                                 L.current_stream()))
    assert torch.equal(out, tokens.attention(q, k, v, 0.2))
    out.fill_(7.0)
    assert (wide == 7.0).all() and (lse[b * heads * n:] == 7.0).all()
    s = 0.2 * torch.einsum("bihd,bjhd->bhij", q.double(), k.double())
    assert ((lse[:b * heads * n].double() - torch.logsumexp(s, 3).reshape(-1)).abs() < 1e-5).all()


# ---- streams, graphs, programs --------------------------------------------------------------------------------------------
def _block(x, w, b, wqkv, wo, table, pos, heads):
    """norm -> q, k, v -> attention with position bias -> projection -> residual"""
    n, c = x.shape[1], x.shape[2]
    y = tokens.layer_norm(x, w, b)
    q, k, v = (y @ wqkv).view(x.shape[0], n, 3, heads, c // heads).unbind(2)
    o = tokens.attention(q, k, v, bias=tokens.relative_bias(table, pos), position=pos)
    return x + o.reshape(x.shape[0], n, c) @ wo


def _block_inputs(dev, seed, b=2, h=8, w=12, c=64, heads=2):
    g = _gen(dev, seed)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)
    pos = tokens.RelativePosition(h, w, 8, 16, dev)
    leaves = [n(b, h * w, c).bfloat16(), 1 + 0.1 * n(c), 0.1 * n(c), (n(c, 3 * c) / 8).bfloat16(), (n(c, c) / 8).bfloat16(), n(pos.rows, heads)]
    return [t.requires_grad_() for t in leaves], pos, n(b, h * w, c).bfloat16()


def test_block_forward_and_backward(gpu_device):
    """A run of the operators together against the same block in 64 bits."""
    leaves, pos, dy = _block_inputs(gpu_device, 21)
    y = _block(*leaves, pos, 2)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    x, w, b, wqkv, wo, table = ref
    n, c = x.shape[1], x.shape[2]
    z = torch.nn.functional.layer_norm(x, (c,), w, b, 1e-5)
    q, k, v = (z @ wqkv).view(2, n, 3, 2, c // 2).unbind(2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(c // 2) + table[pos.bucket_of.long()].t()[:, _index(pos.h, pos.w, gpu_device)]
    o = torch.einsum("bhij,bjhd->bihd", torch.softmax(s, 3), v).reshape(2, n, c)
    yr = x + o @ wo
    want = torch.autograd.grad(yr, ref, dy.double())
    # seven tensors are rounded to bf16 on the way forward and as many on the way back; each rounding moves a tensor by at
    # most U of its norm and the maps between them have gains of order one
    for got, r in zip((y,) + grads, (yr,) + want):
        assert (got.double() - r).norm() <= 14 * U * r.norm()


def test_two_streams_at_once(gpu_device):
    cases = [_block_inputs(gpu_device, 30 + i, h=8 + 4 * i) for i in range(2)]
    want = []
    for leaves, pos, dy in cases:
        y = _block(*leaves, pos, 2)
        want.append((y, torch.autograd.grad(y, leaves, dy)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu_device) for _ in range(2)]
    for _ in range(5):
        got = []
        for st, (leaves, pos, dy) in zip(streams, cases):
            with torch.cuda.stream(st):
                y = _block(*leaves, pos, 2)
                got.append((y, torch.autograd.grad(y, leaves, dy)))
        torch.cuda.synchronize()
        for (y, g), (yw, gw) in zip(got, want):
            assert torch.equal(y, yw) and all(torch.equal(a, b) for a, b in zip(g, gw))


def _token_step(leaves, pos, dy):
    """Norm, bias and attention (split and joined for the few queries) with all their gradients; no library call in it."""
    x, w, b, table = leaves
    y = tokens.layer_norm(x, w, b)
    t = y.unflatten(2, (2, 32))
    o = tokens.attention(t, t, t, bias=tokens.relative_bias(table, pos), position=pos)
    few = tokens.attention(t[:, :3].contiguous(), t, t)
    return [o, few] + list(torch.autograd.grad(o, leaves, dy, retain_graph=False))


def test_captured_graphs_replay(gpu_device):
    """Forward and backward captured into two graphs on one stream, replayed in turns with the program's own eager calls
    between: every replay equals the eager result on the inputs of that moment."""
    pos = tokens.RelativePosition(8, 100, 8, 16, gpu_device)
    g = _gen(gpu_device, 40)
    n = lambda *s: torch.randn(*s, generator=g, device=gpu_device)
    sets = []
    side = torch.cuda.Stream(gpu_device)
    for _ in range(2):
        leaves = [n(1, 800, 64).bfloat16().requires_grad_(), n(64).requires_grad_(), n(64).requires_grad_(), n(pos.rows, 2).requires_grad_()]
        dy = n(1, 800, 2, 32).bfloat16()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _token_step(leaves, pos, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _token_step(leaves, pos, dy)
        sets.append((leaves, dy, graph, out))
    for turn in range(4):
        for leaves, dy, graph, out in sets:
            with torch.no_grad():
                for t in leaves + [dy]:
                    t.copy_(torch.randn(t.shape, generator=g, device=gpu_device))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            for a, b in zip(got, _token_step(leaves, pos, dy)):
                assert torch.equal(a, b), f"turn {turn}"


def _program(h, w, c, heads, sd, pos):
    """A program whose 1x1 convs feed a token block: conv -> norm -> qkv -> attention (position bias) -> conv + residual, and
    the same map's queries over a coarser map without bias."""
    p = Program(h, w)
    x = p.conv("stem", p.image16(), sd["stem"], None, 2, L.ACT_SILU)
    x = p.conv("down", x, sd["down"], None, 2, L.ACT_SILU)
    n = p.layer_norm("norm", x, sd["nw"], sd["nb"], 1e-5)
    qkv = p.conv("qkv", n, sd["qkv"], None, 1, L.ACT_NONE)
    a = p.attention("self", qkv.slice(0, c), qkv.slice(c, c), qkv.slice(2 * c, c), heads, table=sd["table"], position=pos)
    y = p.conv("out", a, sd["out"], None, 1, L.ACT_NONE, residual=x)
    coarse = p.maxpool2(y)
    kv = p.conv("kv", coarse, sd["kv"], None, 1, L.ACT_NONE)
    z = p.attention("cross", qkv.slice(0, c), kv.slice(0, c // 2), kv.slice(c // 2, c // 2), heads, kv_heads=heads // 2)
    p.outputs = {"x": x, "n": n, "qkv": qkv, "a": a, "y": y, "kv": kv, "z": z}
    return p


@pytest.mark.parametrize("size", [64, 96])
def test_program_with_tokens(gpu_device, size):
    c, heads = 64, 4
    hw = size // 4
    g = torch.Generator().manual_seed(size)
    r = lambda *s: torch.randn(*s, generator=g)
    pos = tokens.RelativePosition(hw, hw, 8, 16, gpu_device)
    sd = dict(stem=r(32, 3, 3, 3) / 5, down=r(c, 32, 3, 3) / 16, nw=1 + 0.1 * r(c), nb=0.1 * r(c), qkv=r(3 * c, c, 1, 1) / 8,
              out=r(c, c, 1, 1) / 8, kv=r(c, c, 1, 1) / 8, table=r(pos.rows, heads))
    prog = _program(size, size, c, heads, sd, pos)
    for batch in (2, 1):
        img = torch.rand(batch, 3, size, size, generator=g).to(gpu_device)
        out = {k: v.clone() for k, v in prog.run(img).items()}
        # each token op against the tensors operator on the program's own input, bit for bit
        tok = lambda t, n: t.reshape(batch, -1, n, t.shape[-1] // n)
        assert torch.equal(out["n"], tokens.layer_norm(out["x"], sd["nw"].to(gpu_device), sd["nb"].to(gpu_device), 1e-5))
        q, k, v = (tok(t, heads) for t in out["qkv"].split(c, 3))
        bias = tokens.relative_bias(sd["table"].to(gpu_device), pos)
        assert torch.equal(tok(out["a"], heads), tokens.attention(q, k, v, bias=bias, position=pos))
        k2, v2 = (tok(t, heads // 2) for t in out["kv"].split(c // 2, 3))
        assert torch.equal(tok(out["z"], heads), tokens.attention(q, k2, v2))
        # the plan that C replays and the per-op calls are the same calls
        prog.use_c_plan = False
        per_op = prog.run(img)
        assert all(torch.equal(out[n], per_op[n]) for n in out)
        prog.use_c_plan = True
        timings = []
        prog.run(img, timings=timings)
        assert {"norm", "attn"} <= {t[0] for t in timings}
