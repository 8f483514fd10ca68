"""CPU checks of the token operators (yolo_amd.tokens, engine.Program.layer_norm / .attention): bucket tables, refusals and
workspace sizes of the C ABI (which validates before it touches a GPU), recording into a program."""
import ctypes
import math

import numpy as np
import pytest
import torch

from yolo_amd import lib as L
from yolo_amd import tokens
from yolo_amd.engine import Program

LIB = L.LIB
FAKE = 4096          # an aligned address that no call below reads: every one is refused first


@pytest.mark.parametrize("buckets,far", [(4, 2), (8, 16), (16, 20), (32, 128), (32, 1000)])
def test_axis_buckets(buckets, far):
    n = 3 * far
    b = tokens.axis_buckets(n, buckets, far)
    assert len(b) == 2 * n - 1
    half, near = buckets // 2, buckets // 4
    for d in range(-(n - 1), n):
        got = b[d + n - 1]
        assert 0 <= got < buckets and (got >= half) == (d > 0)
        m = abs(d)
        if m < near:
            want = m
        else:
            # the largest t with m >= near (far / near)^(t / steps), in whole numbers
            steps = half - near
            want = near + max(t for t in range(steps) if m ** steps * near ** t >= near ** steps * far ** t)
        assert got % half == want, (d, got, want)
    assert b[-1] == buckets - 1 and b[0] == half - 1


def test_axis_buckets_far_distance_costs_nothing():
    """Distances that the axis does not have are not searched."""
    assert tokens.axis_buckets(9, 8, 10 ** 12) == [min(m, 2) for m in range(8, 0, -1)] + [0] + \
        [4 + min(m, 2) for m in range(1, 9)]


def test_axis_buckets_refuses():
    with pytest.raises(L.YamdError):
        tokens.axis_buckets(0, 8, 16)
    for buckets, far in [(6, 16), (0, 16), (8, 2), (-4, 3)]:
        with pytest.raises(L.YamdError):
            tokens.axis_buckets(5, buckets, far)


@pytest.mark.parametrize("h,w", [(1, 1), (1, 37), (5, 7), (20, 20), (3, 1)])
def test_relative_position_lists(h, w):
    p = tokens.RelativePosition(h, w, 8, 16, device="cpu")
    assert p.rows == (8 if h == 1 else 64) and p.distances == (2 * h - 1) * (2 * w - 1)
    of = p.bucket_of.numpy()
    start, order = p.start.numpy(), p.order.numpy()
    assert start[0] == 0 and start[-1] == p.distances and sorted(order.tolist()) == list(range(p.distances))
    for r in range(p.rows):
        assert (of[order[start[r]:start[r + 1]]] == r).all()
    bx, by = tokens.axis_buckets(w, 8, 16), tokens.axis_buckets(h, 8, 16)
    for dy in range(-(h - 1), h):
        for dx in range(-(w - 1), w):
            want = bx[dx + w - 1] + (0 if h == 1 else 8 * by[dy + h - 1])
            assert of[(dy + h - 1) * (2 * w - 1) + dx + w - 1] == want


def test_relative_position_refuses():
    for h, w in [(0, 5), (2, 761), (5000, 5000)]:
        with pytest.raises(L.YamdError):
            tokens.RelativePosition(h, w, 8, 16, device="cpu")
    with pytest.raises(L.YamdError):
        tokens.RelativePosition(4, 4, 1028, 2000, device="cpu")            # 1028^2 rows
    assert tokens.RelativePosition(1, 2000, 8, 16, device="cpu").distances == 3999


def test_no_cpu_path():
    x = torch.zeros(4, 8)
    with pytest.raises(L.YamdError, match="GPU"):
        tokens.layer_norm(x)
    q = torch.zeros(1, 4, 1, 8, dtype=torch.bfloat16)
    with pytest.raises(L.YamdError, match="GPU"):
        tokens.attention(q, q, q)
    p = tokens.RelativePosition(2, 2, 8, 16, device="cpu")
    with pytest.raises(L.YamdError, match="GPU"):
        tokens.relative_bias(torch.zeros(p.rows, 2), p)
    with pytest.raises(L.YamdError, match="together"):
        tokens.attention(q, q, q, position=p)


def _norm(**k):
    a = dict(x=FAKE, xs=64, w=FAKE, b=FAKE, pd=0, eps=1e-5, y=FAKE, ys=64, mean=None, rstd=None, rows=4, c=64, dt=1)
    a.update(k)
    return LIB.yamd_layer_norm(a["x"], a["xs"], a["w"], a["b"], a["pd"], a["eps"], a["y"], a["ys"], a["mean"], a["rstd"], a["rows"], a["c"],
                               a["dt"], None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(y=None), dict(c=0), dict(c=16385), dict(rows=-1), dict(dt=2), dict(pd=7), dict(xs=63),
                                 dict(ys=10), dict(mean=FAKE), dict(eps=-1.0), dict(eps=math.nan)])
def test_layer_norm_abi_refuses(bad):
    assert _norm(**bad) == -1
    assert b"layer norm" in LIB.yamd_last_error()


def test_layer_norm_abi_empty_and_workspace():
    assert _norm(rows=0, x=None, y=None) == 0
    n = LIB.yamd_layer_norm_backward_workspace_bytes(1000, 256)
    assert n >= 2 * 256 * 4
    assert LIB.yamd_layer_norm_backward_workspace_bytes(-1, 256) == 0 and LIB.yamd_layer_norm_backward_workspace_bytes(5, 0) == 0
    back = lambda ws, nb, dx=FAKE, dw=FAKE: LIB.yamd_layer_norm_backward(FAKE, 64, FAKE, 64, None, 0, FAKE, FAKE, dx, 64, dw, None, 100, 64, 1,
                                                                         ws, nb, None)
    assert back(None, 0) == -3 and back(FAKE, 511) == -3
    assert back(FAKE, 1 << 20, dx=None, dw=None) == -1


def _desc(**k):
    a = dict(batch=2, heads=4, kv_heads=2, head_dim=64, q_len=100, k_len=100, map_h=0, map_w=0, scale=0.125)
    a.update(k)
    return L.AttentionDesc(**a)


def _tokens(ptr=FAKE, heads=4, d=64, n=100, **k):
    a = dict(data=ptr, batch_stride=n * heads * d, token_stride=heads * d, head_stride=d)
    a.update(k)
    return L.Tokens(**a)


def _attention(desc, bias=None, mask=None, mask_stride=100, ws=None, nb=0, exact=None, **over):
    t = {"q": _tokens(), "k": _tokens(heads=2), "v": _tokens(heads=2), "o": _tokens()}
    t.update(over)
    r = ctypes.byref
    return LIB.yamd_attention(r(desc), r(t["q"]), r(t["k"]), r(t["v"]), mask, mask_stride, bias, r(t["o"]), exact, None, ws, nb, None)


@pytest.mark.parametrize("bad", [dict(batch=0), dict(heads=3), dict(kv_heads=0), dict(head_dim=4), dict(head_dim=12), dict(head_dim=136),
                                 dict(q_len=0), dict(k_len=0), dict(k_len=(1 << 24) + 1), dict(scale=0.0), dict(scale=-1.0),
                                 dict(scale=math.inf), dict(scale=math.nan), dict(scale=1e-30)])
def test_attention_abi_refuses_descriptors(bad):
    assert _attention(_desc(**bad)) == -1
    assert b"attention" in LIB.yamd_last_error()
    assert LIB.yamd_attention_workspace_bytes(ctypes.byref(_desc(**bad)), 0) == 0
    assert LIB.yamd_attention_backward_workspace_bytes(ctypes.byref(_desc(**bad)), 0) == 0


@pytest.mark.parametrize("name", ["q", "k", "v", "o"])
@pytest.mark.parametrize("bad", [dict(data=None), dict(data=FAKE + 8), dict(token_stride=12), dict(token_stride=0), dict(head_stride=4),
                                 dict(batch_stride=-8), dict(token_stride=(1 << 23) + 8)])
def test_attention_abi_refuses_tensors(name, bad):
    assert _attention(_desc(), **{name: _tokens(heads=4 if name in "qo" else 2, **bad)}) == -1


@pytest.mark.parametrize("bad", [dict(token_stride=8), dict(token_stride=248), dict(head_stride=8), dict(head_stride=56), dict(batch_stride=0),
                                 dict(batch_stride=25592), dict(token_stride=64, head_stride=6392)])
def test_attention_abi_refuses_results_that_overlap(bad):
    """Inputs may repeat memory, results may not; (batch, head, token) order is as good as (batch, token, head)."""
    r, d, ok, kv = ctypes.byref, _desc(), _tokens(), _tokens(heads=2)
    assert _attention(d, o=_tokens(**bad)) == -1 and b"overlap" in LIB.yamd_last_error()
    back = lambda dq=ok, dk=kv, dv=kv: LIB.yamd_attention_backward(r(d), r(ok), r(kv), r(kv), None, 0, None, r(ok), None, FAKE, r(ok), r(dq), r(dk),
                                                                   r(dv), None, None, 0, None)
    assert back(dq=_tokens(**bad)) == -1 and b"overlap" in LIB.yamd_last_error()
    for two in (dict(token_stride=8), dict(token_stride=120), dict(batch_stride=0)):
        assert back(dk=_tokens(heads=2, **two)) == -1 and back(dv=_tokens(heads=2, **two)) == -1 and b"overlap" in LIB.yamd_last_error()
    heads_first = _tokens(token_stride=64, head_stride=6400)
    assert back(dq=heads_first) == -3                                            # all that is missing is the workspace


def test_attention_abi_refuses_sizes_beyond_a_launch():
    for k in (dict(batch=1 << 10, heads=1 << 10, kv_heads=1 << 10, q_len=1025, k_len=1), dict(batch=1 << 10, heads=1 << 10, kv_heads=1 << 10, k_len=1025)):
        assert _attention(_desc(**k)) == -1 and b"2^30" in LIB.yamd_last_error()
        assert LIB.yamd_attention_backward_workspace_bytes(ctypes.byref(_desc(**k)), 0) == 0
    assert LIB.yamd_relative_bias_backward(FAKE, FAKE, FAKE, 9, 2, (1 << 20) + 1, FAKE, 0, None) == -1


def test_attention_abi_refuses_bias_mask_workspace():
    assert _attention(_desc(), bias=FAKE) == -1                                  # no map
    assert _attention(_desc(map_h=10, map_w=11), bias=FAKE) == -1                # not q_len positions
    assert _attention(_desc(map_h=2, map_w=800, q_len=1600, k_len=1600), bias=FAKE) == -1
    assert _attention(_desc(), mask=FAKE, mask_stride=99) == -1
    assert _attention(_desc(), exact=FAKE + 4) == -1
    big = _desc(batch=1, heads=1, kv_heads=1, q_len=1, k_len=100000)
    need = LIB.yamd_attention_workspace_bytes(ctypes.byref(big), 0)
    assert need > 0
    t = dict(q=_tokens(heads=1, n=1), k=_tokens(heads=1, n=100000), v=_tokens(heads=1, n=100000), o=_tokens(heads=1, n=1))
    assert _attention(big, **t) == -3 and _attention(big, ws=FAKE, nb=need - 1, **t) == -3 and _attention(big, ws=FAKE + 4, nb=need, **t) == -3
    assert LIB.yamd_attention_workspace_bytes(ctypes.byref(_desc(batch=64, q_len=1600, k_len=1600)), 0) == 0


def test_attention_backward_abi_refuses():
    r = ctypes.byref
    q, k = _tokens(), _tokens(heads=2)

    def back(desc, bias=None, dbias=None, lse=FAKE, exact=None, ws=FAKE, nb=1 << 40, dq=q, dk=k):
        return LIB.yamd_attention_backward(r(desc), r(q), r(k), r(k), None, 0, bias, r(q), exact, lse, r(q), r(dq), r(dk), r(k), dbias, ws, nb, None)

    d = _desc(map_h=10, map_w=10)
    assert back(d, lse=None) == -1
    assert back(d, dbias=FAKE) == -1                        # a gradient of no bias
    assert back(d, bias=FAKE, dbias=FAKE) == -1             # needs the exact output
    assert back(d, dq=_tokens(token_stride=4)) == -1 and back(d, dk=_tokens(heads=2, data=None)) == -1
    need = LIB.yamd_attention_backward_workspace_bytes(r(d), 1)
    assert need > LIB.yamd_attention_backward_workspace_bytes(r(d), 0) > 0
    assert back(d, ws=None) == -3 and back(d, bias=FAKE, dbias=FAKE, exact=FAKE, nb=need - 1) == -3
    assert LIB.yamd_attention_backward_workspace_bytes(r(_desc()), 1) == 0      # a bias without a map


def test_relative_bias_abi_refuses():
    call = lambda **k: LIB.yamd_relative_bias(*{**dict(t=FAKE, dt=0, of=FAKE, n=9, h=2, nb=4, o=FAKE, st=None), **k}.values())
    back = lambda **k: LIB.yamd_relative_bias_backward(*{**dict(g=FAKE, order=FAKE, start=FAKE, n=9, h=2, nb=4, t=FAKE, dt=0, st=None), **k}.values())
    for bad in (dict(t=None), dict(dt=3), dict(n=0), dict(h=0), dict(h=65536), dict(nb=0)):
        assert call(**bad) == -1 and back(**bad) == -1
    assert call(of=None) == -1 and call(o=None) == -1 and back(order=None) == -1 and back(g=None) == -1


def test_program_records_tokens():
    p = Program(64, 64)
    x = p.buffer(8, 8, 64)
    qkv = p.buffer(8, 8, 192)
    n = p.layer_norm("n", x, torch.ones(64), torch.zeros(64))
    pos = tokens.RelativePosition(8, 8, 8, 16, device="cpu")
    y = p.attention("a", qkv.slice(0, 64), qkv.slice(64, 64), qkv.slice(128, 64), 2, table=torch.zeros(pos.rows, 2), position=pos)
    assert (n.h, n.w, n.c) == (8, 8, 64) and (y.h, y.w, y.c) == (8, 8, 64)
    assert p._inputs_of(p.ops[0]) == [x] and len(p._inputs_of(p.ops[1])) == 3
    flops, byts = p.op_cost(p.ops[1], 3)
    assert flops == 4 * 3 * 64 * 64 * 64 and byts == 3 * 2 * 4 * 64 * 64
    grid = p.buffer(4, 4, 128)
    for q, k, v, kw in [(qkv.slice(0, 64), qkv.slice(64, 32), qkv.slice(128, 64), dict(heads=2)),
                        (qkv.slice(0, 60), qkv.slice(64, 60), qkv.slice(128, 60), dict(heads=2)),
                        (qkv.slice(4, 64), qkv.slice(64, 64), qkv.slice(128, 64), dict(heads=2)),
                        (qkv.slice(0, 64), grid.slice(0, 64), grid.slice(64, 64), dict(heads=2, table=torch.zeros(pos.rows, 2), position=pos)),
                        (qkv.slice(0, 64), qkv.slice(64, 64), qkv.slice(128, 64), dict(heads=2, position=pos))]:
        with pytest.raises(L.YamdError):
            p.attention("bad", q, k, v, **kw)
    fp32, wide = p.buffer(8, 8, 64, torch.float32), p.buffer(8, 8, 72)
    for x, out in [(fp32, None), (x, fp32)]:
        with pytest.raises(L.YamdError):
            p.layer_norm("bad", x, None, None, out=out)
    for out in (fp32, wide.slice(4, 64), qkv.slice(128, 64), qkv.slice(96, 64)):
        with pytest.raises(L.YamdError):
            p.attention("bad", qkv.slice(0, 64), qkv.slice(64, 64), qkv.slice(128, 64), 2, out=out)


def test_plan_takes_token_ops_and_refuses_beyond():
    ops = (L.PlanOp * 1)()
    ops[0].kind = L.OP_ATTENTION
    h = ctypes.c_void_p()
    assert LIB.yamd_plan_create(ops, 1, 2, 64, 64, ctypes.byref(h)) == 0
    failed = ctypes.c_int(-1)
    assert LIB.yamd_plan_run(h, FAKE, None, ctypes.byref(failed)) == -1 and failed.value == 0      # an empty descriptor
    LIB.yamd_plan_destroy(h)
    ops[0].kind = L.OP_ATTENTION + 1
    assert LIB.yamd_plan_create(ops, 1, 2, 64, 64, ctypes.byref(h)) == -1


def test_buckets_cover_every_pair_once():
    """The distance that the library reads for a pair of positions, a(query) - a(key) + a(last), against (dy, dx)."""
    h, w = 6, 9
    t = np.arange(h * w)
    a = t + t // w * (w - 1)
    got = a[:, None] - a[None, :] + a[-1]
    want = (t[:, None] // w - t[None, :] // w + h - 1) * (2 * w - 1) + t[:, None] % w - t[None, :] % w + w - 1
    assert (got == want).all()
