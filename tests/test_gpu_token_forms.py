"""GPU tests of the token operators' less usual forms, against the 64-bit reference and bounds of test_gpu_tokens.py."""
import ctypes
import math
import threading

import pytest
import torch

from test_gpu_tokens import F, U, _block, _block_inputs, _check, _index, _inputs, _norm_case, _reference, _token_step, _within
from yolo_amd import lib as L
from yolo_amd import tokens
from yolo_amd.engine import Program

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h,w,heads,d", [(9, 12, 2, 64), (11, 13, 3, 40), (1, 333, 2, 128), (20, 20, 8, 32)])
def test_frozen_bias_gives_the_gradients_of_a_learned_one(gpu_device, h, w, heads, d):
    """A bias that needs no gradient has no sums by distance; dq, dk and dv are the same bits."""
    (q, k, v), do, g = _inputs(gpu_device, h * w + d, 2, h * w, h * w, heads, heads, d)
    pos = tokens.RelativePosition(h, w, 8, 16, gpu_device)
    table = torch.randn(pos.rows, heads, generator=g, device=gpu_device).requires_grad_()
    mask = torch.rand(2, h * w, generator=g, device=gpu_device) < 0.7
    learned = tokens.relative_bias(table, pos)
    want = torch.autograd.grad(tokens.attention(q, k, v, None, mask, learned, pos), (q, k, v, table), do)
    frozen = learned.detach()
    got = torch.autograd.grad(tokens.attention(q, k, v, None, mask, frozen, pos), (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ref, tol = _reference(q, k, v, 1 / math.sqrt(d), mask, frozen, (h, w), do)
    for n, x in zip(("dq", "dk", "dv"), got):
        _within(n, x, ref[n], tol[n])


def test_attention_result_may_change_before_its_backward_pass(gpu_device):
    """The backward pass does not read o (it has the unrounded one)."""
    leaves, do, _ = _inputs(gpu_device, 31, 2, 60, 90, 2, 1, 64)
    want = torch.autograd.grad(tokens.attention(*leaves), leaves, do)
    o = tokens.attention(*leaves)
    o += 1.0
    got = torch.autograd.grad(o, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("b,h,w,heads,kv,d", [
    (2, 9, 12, 4, 2, 64), (1, 11, 13, 4, 1, 40), (1, 1, 333, 8, 2, 32), (2, 1, 50, 4, 2, 64), (1, 5, 7, 8, 4, 16), (1, 1, 1, 2, 1, 8),
    (1, 20, 20, 4, 2, 128), (2, 7, 9, 6, 2, 96), (1, 1, 700, 4, 1, 104), (3, 8, 8, 2, 1, 120)])
@pytest.mark.parametrize("masked", [False, True])
def test_bias_with_shared_key_heads(gpu_device, b, h, w, heads, kv, d, masked):
    """dk and dv add over the heads of a group, each with its own bias."""
    n = h * w
    (q, k, v), do, g = _inputs(gpu_device, n + heads + d, b, n, n, heads, kv, d)
    pos = tokens.RelativePosition(h, w, 8, 16, gpu_device)
    table = torch.randn(pos.rows, heads, generator=g, device=gpu_device).requires_grad_()
    mask = None
    if masked:
        mask = torch.rand(b, n, generator=g, device=gpu_device) < 0.6
        mask[-1] = False
    _check(gpu_device, q, k, v, do, mask=mask, table=table, pos=pos)


@pytest.mark.parametrize("lq,lk,heads,kv,d,biased", [(70, 130, 4, 2, 64, False), (300, 2, 2, 2, 64, False), (33, 700, 2, 1, 96, False),
                                                     (128, 64, 1, 1, 32, False), (1, 1, 1, 1, 8, False), (5, 3000, 4, 2, 128, False),
                                                     (100, 100, 2, 1, 40, True)])
def test_backward_from_the_rounded_result(gpu_device, lq, lk, heads, kv, d, biased):
    """Through the C ABI without o_exact: D = rowsum(do o) takes over the rounding of o."""
    b, scale = 2, 1 / math.sqrt(d)
    leaves, do, g = _inputs(gpu_device, lq + lk + d, b, lq, lk, heads, kv, d)
    q, k, v = (t.detach() for t in leaves)
    bias = torch.randn(heads, 2 * lk - 1, generator=g, device=gpu_device) if biased else None
    desc = L.AttentionDesc(b, heads, kv, d, lq, lk, int(biased), lk if biased else 0, scale)
    r, tk = ctypes.byref, lambda t: ctypes.byref(L.Tokens(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)))
    room = lambda n: torch.empty(max(n, 1), dtype=torch.uint8, device=gpu_device)
    o, lse = torch.empty_like(q), torch.empty(b, heads, lq, device=gpu_device)
    grads = [torch.full_like(t, math.nan) for t in (q, k, v)]
    n = L.LIB.yamd_attention_workspace_bytes(r(desc), int(biased))
    ws = room(n)
    bp = None if bias is None else bias.data_ptr()
    L.check(L.LIB.yamd_attention(r(desc), tk(q), tk(k), tk(v), None, 0, bp, tk(o), None, lse.data_ptr(), ws.data_ptr(), n, L.current_stream()))
    n = L.LIB.yamd_attention_backward_workspace_bytes(r(desc), 0)
    ws2 = room(n)
    L.check(L.LIB.yamd_attention_backward(r(desc), tk(q), tk(k), tk(v), None, 0, bp, tk(o), None, lse.data_ptr(), tk(do),
                                          *(tk(t) for t in grads), None, ws2.data_ptr(), n, L.current_stream()))
    want, tol = _reference(q, k, v, scale, None, bias, (1, lk) if biased else None, do)
    # the error of o reaches D, and dS by P times it: added to the bounds with the exact o
    Q, G = q.double().transpose(1, 2), do.double().transpose(1, 2)
    K = k.double().transpose(1, 2).repeat_interleave(heads // kv, 1)
    s = scale * Q @ K.transpose(2, 3)
    if biased:
        s = s + bias.double()[:, _index(1, lk, gpu_device)]
    p = torch.softmax(s, 3)
    e_ds = 1.02 * p * (G.abs() * tol["o"].transpose(1, 2)).sum(3, keepdim=True)
    fold = lambda t: t.reshape(b, kv, heads // kv, lk, d).sum(2)
    tol["dq"] = tol["dq"] + (1.02 * scale * e_ds @ K.abs()).transpose(1, 2)
    tol["dk"] = tol["dk"] + 1.02 * scale * fold(e_ds.transpose(2, 3) @ Q.abs()).transpose(1, 2)
    for name, x in zip(("dq", "dk", "dv"), grads):
        _within(name, x, want[name], tol[name])
    _within("o", o, want["o"], tol["o"])


def test_two_host_threads_at_once(gpu_device):
    """Two threads, each with its stream and its inputs, forward and backward: what one thread alone gets."""
    cases = [_block_inputs(gpu_device, 60 + i, h=7 + 4 * i) for i in range(2)]

    def step(leaves, pos, dy):
        y = _block(*leaves, pos, 2)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    got, start = [[], []], threading.Barrier(2)

    def work(i):
        with torch.cuda.device(gpu_device), torch.cuda.stream(torch.cuda.Stream(gpu_device)):
            start.wait()
            for _ in range(20):
                got[i].append(step(*cases[i]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for i in range(2):
        assert len(got[i]) == 20
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))


@pytest.mark.parametrize("c,first,n", [(64, 0, 64), (40, 0, 40), (24, 3, 17)])
def test_program_normalises_in_place(gpu_device, c, first, n):
    g = torch.Generator().manual_seed(c)
    sd = dict(w=torch.randn(c, 3, 3, 3, generator=g), nw=torch.randn(n, generator=g), nb=torch.randn(n, generator=g))
    out = []
    for in_place in (False, True):
        p = Program(32, 32)
        x = p.conv("c", p.image16(), sd["w"], None, 2, L.ACT_NONE).slice(first, n)
        y = x if in_place else p.buffer(x.h, x.w, c).slice(first, n)
        p.outputs = {"y": p.layer_norm("n", x, sd["nw"], sd["nb"], out=y)}
        for batch in (3, 1):
            images = torch.rand(batch, 3, 32, 32, generator=torch.Generator().manual_seed(batch)).to(gpu_device)
            out.append(p.run(images)["y"].clone())
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[3])


def _captured(step):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


@pytest.mark.parametrize("which", ["layer_norm", "relative_bias", "attention", "attention over views"])
def test_captured_backward_with_live_eager_results_is_refused(gpu_device, which):
    """Each operator stops a captured backward pass before it reaches a leaf whose accumulator is an eager graph's on the default
    stream; once the eager result is gone, the same step is captured and replays."""
    (q, k, v), do, g = _inputs(gpu_device, 5, 1, 96, 96, 2, 2, 32)
    pos = tokens.RelativePosition(8, 12, 8, 16, gpu_device)
    n = lambda *s: torch.randn(*s, generator=g, device=gpu_device)
    if which == "layer_norm":
        leaves = [n(40, 64).bfloat16().requires_grad_(), n(64).requires_grad_(), n(64).requires_grad_()]
        do, forward = n(40, 64).bfloat16(), lambda: tokens.layer_norm(*leaves)
    elif which == "relative_bias":
        leaves = [n(pos.rows, 2).requires_grad_()]
        do, forward = n(2, pos.distances), lambda: tokens.relative_bias(leaves[0], pos)
    elif which == "attention":
        leaves, forward = [q, k, v], lambda: tokens.attention(q, k, v)
    else:                                                    # (the leaf lies behind torch's own nodes)
        leaves = [torch.stack((q, k, v), 2).detach().requires_grad_()]
        forward = lambda: tokens.attention(*leaves[0].unbind(2))
    step = lambda: torch.autograd.grad(forward(), leaves, do)
    want = step()                                            # (its graph is gone when it returns)
    alive = forward()
    with pytest.raises(RuntimeError, match="eager result"):
        _captured(step)
    with torch.cuda.stream(torch.cuda.Stream(gpu_device)):   # without a capture nothing is refused
        again = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    del alive
    graph, out = _captured(step)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_captured_backward_refuses_through_a_whole_step(gpu_device):
    pos = tokens.RelativePosition(8, 100, 8, 16, gpu_device)
    n = lambda *s: torch.randn(*s, device=gpu_device)
    leaves = [n(1, 800, 64).bfloat16().requires_grad_(), n(64).requires_grad_(), n(64).requires_grad_(), n(pos.rows, 2).requires_grad_()]
    dy = n(1, 800, 2, 32).bfloat16()
    alive = tokens.layer_norm(*leaves[:3])
    with pytest.raises(RuntimeError, match="eager result"):
        _captured(lambda: _token_step(leaves, pos, dy))
    del alive
    want = _token_step(leaves, pos, dy)
    want = [t.detach() for t in want]
    graph, out = _captured(lambda: [t.detach() for t in _token_step(leaves, pos, dy)])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_capture_asks_for_other_leaves_than_the_live_result(gpu_device):
    """An eager result that holds only a leaf whose gradient the captured pass does not ask for is in nobody's way."""
    (q, k, v), do, _ = _inputs(gpu_device, 6, 1, 50, 70, 2, 2, 32)
    step = lambda: torch.autograd.grad(tokens.attention(q, k, v), (q,), do)
    want = step()
    alive = tokens.layer_norm(k)
    graph, out = _captured(step)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and alive.grad_fn is not None


@pytest.mark.parametrize("wanted", ["q", "k", "v", "bias", "qv", "k bias"])
def test_gradients_of_some_arguments_only(gpu_device, wanted):
    """The others need none: the same bits as when all do."""
    h, w, heads = 7, 12, 2
    (q, k, v), do, g = _inputs(gpu_device, 12, 2, h * w, h * w, heads, heads, 40)
    pos = tokens.RelativePosition(h, w, 8, 16, gpu_device)
    bias = tokens.relative_bias(torch.randn(pos.rows, heads, generator=g, device=gpu_device), pos).requires_grad_()
    names = ["q", "k", "v", "bias"]
    step = lambda leaves, asked: torch.autograd.grad(tokens.attention(*leaves[:3], bias=leaves[3], position=pos), asked, do)
    want = dict(zip(names, step([q, k, v, bias], [q, k, v, bias])))
    on = [n in (wanted.split() if " " in wanted or wanted == "bias" else wanted) for n in names]
    leaves = [t.detach().clone().requires_grad_(x) for t, x in zip((q, k, v, bias), on)]
    for n, got in zip([n for n, x in zip(names, on) if x], step(leaves, [t for t, x in zip(leaves, on) if x])):
        assert torch.equal(got, want[n]), n


def test_more_images_than_waves_share_a_bias(gpu_device):
    """The sums by distance over 20 and 33 images: more than the 16 waves that take them in turns."""
    for b in (20, 33):
        (q, k, v), do, g = _inputs(gpu_device, b, b, 150, 150, 1, 1, 16)
        pos = tokens.RelativePosition(10, 15, 8, 16, gpu_device)
        table = torch.randn(pos.rows, 1, generator=g, device=gpu_device).requires_grad_()
        _check(gpu_device, q, k, v, do, table=table, pos=pos)


def test_very_many_small_images(gpu_device):
    (q, k, v), do, _ = _inputs(gpu_device, 3, 70001, 1, 3, 2, 1, 16)
    _check(gpu_device, q, k, v, do)


def test_mask_rows_of_a_wider_mask(gpu_device):
    (q, k, v), do, g = _inputs(gpu_device, 4, 3, 40, 70, 2, 2, 32)
    wide = torch.rand(3, 100, generator=g, device=gpu_device) < 0.5
    mask = wide[:, 7:77]
    assert mask.data_ptr() % 4 and not mask.is_contiguous()
    want = torch.autograd.grad(tokens.attention(q, k, v, None, mask.contiguous()), (q, k, v), do)
    got = torch.autograd.grad(tokens.attention(q, k, v, None, mask), (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layer_norm_gradient_from_a_longer_vector(gpu_device):
    """A gradient that starts off a 16-byte boundary takes the kernels of single channels: held to the bound."""
    g = torch.Generator(device=gpu_device).manual_seed(8)
    n = lambda *s: torch.randn(*s, generator=g, device=gpu_device)
    for c in (64, 512, 1024, 8192):
        x, w, b = n(70, c).requires_grad_(), n(c).requires_grad_(), n(c).requires_grad_()
        dy = torch.cat([n(3), n(70 * c)])[3:].view(70, c)
        assert dy.data_ptr() % 16 and dy.is_contiguous()
        y = tokens.layer_norm(x, w, b)
        want, tol = _norm_case(gpu_device, x, w, b, 1e-5, dy, F)
        for name, a, r, t in zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy), want[1:], tol[1:]):
            _within(name, a, r, t + F * (r.abs() + t))


@pytest.mark.parametrize("b,lq,lk,heads,kv,d,hw", [(2, 300, 8400, 2, 2, 32, None), (1, 1, 8400, 8, 2, 64, None), (1, 1600, 1600, 4, 2, 128, None),
                                                   (1, 1447, 1447, 2, 2, 40, (1, 1447)), (1, 1600, 1600, 2, 2, 64, (40, 40)),
                                                   (1, 1444, 1444, 2, 1, 104, (38, 38))])
def test_long_axes_in_norm(gpu_device, b, lq, lk, heads, kv, d, hw):
    """Elementwise bounds add worst cases over all keys.  Relative to the whole tensor a result carries two independent roundings to
    bf16 (of P or dS, and its own), each at most U / sqrt(3) of it in the root mean square: twice that of both is allowed.  The
    bias gradient takes float32 dS, whose error is that of D: one rounding's share."""
    (q, k, v), do, g = _inputs(gpu_device, lq + lk + d, b, lq, lk, heads, kv, d)
    bias, kw = None, {}
    if hw:
        pos = tokens.RelativePosition(*hw, 16, 40, gpu_device)
        bias = tokens.relative_bias(torch.randn(pos.rows, heads, generator=g, device=gpu_device), pos).requires_grad_()
        kw = dict(bias=bias, position=pos)
    o = tokens.attention(q, k, v, **kw)
    leaves = [q, k, v] + ([bias] if hw else [])
    grads = torch.autograd.grad(o, leaves, do)
    want, _ = _reference(q, k, v, 1 / math.sqrt(d), None, bias, hw, do)
    rounding = U / math.sqrt(3)
    for n, got in zip(("dq", "dk", "dv", "dbias", "o"), grads + (() if hw else (None,)) + (o,)):
        if got is not None:
            off = ((got.detach().double() - want[n]).norm() / want[n].norm()).item()
            assert off <= (rounding if n == "dbias" else 2 * math.sqrt(2) * rounding), (n, off)


@pytest.mark.parametrize("h,w,d", [(2, 760, 128), (3, 759, 40), (2, 760, 64), (1, 5001, 8), (600, 3, 96)])
def test_widest_and_longest_maps(gpu_device, h, w, d):
    """The most LDS that a bias takes, and distances far beyond a tile."""
    n = h * w
    (q, k, v), do, g = _inputs(gpu_device, n + d, 1, n, n, 1, 1, d)
    pos = tokens.RelativePosition(h, w, 8, 64, gpu_device)
    table = torch.randn(pos.rows, 1, generator=g, device=gpu_device).requires_grad_()
    _check(gpu_device, q, k, v, do, table=table, pos=pos)
