"""CPU checks of token operators in recorded programs: where their maps come to lie, and what the rewrites leave alone."""
import pytest
import torch

from yolo_amd import lib as L
from yolo_amd.engine import Program


def _maps(*channels):
    p = Program(64, 64)
    return p, [p.buffer(8, 8, c) for c in channels]


def test_attention_result_must_not_overlap_an_operand_that_cat_moved():
    p, (q, k, v, x) = _maps(64, 64, 64, 64)
    whole = p.cat([k, x])
    for out in (whole.slice(0, 64), whole.slice(32, 64)):
        with pytest.raises(L.YamdError, match="overlaps"):
            p.attention("a", q, k, v, 2, out=out)
    with pytest.raises(L.YamdError, match="overlaps"):
        p.attention("a", whole.slice(32, 64), q, v, 2, out=x)
    assert p.attention("a", q, k, v, 2, out=x) == x
    assert p.attention("b", q, whole.slice(0, 64), v, 2, out=whole.slice(64, 64)) == whole.slice(64, 64)
    p._buffers_for(1, "cpu")


def test_attention_maps_that_cat_moves_off_their_alignment():
    # moved before the call
    p, (q, k, v, narrow) = _maps(64, 64, 64, 12)
    p.cat([narrow, k])
    with pytest.raises(L.YamdError, match="multiple of 8"):
        p.attention("a", q, k, v, 2)
    # moved afterwards: refused when the program is finished, before anything runs, and every time
    p, (q, k, v, narrow) = _maps(64, 64, 64, 12)
    y = p.attention("a", q, k, v, 2)
    p.cat([narrow, y])
    for _ in range(2):
        with pytest.raises(L.YamdError, match=r"attention\[a\].*multiple of 8"):
            p._buffers_for(1, "cpu")
    # a whole buffer of 12 + 64 channels leaves no pixel aligned, wherever the map starts in it
    p, (q, k, v, narrow) = _maps(64, 64, 64, 12)
    y = p.attention("a", q, k, v, 2)
    p.cat([y, narrow])
    with pytest.raises(L.YamdError, match="multiple of 8"):
        p._buffers_for(1, "cpu")
    p, (q, k, v, wide) = _maps(64, 64, 64, 16)
    p.cat([wide, p.attention("a", q, k, v, 2)])
    p._buffers_for(1, "cpu")


def _upsampled(write_between):
    """low -> 2x -> cat with side -> 1x1 conv, with something written in between: over low, over the upsampled map, elsewhere."""
    p = Program(64, 64)
    low, side = p.buffer(8, 8, 64), p.buffer(16, 16, 64)
    up = p.upsample2x(low)
    write_between(p, low, up)
    p.conv("reader", p.cat([up, side]), torch.zeros(64, 128, 1, 1), None, 1, L.ACT_NONE)
    p._buffers_for(1, "cpu")
    return [op[0] for op in p.ops]


def test_upsampling_stays_where_its_source_is_normalised_in_place():
    assert _upsampled(lambda p, low, up: None) == ["conv_cat2"]
    assert _upsampled(lambda p, low, up: p.layer_norm("n", low, None, None)) == ["norm", "conv_cat2"]
    assert _upsampled(lambda p, low, up: p.layer_norm("n", low, None, None, out=low)) == ["up2", "norm", "conv"]
    qkv = lambda p: [p.buffer(8, 8, 64) for _ in range(3)]
    assert _upsampled(lambda p, low, up: p.attention("a", *qkv(p), 1)) == ["attn", "conv_cat2"]
    assert _upsampled(lambda p, low, up: p.attention("a", *qkv(p), 1, out=low)) == ["up2", "attn", "conv"]
    wide = lambda p: [p.buffer(16, 16, 64) for _ in range(3)]
    assert _upsampled(lambda p, low, up: p.attention("a", *wide(p), 1, out=up)) == ["up2", "attn", "conv"]


def test_every_op_names_its_results():
    p = Program(64, 64)
    x = p.buffer(8, 8, 32)
    y = p.conv("c", x, torch.zeros(32, 32, 1, 1), None, 1, L.ACT_NONE)
    a, b = p.buffer(8, 8, 16), p.buffer(8, 8, 16)
    p.conv("s", x, torch.zeros(32, 32, 1, 1), None, 1, L.ACT_NONE, out=a, out2=b)
    u, m = p.upsample2x(x), p.maxpool2(x)
    d = p.conv_transpose2x("t", x, torch.zeros(32, 32, 2, 2), None)
    pools = p.buffer(8, 8, 96)
    p.maxpool5_cascade(x, *(pools.slice(32 * i, 32) for i in range(3)))
    n = p.layer_norm("n", x, None, None)
    o = p.attention("o", x, y, n, 1)
    got = [p._results_of(op) for op in p.ops]
    t = p.ops[4][3]                                          # the 1x1 conv in front of the scatter
    assert got == [[y], [a, b], [u], [m], [t], [d], [pools.slice(32 * i, 32) for i in range(3)], [n], [o]]
