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
