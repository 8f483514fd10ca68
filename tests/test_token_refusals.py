"""CPU checks of what the token operators refuse, beyond tests/test_tokens.py."""
import ctypes
import glob
import os
import re

import pytest
import torch

from conftest import ROOT

from yolo_amd import lib as L
from yolo_amd import tokens

LIB = L.LIB
FAKE = 4096          # an aligned address that no call below reads: every one is refused first


def test_layer_norm_in_place_needs_one_stride():
    norm = lambda ys, rows: LIB.yamd_layer_norm(FAKE, 64, None, None, 0, 1e-5, FAKE, ys, None, None, rows, 64, 1, None)
    for ys in (72, 128):
        assert norm(ys, 2) == -1 and b"in place" in LIB.yamd_last_error()


def test_inline_assembly_declares_what_it_writes():
    """Assembly that sets m0 names it among what it writes; a compiler that kept something there would lose it otherwise."""
    found = 0
    for f in glob.glob(os.path.join(ROOT, "yolo_amd", "csrc", "*.h")) + glob.glob(os.path.join(ROOT, "yolo_amd", "csrc", "*.hip")):
        for block in re.findall(r"\basm\s+(?:volatile\s*)?\((.*?)\);", open(f).read(), re.S):
            if re.search(r"s_mov_b32 m0", block):
                found += 1
                assert '"m0"' in block.rsplit(":", 1)[1], (f, block)
    assert found >= 2


def _calls():
    """(operator over its floating-point arguments, those arguments)"""
    x, w = torch.randn(4, 8), torch.ones(8)
    q = torch.randn(1, 4, 1, 8).bfloat16()
    pos = tokens.RelativePosition(2, 2, 8, 16, device="cpu")
    table, bias = torch.zeros(pos.rows, 1), torch.zeros(1, pos.distances)
    return [(lambda x, w, b: tokens.layer_norm(x, w, b), [x, w, w.clone()]),
            (lambda q, k, v, b: tokens.attention(q, k, v, bias=b, position=pos), [q, q.clone(), q.clone(), bias]),
            (lambda t: tokens.relative_bias(t, pos), [table])]


def test_forward_mode_tangents_are_refused():
    """(before anything else, so that a CPU tensor shows it; a tensor without a tangent gets to the next check)"""
    with torch.autograd.forward_ad.dual_level():
        for op, args in _calls():
            for i in range(len(args)):
                dual = list(args)
                dual[i] = torch.autograd.forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(L.YamdError, match="forward-mode"):
                    op(*dual)
            with pytest.raises(L.YamdError, match="GPU"):
                op(*args)


def test_traces_are_refused():
    for op, args in _calls():
        with pytest.raises(L.YamdError, match="jit.trace"):
            torch.jit.trace(op, tuple(args))
        with pytest.raises(L.YamdError, match="GPU"):
            op(*args)


def test_a_bias_without_gradient_needs_no_room_for_its_sums():
    r = ctypes.byref
    d = L.AttentionDesc(8, 8, 8, 64, 6400, 6400, 80, 80, 0.125)
    size = LIB.yamd_attention_backward_workspace_bytes
    plain, summed = size(r(d), 0), size(r(d), 1)
    assert summed - plain > 8 * 8 * 6400 * 6400 // 64 * 4 * 0.9
    t = L.Tokens(FAKE, 6400 * 512, 512, 64)
    back = lambda dbias, nb: LIB.yamd_attention_backward(r(d), r(t), r(t), r(t), None, 0, FAKE, r(t), FAKE, FAKE, r(t), r(t), r(t), r(t), dbias,
                                                         FAKE, nb, None)
    # refused for want of room, with the room that is wanted in the message
    assert back(None, plain - 1) == -3 and f"needs {plain} ".encode() in LIB.yamd_last_error()
    assert back(FAKE, summed - 1) == -3 and f"needs {summed} ".encode() in LIB.yamd_last_error()


def test_attention_backward_takes_o_in_one_of_two_forms():
    r = ctypes.byref
    d = L.AttentionDesc(1, 2, 2, 64, 100, 100, 0, 0, 0.125)
    t = L.Tokens(FAKE, 12800, 128, 64)
    back = lambda o, exact: LIB.yamd_attention_backward(r(d), r(t), r(t), r(t), None, 0, None, o, exact, FAKE, r(t), r(t), r(t), r(t), None,
                                                        None, 0, None)
    odd = L.Tokens(FAKE + 2, 12800, 128, 64)
    assert back(None, None) == -1 and back(r(odd), None) == -1 and back(r(odd), FAKE) == -1 and back(None, FAKE + 4) == -1
    assert back(None, FAKE) == -3 and back(r(t), FAKE) == -3 and back(r(t), None) == -3          # all that is missing is the workspace
