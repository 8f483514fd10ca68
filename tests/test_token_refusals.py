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
