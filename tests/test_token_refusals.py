"""CPU checks of what the token operators refuse, beyond tests/test_tokens.py."""
import ctypes

import pytest
import torch

from yolo_amd import lib as L
from yolo_amd import tokens

LIB = L.LIB
FAKE = 4096          # an aligned address that no call below reads: every one is refused first


def test_layer_norm_in_place_needs_one_stride():
    norm = lambda ys, rows: LIB.yamd_layer_norm(FAKE, 64, None, None, 0, 1e-5, FAKE, ys, None, None, rows, 64, 1, None)
    for ys in (72, 128):
        assert norm(ys, 2) == -1 and b"in place" in LIB.yamd_last_error()
