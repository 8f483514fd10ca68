"""GPU tests of the token operators' less usual forms, against the 64-bit reference and bounds of test_gpu_tokens.py."""
import math

import pytest
import torch

from test_gpu_tokens import _check, _inputs, _reference, _within
from yolo_amd import tokens

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
