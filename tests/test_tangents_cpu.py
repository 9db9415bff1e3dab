"""Forward-mode tangents: the decoding entries compute none, so tensors that carry one
are refused (on the CPU up to the device checks)."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from fireprot_amd import _native, rotary


def test_differentiated():
    x, y = torch.zeros(2, 3, 4, 32), torch.zeros(3)
    assert not _native.differentiated(x, None, y)
    assert _native.differentiated(x, None, torch.zeros(3, requires_grad=True))
    with torch.no_grad():
        assert not _native.differentiated(torch.zeros(3, requires_grad=True))
    with forward_ad.dual_level():
        assert not _native.differentiated(x, None, y)
        dual = forward_ad.make_dual(y, torch.ones(3))
        assert _native.differentiated(x, None, dual)
        with torch.no_grad():  # a tangent is carried on all the same
            assert _native.differentiated(dual, x)
    assert not _native.differentiated(x, y)


def test_rotary_refuses_a_tangent():
    f, p = rotary.rotary_frequencies(32), torch.arange(3)
    x, t = torch.zeros(2, 3, 4, 32), torch.ones(2, 3, 4, 32)
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(x, t)
        for call in (lambda: rotary.apply_rotary(dual, None, p, f),
                     lambda: rotary.apply_rotary(x, dual, p, f),
                     lambda: rotary.apply_rotary(x, None, p, f, q_out=dual),
                     lambda: rotary.rotary_backward(dual, None, p, f)):
            with pytest.raises(ValueError, match="no autograd graph"):
                call()
