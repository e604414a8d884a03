"""What tells a dual tensor from another, on the host."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from m2_b200 import ops


def test_tangents_are_found():
    x, n = torch.ones(3), torch.arange(3)
    ops._no_tangents("f", x, None, n)
    with fwAD.dual_level():
        ops._no_tangents("f", x, None, n)
        dual = fwAD.make_dual(x, torch.ones(3))
        for t in (dual, dual * 2, dual[1:], dual.bfloat16()):
            with pytest.raises(RuntimeError, match="f has no forward-mode"):
                ops._no_tangents("f", x, t)
        ops._no_tangents("f", fwAD.unpack_dual(dual).primal)

    def g(t):
        ops._no_tangents("g", t)
        return t * 2

    with pytest.raises(RuntimeError, match="g has no forward-mode"):
        torch.func.jvp(g, (x,), (x,))
