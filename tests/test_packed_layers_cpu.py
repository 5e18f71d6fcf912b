"""The host side of packed layers, without a GPU."""

import pytest
import torch
from torch.autograd import forward_ad

from aimet_amd.quantization.affine.packed import _refuse_gradients


def test_tangents_are_refused():
    x, t = torch.randn(3), torch.ones(3)
    with forward_ad.dual_level():
        _refuse_gradients("call", x, None)
        dual = forward_ad.make_dual(x, t)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                _refuse_gradients("call", None, dual * 2)
    _refuse_gradients("call", x, None)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda v: _refuse_gradients("call", v), (x,), (t,))
