"""Layer norm and cross attention under torch's transforms, as far as no device is needed."""
import pytest
import torch
from torch.autograd import forward_ad


def _calls(x):
    """(an operator on x alone, one per input that may carry a tangent), on the binding itself: no check of the device in front."""
    from glenet_amd import _lib
    ops = _lib.torch_ops()
    other = torch.randn(x.shape)
    w = torch.randn(x.shape[-1])
    ln, xa = ops.layer_norm.default, ops.cross_attention.default

    def four(t):
        return t.view(1, -1, 1, t.shape[-1])

    return [lambda t: ln(t, None, None, 1e-5), lambda t: ln(other, t[0], w, 1e-5), lambda t: ln(other, w, t[0], 1e-5),
            lambda t: xa(four(t), four(other), four(other), None, None, None, 1.0),
            lambda t: xa(four(other), four(t), four(other), None, None, None, 1.0),
            lambda t: xa(four(other), four(other), four(t), None, None, None, 1.0)]


@pytest.mark.parametrize("index", range(6))
def test_a_forward_mode_tangent_is_refused(index):
    x, t = torch.randn(3, 8), torch.randn(3, 8)
    call = _calls(x)[index]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, (x,), (t,))
