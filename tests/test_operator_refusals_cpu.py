"""Refusals of layer norm, the orthogonaliser and cross attention that need no device."""
import pytest
import torch


def test_layer_norm_refuses():
    from glenet_amd import _lib
    from glenet_amd.norm import layer_norm
    x = torch.zeros(3, 8)
    with pytest.raises(_lib.GlxError, match="no CPU path"):
        layer_norm(x)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        layer_norm(x.double())
    with pytest.raises(ValueError, match="shape"):
        layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="one type"):
        layer_norm(x, torch.ones(8).half())
    with pytest.raises(ValueError, match="one type"):
        layer_norm(x.half(), torch.ones(8).half(), torch.zeros(8))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.zeros(()))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
