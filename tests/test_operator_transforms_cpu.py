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


def _layer_norm(x, w, b):
    from glenet_amd.norm import layer_norm
    return layer_norm(x, w, b)


def _attention(q, k, mask):
    from glenet_amd.attention import cross_attention
    return cross_attention(q, k, k, key_mask=mask)


def _gradients(f):
    def run(*args):
        leaves = [a.detach().requires_grad_() if a.is_floating_point() else a for a in args]
        y = f(*leaves)
        return (y, *torch.autograd.grad(y.sum(), [a for a in leaves if a.requires_grad]))
    return run


def _fakes(name, dtype):
    if name == "layer_norm":
        return _layer_norm, [torch.empty(5, 7, 24, device="cuda", dtype=dtype), torch.empty(24, device="cuda"), torch.empty(24, device="cuda")]
    return _attention, [torch.empty(2, 5, 4, 24, device="cuda", dtype=dtype), torch.empty(2, 9, 2, 24, device="cuda", dtype=dtype),
                        torch.empty(2, 9, device="cuda", dtype=torch.bool)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["layer_norm", "cross_attention"])
def test_a_traced_function_keeps_the_operator(name, dtype):
    """Device tensors without storage: the trace holds the operator, with the shape and type it gives, and no bare allocation."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    with FakeTensorMode():
        f, args = _fakes(name, dtype)
        graph = make_fx(f)(*args)
        out = graph(*args)
        assert (out.shape, out.dtype, out.device) == (args[0].shape, args[0].dtype, args[0].device)
    used = {str(n.target) for n in graph.graph.nodes if n.op == "call_function"}
    assert "glenet.%s.default" % name in used and not any("empty" in u for u in used)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_of_the_training_passes(dtype):
    """What the autograd nodes call, traced: results and gradients as the device gives them, None for those nobody wants."""
    from glenet_amd import _lib
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    ops = _lib.torch_ops()

    def sizes(*ts):
        return [None if t is None else (tuple(t.shape), t.dtype) for t in ts]

    def norm(x, w, b):
        y, mean, rstd = ops.layer_norm_train.default(x, w, b, 1e-5)
        return (y, mean, rstd, *ops.layer_norm_backward.default(y, x, w, mean, rstd, torch.float32, [True, True, True]),
                *ops.layer_norm_backward.default(y, x, w, mean, rstd, torch.float32, [False, True, False]))

    def attend(q, k, mask):
        out, lse, rest = ops.cross_attention_train.default(q, k, k, None, None, mask, 1.0)
        saved = (out, q, k, k, None, None, mask, out, lse, rest, 1.0)
        return (out, lse, rest, *ops.cross_attention_backward.default(*saved, [True, True, True]),
                *ops.cross_attention_backward.default(*saved, [False, False, True]))

    with FakeTensorMode():
        x, w, b = _fakes("layer_norm", dtype)[1]
        graph = make_fx(norm)(x, w, b)
        f32, rows, width = torch.float32, ((35,), torch.float32), ((24,), torch.float32)
        assert sizes(*graph(x, w, b)) == [((5, 7, 24), dtype), rows, rows, ((5, 7, 24), dtype), width, width, None, width, None]
        q, k, mask = _fakes("cross_attention", dtype)[1]
        graph = make_fx(attend)(q, k, mask)
        big, small = ((2, 5, 4, 24), dtype), ((2, 9, 2, 24), dtype)
        rest = ((0,), f32) if dtype == f32 else ((2, 5, 4, 24), torch.bfloat16)
        assert sizes(*graph(q, k, mask)) == [big, ((2, 5, 4), f32), rest, big, small, small, None, None, small]
    assert sum("backward" in str(n.target) for n in graph.graph.nodes) == 2


def test_tensors_without_a_device_are_refused_by_the_binding():
    from glenet_amd import _lib
    ops = _lib.torch_ops()
    x = torch.zeros(2, 5, 4, 16)
    with pytest.raises(NotImplementedError, match="CPU"):
        ops.layer_norm.default(x, None, None, 1e-5)
    with pytest.raises(NotImplementedError, match="CPU"):
        ops.cross_attention.default(x, x, x, None, None, None, 1.0)


def test_what_launches_on_raw_pointers_is_not_traced():
    """The orthogonaliser is outside autograd and no operator of torch: a trace of it would return memory that nobody wrote."""
    from glenet_amd import _lib
    from glenet_amd.optim import orthogonalize
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    with FakeTensorMode():
        m = torch.empty(20, 30, device="cuda")
        with pytest.raises(_lib.GlxError, match="cannot be traced"):
            make_fx(lambda t: orthogonalize(t))(m)
        with pytest.raises(_lib.GlxError, match="cannot be traced"):
            orthogonalize([m])
    with pytest.raises(_lib.GlxError, match="cannot be traced"):
        make_fx(lambda t: (_lib.call("glx_abi_version"), t * 2)[1])(torch.ones(3))


def test_nor_is_it_by_the_script_tracer():
    from glenet_amd import _lib
    with pytest.raises(_lib.GlxError, match="cannot be traced"):
        torch.jit.trace(lambda t: (_lib.call("glx_abi_version"), t * 2)[1], torch.ones(3))
    assert torch._C._get_tracing_state() is None
