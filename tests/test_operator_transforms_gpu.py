"""Layer norm and cross attention under torch's transforms, on the device."""
import pytest
import torch
from torch.autograd import forward_ad

from test_operator_transforms_cpu import _attention, _gradients, _layer_norm

pytestmark = pytest.mark.gpu


def _args(name, dtype, dev, seed):
    g = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g).to(dev)

    if name == "layer_norm":
        return _layer_norm, [normal(5, 7, 24).to(dtype), normal(24), normal(24)]
    mask = (torch.rand(2, 9, generator=g) < 0.6).to(dev)
    return _attention, [normal(2, 5, 4, 24).to(dtype), normal(2, 9, 2, 24).to(dtype), mask]


@pytest.mark.parametrize("name", ["layer_norm", "cross_attention"])
def test_a_forward_mode_tangent_is_refused(dev, name):
    f, args = _args(name, torch.float32, dev, 0)
    with forward_ad.dual_level():
        for i in range(2):
            duals = list(args)
            duals[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*duals)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f(*duals)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: f(x, *args[1:]), (args[0],), (args[0],))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("name", ["layer_norm", "cross_attention"])
def test_a_traced_function_gives_what_the_function_gives(dev, name, train, dtype):
    """Traced on one set of inputs, run on another."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, args = _args(name, dtype, dev, 1)
    f = _gradients(f) if train else f
    graph = make_fx(f)(*args)
    _, other = _args(name, dtype, dev, 2)
    for inputs in (other, args):
        want, got = f(*inputs), graph(*inputs)
        for a, b in zip(want if train else (want,), got if train else (got,)):
            assert torch.equal(a, b) and bool(torch.isfinite(a).all())


@pytest.mark.parametrize("name", ["layer_norm", "cross_attention"])
def test_functional_transforms(dev, name):
    """vmap takes one call per sample; torch.func.grad, whose levels the nodes do not know, is refused."""
    f, args = _args(name, torch.float32, dev, 3)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda x: f(x, *args[1:]).sum())(args[0])
    rows = torch.stack([args[0], args[0] * 2])
    both = torch.func.vmap(lambda x: f(x, *args[1:]))(rows)
    assert torch.equal(both[0], f(rows[0], *args[1:])) and torch.equal(both[1], f(rows[1], *args[1:]))


@pytest.mark.parametrize("name", ["layer_norm", "cross_attention"])
def test_a_direct_call_of_a_training_pass_has_no_gradient_of_its_own(dev, name):
    from glenet_amd import _lib
    ops = _lib.torch_ops()
    _, args = _args(name, torch.float32, dev, 4)
    x = args[0].requires_grad_()
    if name == "layer_norm":
        y = ops.layer_norm_train.default(x, None, None, 1e-5)[0]
    else:
        y = ops.cross_attention_train.default(x, args[1], args[1], None, None, None, 1.0)[0]
    with pytest.raises(RuntimeError, match="not implemented"):
        y.sum().backward()


def test_the_orthogonaliser_is_not_traced(dev):
    from glenet_amd import _lib
    from glenet_amd.optim import orthogonalize
    from torch.fx.experimental.proxy_tensor import make_fx
    m = torch.randn(20, 30, device=dev)
    with pytest.raises(_lib.GlxError, match="cannot be traced"):
        make_fx(lambda t: orthogonalize(t))(m)
    assert torch.equal(orthogonalize(m), orthogonalize(m))       # (nothing of the trace is left)


@pytest.mark.parametrize("name", ["layer_norm", "cross_attention"])
def test_compiled_and_exported_functions(dev, name):
    """torch.compile with the operators' own gradients, torch.export and the script tracer: the function's results, to the bit."""
    f, args = _args(name, torch.float32, dev, 5)
    leaves = [a.requires_grad_() if a.is_floating_point() else a for a in args]
    wanted = [a for a in leaves if a.requires_grad]

    def both(g):
        y = g(*leaves)
        return [y] + list(torch.autograd.grad(y.sum(), wanted))

    for a, b in zip(both(f), both(torch.compile(f, backend="aot_eager"))):
        assert torch.equal(a, b)

    class Module(torch.nn.Module):
        def forward(self, *a):
            return f(*a)

    with torch.no_grad():
        want = f(*leaves)
        assert torch.equal(torch.export.export(Module(), tuple(args)).module()(*args), want)
        assert torch.equal(torch.jit.trace(f, tuple(args), check_trace=False)(*args), want)
