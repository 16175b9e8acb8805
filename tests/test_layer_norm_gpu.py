"""glenet_amd.norm.layer_norm (csrc/glx_layernorm.hip) against the formulas in 64 bits, every form of the kernels (part of a
wave, a wave, a block per row, rows in passes), both directions.

Tolerances.  u = 2^-24.  A sum's error is at most depth * u * sum |terms|; a thread adds at most 64 values, the tree behind it
has at most 10 + 16 steps: depth 96 covers every row sum, and with the handful of roundings behind it K = 128.  With
s = max |x - mean| / sd and r = max |x| / sd of the inputs, |d xhat| <= K u (r + s) covers mean, variance and the product.  The
column sums add at most rows terms in a chain: depth min(rows, 128 + 64) + 20.  A result of fewer bits adds half a step of itself."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
K = 128
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}       # half a subnormal step
SHAPES = [(1, 1), (3, 5), (2, 32), (128, 256), (1000, 63), (17, 64), (5000, 65), (33, 511), (70, 1024), (9, 2049), (5, 4097),
          (300, 8200), (2, 20736), (3, 40001), (2, 70001)]


def _formula(x, w, b, gy, eps):
    x, gy = x.double(), gy.double()
    mean = x.mean(1, keepdim=True)
    sd = ((x - mean) ** 2).mean(1, keepdim=True).add(eps).sqrt()
    xh = (x - mean) / sd
    wd = w.double() if w is not None else torch.ones_like(x[0])
    y = xh * wd + (b.double() if b is not None else 0.0)
    g = gy * wd
    dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) / sd
    return y, dx, (gy * xh).sum(0), gy.sum(0), mean, sd, xh


def _inputs(rows, width, dtype, wdtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, width, generator=g) * 1.5 + 0.7).to(dtype).to(dev)
    w = (1 + 0.2 * torch.randn(width, generator=g)).to(wdtype).to(dev)
    b = (0.3 * torch.randn(width, generator=g)).to(wdtype).to(dev)
    gy = torch.randn(rows, width, generator=g).to(dtype).to(dev)
    return x, w, b, gy


def _check(got, want, tol, dtype, what):
    got, want = got.detach().double(), want.double()
    lim = tol + HALF[dtype] * want.abs() * (1 + 2.0 ** -7) + TINY[dtype]
    bad = (got - want).abs() > lim
    assert not bool(bad.any()), "%s: %d values off, worst %.3g of its limit" % (
        what, int(bad.sum()), float(((got - want).abs() / lim.clamp_min(1e-300)).max()))


def _limits(x, w, gy, mean, sd, xh):
    """The bounds of the module's docstring, per row (y, dx) and per column (dw, db)."""
    xd, rows = x.double(), x.shape[0]
    exh = K * U * ((xd.abs().amax(1, keepdim=True) + (xd - mean).abs().amax(1, keepdim=True)) / sd + 1)
    wmax = w.double().abs().max() if w is not None else torch.tensor(1.0, dtype=torch.float64, device=x.device)
    g = gy.double().abs().amax(1, keepdim=True) * wmax
    xm = xh.abs().amax(1, keepdim=True)
    # dx = (g - s1 - xh s2) / sd with |s1| <= g, |s2| <= g (mean |xh| <= 1): every factor's error once
    edx = g / sd * (K * U * (2 + 2 * xm) + exh * (2 + 2 * xm))
    depth = min(rows, 192) + 20
    edw = depth * U * (gy.double().abs() * xh.abs()).sum(0) + (gy.double().abs() * exh).sum(0)
    edb = depth * U * gy.double().abs().sum(0)
    return exh * wmax + 4 * U, edx, edw, edb


@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float32)])
def test_layer_norm_and_its_gradients(dev, rows, width, dtype, wdtype):
    from glenet_amd.norm import layer_norm
    x, w, b, gy = _inputs(rows, width, dtype, wdtype, rows * 7 + width, dev)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = layer_norm(x, w, b, 1e-3)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), gy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == db.dtype == wdtype
    with torch.no_grad():
        ry, rdx, rdw, rdb, mean, sd, xh = _formula(x, w, b, gy, 1e-3)
        ey, edx, edw, edb = _limits(x, w, gy, mean, sd, xh)
        _check(y, ry, ey + HALF[torch.float32] * ry.abs(), dtype, "y")
        _check(dx, rdx, edx, dtype, "dx")
        _check(dw, rdw, edw, wdtype, "dw")
        _check(db, rdb, edb, wdtype, "db")
        again = layer_norm(x, w, b, 1e-3)
    assert torch.equal(again, y)
    y2 = layer_norm(x, w, b, 1e-3)
    for p, q in zip(torch.autograd.grad(y2, (x, w, b), gy), (dx, dw, db)):
        assert torch.equal(p, q)                                       # fixed summation orders


def test_layer_norm_gradients_equal_differences(dev):
    """The gradients of a scalar against central differences of the FORMULA's forward in 64 bits."""
    from glenet_amd.norm import layer_norm
    x, w, b, gy = _inputs(3, 7, torch.float32, torch.float32, 5, dev)
    for t in (x, w, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(layer_norm(x, w, b, 1e-2), (x, w, b), gy)
    with torch.no_grad():
        def value(xx, ww, bb):
            return float((_formula(xx, ww, bb, gy, 1e-2)[0] * gy.double()).sum())
        args = [t.detach().double() for t in (x, w, b)]
        h = 1e-5
        for k, g in enumerate(grads):
            for e in range(args[k].numel()):
                up, down = [a.clone() for a in args], [a.clone() for a in args]
                up[k].view(-1)[e] += h
                down[k].view(-1)[e] -= h
                want = (value(*up) - value(*down)) / (2 * h)
                # differences: h^2 times a third derivative of order 10, and 2^-53 / h; the kernel: K u times terms of order 10
                assert abs(float(g.view(-1)[e]) - want) < 10 * h * h * 10 + 1e-9 + 10 * K * U


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_weight_or_bias(dev, weight, bias):
    from glenet_amd.norm import layer_norm
    x, w, b, gy = _inputs(37, 130, torch.float32, torch.float32, 3, dev)
    w, b = (w if weight else None), (b if bias else None)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = layer_norm(x, w, b)
    grads = dict(zip([n for n, t in (("x", x), ("w", w), ("b", b)) if t is not None], torch.autograd.grad(y, leaves, gy)))
    with torch.no_grad():
        ry, rdx, rdw, rdb, mean, sd, xh = _formula(x, w, b, gy, 1e-5)
        ey, edx, edw, edb = _limits(x, w, gy, mean, sd, xh)
        _check(y, ry, ey + U * ry.abs(), torch.float32, "y")
        _check(grads["x"], rdx, edx, torch.float32, "dx")
        if weight:
            _check(grads["w"], rdw, edw, torch.float32, "dw")
        if bias:
            _check(grads["b"], rdb, edb, torch.float32, "db")


def test_layer_norm_of_strided_and_expanded_tensors(dev):
    """Rows apart, transposed tensors, a 3-D batch, a broadcast gradient (strides 0), one gradient alone."""
    from glenet_amd.norm import layer_norm
    g = torch.Generator().manual_seed(2)
    big = torch.randn(50, 3, 96, generator=g).to(dev)
    w = torch.randn(96, generator=g).to(dev)
    for x in (big[:, 1, :], big.transpose(0, 1), big[::2, 2], big[:, 0, :].t().contiguous().t(), big[0, 0], big[:, :, 1:97 - 1 + 1]):
        ww = w if x.shape[-1] == 96 else w[:x.shape[-1]]
        got = layer_norm(x, ww, None)
        assert torch.equal(got, layer_norm(x.contiguous().clone(), ww.contiguous(), None)) and got.shape == x.shape
    x = big[:, 1, :].detach().requires_grad_(True)
    dx, = torch.autograd.grad(layer_norm(x, w, None).sum(), x)
    x2 = x.detach().clone().requires_grad_(True)
    dx2, = torch.autograd.grad(layer_norm(x2, w, None), x2, torch.ones(50, 96, device=dev))
    assert torch.equal(dx, dx2)
    wl = w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(layer_norm(x.detach(), wl, None).sum(), wl)
    assert dw.shape == wl.shape


def test_layer_norm_of_nothing_and_of_broken_rows(dev):
    from glenet_amd.norm import layer_norm
    x = torch.zeros(0, 40, device=dev, requires_grad=True)
    w = torch.ones(40, device=dev, requires_grad=True)
    b = torch.zeros(40, device=dev, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == (0, 40) and dx.shape == (0, 40) and not bool(dw.any()) and not bool(db.any())
    x = torch.randn(6, 33, device=dev)
    want = layer_norm(x, None, None)
    x2 = x.clone()
    x2[2, 5] = float("nan")
    x2[4, 0] = float("inf")
    got = layer_norm(x2, None, None)
    for r in range(6):                                # a broken row breaks itself alone
        if r in (2, 4):
            assert bool(torch.isnan(got[r]).any())
        else:
            assert torch.equal(got[r], want[r])
    const = layer_norm(torch.full((3, 100), 7.25, device=dev), None, None)
    assert not bool(const.any())


def test_layer_norm_in_a_captured_graph_beside_eager_work(dev):
    """Forward + backward recorded into a graph, replayed with new inputs and eager calls between the replays."""
    from glenet_amd import _lib
    from glenet_amd.norm import layer_norm
    x, w, b, gy = _inputs(200, 192, torch.float32, torch.float32, 9, dev)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step():
        y = layer_norm(x, w, b)
        return [y] + list(torch.autograd.grad(y, leaves, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = _lib.new_graph()
    with torch.cuda.graph(graph):
        out = step()
    for it in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(200, 192, device=dev) * (it + 1))
            gy.copy_(torch.randn(200, 192, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q)


def test_layer_norm_module(dev):
    from glenet_amd.norm import LayerNorm
    m = LayerNorm(48).to(dev)
    x = torch.randn(4, 5, 48, device=dev)
    y = m(x)
    y.square().mean().backward()
    assert m.weight.grad.shape == (48,) and m.bias.grad.shape == (48,)
    assert float((y.detach().mean(-1)).abs().max()) < 1e-5
    with pytest.raises(ValueError):
        m(torch.randn(4, 47, device=dev))


def test_gradients_are_not_differentiated_again(dev):
    """Asking for a second derivative says so; a first one under create_graph is what it was."""
    from glenet_amd.attention import cross_attention
    from glenet_amd.norm import layer_norm
    x = torch.randn(5, 1, 24, device=dev, requires_grad=True)
    cnt = torch.tensor([5], dtype=torch.int32, device=dev)
    for f in (lambda: layer_norm(x), lambda: cross_attention(x, x, x, cnt, cnt)):
        want, = torch.autograd.grad(f().square().sum(), x)
        got, = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        assert torch.equal(want, got)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(got.sum(), x)
