"""glenet_amd.optim.orthogonalize (csrc/glx_orthogonal.hip) against the definition in 64 bits, and FlatMuon against the update's
formulas in 64 bits.

Tolerance of the orthogonaliser, relative in the Frobenius norm.  A step maps a singular value s to s p(s^2), slope at most
a = 3.4445 (at 0), so what is lost in X_0 grows by at most a^5 = 485 in five steps; operands are held to 2^-22, products of them
to 2^-21 with the sum's rounding, and a step adds no more: 4 x 485 x 2^-22.  bfloat16 runs its five steps on one Gram matrix,
whose perturbations grow by a^2 per step: a^8 2^-22 = 5e-3.  A result of fewer bits adds half a step of its type."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

COEFFS = (3.4445, -4.7750, 2.0315)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LIMIT = {torch.float32: 4 * 485 * 2.0 ** -22, torch.float16: 4 * 485 * 2.0 ** -22, torch.bfloat16: 3.4445 ** 8 * 2.0 ** -22}
SHAPES = [(1, 1), (1, 9), (9, 1), (5, 3), (16, 700), (32, 32), (64, 64), (65, 64), (100, 300), (128, 128), (1000, 128), (129, 129),
          (130, 900), (190, 200), (256, 1111), (700, 700), (40, 5001), (2100, 2100), (2500, 2060)]


def _exact(m, steps=5, coeffs=COEFFS, eps=1e-7):
    x = m.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + eps)
    a, b, c = coeffs
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if tall else x


def _gradient(r, c, seed, dev, dtype=torch.float32, size=1e-2):
    """Errors x activations over a batch of samples, channels of unequal scale: a spectrum over several powers of ten."""
    g = torch.Generator().manual_seed(seed)
    s = max(8, min(r, c))
    e = torch.randn(s, r, generator=g) * torch.exp(torch.randn(r, generator=g))
    a = torch.randn(s, c, generator=g) * torch.exp(torch.randn(c, generator=g))
    return (e.to(dev).t() @ a.to(dev) * (size / s)).to(dtype)


def _off(got, want):
    return float((got.double() - want).norm() / want.norm().clamp_min(1e-300))


@pytest.mark.parametrize("r,c", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_orthogonalize(dev, r, c, dtype):
    from glenet_amd.optim import orthogonalize
    m = _gradient(r, c, r * 31 + c, dev, dtype)
    keep = m.clone()
    o = orthogonalize(m)
    assert o.shape == m.shape and o.dtype == dtype and torch.equal(m, keep)
    assert _off(o, _exact(m)) < LIMIT[dtype] + HALF[dtype]
    assert torch.equal(o, orthogonalize(m))


def test_a_list_gives_what_its_matrices_give_alone(dev):
    from glenet_amd.optim import orthogonalize
    mats = [_gradient(r, c, i, dev) for i, (r, c) in enumerate(SHAPES[:16] * 4)]            # more than one launch's table
    outs = orthogonalize(mats)
    assert isinstance(outs, list)
    for m, o in zip(mats, outs):
        assert torch.equal(o, orthogonalize(m))
    batch = torch.stack([_gradient(48, 80, i, dev) for i in range(6)]).view(2, 3, 48, 80)
    got = orthogonalize(batch)
    assert got.shape == batch.shape and torch.equal(got[1, 2], orthogonalize(batch[1, 2]))
    assert orthogonalize(batch[:0]).shape == (0, 3, 48, 80)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 7, 12])
@pytest.mark.parametrize("shape", [(96, 200), (160, 400), (150, 150)])
def test_other_numbers_of_steps(dev, steps, shape):
    """a^steps instead of a^5; from eight steps on the singular values have arrived and the growth has ended."""
    from glenet_amd.optim import orthogonalize
    m = _gradient(*shape, steps, dev)
    limit = 4 * 3.4445 ** min(steps, 7) * 2.0 ** -22 * max(1, steps)
    assert _off(orthogonalize(m, steps=steps), _exact(m, steps)) < limit


def test_other_coefficients(dev):
    from glenet_amd.optim import orthogonalize
    m = _gradient(140, 300, 3, dev)
    for coeffs in ((1.875, -1.25, 0.375), (1.5, -0.5, 0.0), (1.0, 0.0, 0.0)):
        assert _off(orthogonalize(m, coefficients=coeffs), _exact(m, 5, coeffs)) < LIMIT[torch.float32]
    # T_5(0.9 x), the steepest that maps [0, 1] into itself: five steps raise what is lost in X_0 by at most (max |f'|) ^ 5,
    # |f'| = 4.5 |U_4(0.9 x)| <= 8.1 (at x = 1; 4.5 at 0, 4.5 * 1.25 between)
    steep = (4.5, -14.58, 9.44784)
    for dtype in (torch.float32, torch.bfloat16):
        g = _gradient(140, 900, 4, dev, dtype)
        assert _off(orthogonalize(g, coefficients=steep), _exact(g, 5, steep)) < 4 * 8.1 ** 5 * 2.0 ** -22 + HALF[dtype]
    o = orthogonalize(torch.randn(200, 260, device=dev), steps=30, coefficients=(1.875, -1.25, 0.375)).double()
    assert float((o @ o.t() - torch.eye(200, device=dev, dtype=torch.float64)).abs().max()) < 200 * 2.0 ** -21


@pytest.mark.parametrize("size", [1e30, 1e12, 1e-6, 1e-9, 1e-14, 1e-25])
def test_matrices_of_any_size(dev, size):
    """The norm neither overflows nor loses a gradient far below eps (which the formula then divides by)."""
    from glenet_amd.optim import orthogonalize
    for shape in ((60, 90), (150, 400), (200, 200)):
        m = _gradient(*shape, 1, dev) * size
        assert _off(orthogonalize(m), _exact(m)) < LIMIT[torch.float32], shape


def test_zero_and_broken_matrices(dev):
    from glenet_amd.optim import orthogonalize
    good = _gradient(70, 50, 2, dev)
    bad = good.clone()
    bad[3, 4] = float("nan")
    inf = _gradient(150, 300, 2, dev)
    inf[0, 0] = float("inf")
    zero, one, z, n, i, g2 = orthogonalize([torch.zeros(200, 300, device=dev), torch.zeros(1, 1, device=dev),
                                            torch.zeros(30, 20, device=dev), bad, inf, good])
    assert not bool(zero.any()) and not bool(one.any()) and not bool(z.any())
    assert bool(torch.isnan(n).any()) and bool(torch.isnan(i).any())
    assert torch.equal(g2, orthogonalize(good))


def test_strided_matrices_and_another_stream(dev):
    from glenet_amd.optim import orthogonalize
    big = _gradient(300, 500, 4, dev)
    want = orthogonalize(big[10:110, 20:90].contiguous())
    assert torch.equal(orthogonalize(big[10:110, 20:90]), want)
    assert torch.equal(orthogonalize(big[:, 3:4]), orthogonalize(big[:, 3:4].contiguous()))
    assert torch.equal(orthogonalize(big.t()[20:90, 10:110]), orthogonalize(big.t()[20:90, 10:110].contiguous()))
    assert torch.equal(orthogonalize(big[:1].expand(40, 500)), orthogonalize(big[:1].expand(40, 500).contiguous()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = orthogonalize(big[10:110, 20:90])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want)
    m = big.clone().requires_grad_(True)
    assert not orthogonalize(m).requires_grad


def test_orthogonalize_in_two_captured_graphs(dev):
    """Each graph has its own workspace: replayed in turn and beside eager calls they keep their results."""
    from glenet_amd import _lib
    from glenet_amd.optim import orthogonalize
    a, b = [_gradient(90, 140, 1, dev), _gradient(200, 700, 2, dev)], [_gradient(260, 260, 3, dev)]
    orthogonalize(a), orthogonalize(b)
    graphs = []
    for mats in (a, b):
        g = _lib.new_graph()
        with torch.cuda.graph(g):
            out = orthogonalize(mats)
        graphs.append((g, mats, out))
    for it in range(3):
        for _, mats, _ in graphs:
            for m in mats:
                m.copy_(torch.randn_like(m) * (it + 1))
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, mats, out in graphs:
            for o, w in zip(out, orthogonalize(mats)):
                assert torch.equal(o, w)


# ------------------------------------------------------------------------------------------------ FlatMuon
def _params(dev):
    g = torch.Generator().manual_seed(0)
    shapes = [(64, 33), (7,), (3, 3, 3, 16, 32), (1,), (256, 324), (1, 256), (40, 24, 1)]
    ps = [torch.nn.Parameter((torch.randn(s, generator=g) * 0.3).to(dev)) for s in shapes]
    return ps + [torch.nn.Parameter((torch.randn(s, generator=g) * 0.3).to(dev).contiguous(memory_format=torch.channels_last))
                 for s in [(32, 16, 3, 3), (8, 16, 1, 1)]]


def _memory(t):
    """A parameter's elements in memory order, as its matrix."""
    if t.dim() == 4:
        t = t.permute(0, 2, 3, 1)
    return t.reshape(-1, t.shape[-1]) if t.dim() == 5 else t.reshape(t.shape[0], -1)


@pytest.mark.parametrize("max_norm,lookahead", [(None, True), (0.5, True), (10.0, False)])
def test_flat_muon_steps_as_its_formulas(dev, max_norm, lookahead):
    """Four steps with a moving schedule.  Limits: a matrix' step is lr 0.2 sqrt(max) O with O off by LIMIT (relative in the
    Frobenius norm) and an fp32 rounding of p; the other tensors follow AdamW to a few roundings of p and of the step."""
    from glenet_amd.optim import FlatMuon
    ours = _params(dev)
    opt = FlatMuon(ours, lr=3e-3, betas=(0.9, 0.99), weight_decay=0.01, max_norm=max_norm, lookahead=lookahead)
    assert [s is not None for s in opt.matrix_shapes] == [True, False, True, False, True, False, True, True, True]
    assert opt.matrix_shapes[2] == (432, 32) and opt.matrix_shapes[7] == (32, 144)
    ref = [p.detach().double().clone() for p in ours]
    m1, m2 = [torch.zeros_like(r) for r in ref], [torch.zeros_like(r) for r in ref]
    slack = [0.0] * len(ref)
    g = torch.Generator(device=dev).manual_seed(1)
    for it in range(4):
        lr, b1 = 3e-3 * (1 + it), 0.9 - 0.01 * it
        opt.set_lr(lr, b1)
        grads = [torch.randn(p.shape, device=dev, generator=g) * 0.1 for p in ours]
        for p, gr in zip(ours, grads):
            p.grad = gr.clone()
        opt.step()
        norm = math.sqrt(sum(float((gr.double() ** 2).sum()) for gr in grads))
        assert abs(float(opt.grad_norm) / norm - 1) < 1e-6
        coef = min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0
        for i, (gr, rc) in enumerate(zip(grads, opt.matrix_shapes)):
            gd = gr.double() * coef
            m1[i] = m1[i] + (gd - m1[i]) * (1 - b1)
            if rc is not None:
                u = gd + (m1[i] - gd) * b1 if lookahead else m1[i]
                o = _exact(_memory(u))
                shape = (ref[i].permute(0, 2, 3, 1) if ref[i].dim() == 4 else ref[i]).shape
                o = o.reshape(shape)
                o = o.permute(0, 3, 1, 2) if ref[i].dim() == 4 else o
                size = lr * 0.2 * math.sqrt(max(rc))
                ref[i] = ref[i] * (1 - lr * 0.01) - size * o
                # (u itself carries fp32 roundings, which the steps amplify like those of X_0)
                slack[i] += size * (LIMIT[torch.float32] + 485 * 4 * 2.0 ** -24) * float(o.norm())
            else:
                m2[i] = m2[i] * 0.99 + gd * gd * 0.01
                ref[i] = ref[i] * (1 - lr * 0.01) - lr / (1 - b1 ** (it + 1)) * m1[i] / ((m2[i] / (1 - 0.99 ** (it + 1))).sqrt() + 1e-8)
                # step sizes of order lr; powf and the moments to ~2^-18 of it
                slack[i] += 4 * lr * 2.0 ** -18 * math.sqrt(ref[i].numel())
            slack[i] += 4 * 2.0 ** -24 * float(ref[i].norm())
        for i, p in enumerate(ours):
            assert float((p.detach().double() - ref[i]).norm()) < slack[i], (it, i)
    assert int(opt.step_count) == 4
    sd = opt.state_dict()
    again = FlatMuon(_params(dev))
    again.load_state_dict(sd)
    assert torch.equal(again.exp_avg, opt.exp_avg) and int(again.step_count) == 4


def test_flat_muon_shapes_are_the_callers_to_choose(dev):
    from glenet_amd.optim import FlatMuon
    ps = _params(dev)
    opt = FlatMuon(ps, shapes={ps[0]: None, ps[4]: (324, 256)})
    assert opt.matrix_shapes[0] is None and opt.matrix_shapes[4] == (324, 256)
    with pytest.raises(ValueError):
        FlatMuon(ps, shapes={ps[0]: (3, 5)})
    only = [torch.nn.Parameter(torch.randn(5, device=dev))]
    opt = FlatMuon(only, lr=0.1)
    only[0].grad = torch.ones(5, device=dev)
    before = only[0].detach().clone()
    opt.step()                                                   # no matrix at all: AdamW
    assert bool((only[0].detach() < before).all())


def test_flat_muon_in_a_captured_graph(dev):
    from glenet_amd import _lib
    from glenet_amd.optim import FlatMuon
    a, b = _params(dev), _params(dev)
    oa, ob = FlatMuon(a, lr=1e-2), FlatMuon(b, lr=1e-2)
    graph = _lib.new_graph()
    with torch.cuda.graph(graph):
        oa.step(packed=True)
    for it in range(4):
        gr = torch.randn(oa.n, device=dev)
        oa.flat_grad.copy_(gr)
        ob.flat_grad.copy_(gr)
        oa.set_lr(1e-2 / (it + 1), 0.9)
        ob.set_lr(1e-2 / (it + 1), 0.9)
        graph.replay()
        torch.cuda.synchronize()
        ob.step(packed=True)
        torch.cuda.synchronize()
        assert torch.equal(oa.flat_param, ob.flat_param) and torch.equal(oa.exp_avg, ob.exp_avg)


def test_the_training_step_takes_flat_muon(dev):
    """glenet_vr.StaticTrainStep(optimizer=FlatMuon(...)): recorded, replayed, parameters move and stay finite."""
    from glenet_amd import glenet_vr as gvr
    from glenet_amd.optim import FlatMuon
    from test_train_step_gpu import JIT, _batch, _small_model
    model = _small_model(dev)
    pts, bidx, gt, unc = _batch(dev, [52, 53], 6000)
    opt = FlatMuon(model.parameters(), lr=1e-3, max_norm=10.0)
    pipe = gvr.StaticTrainStep(model, 2, pts.shape[0] + 700, max_gt=gt.shape[1], optimizer=opt, seed_rois_with_gt=JIT)
    pipe.calibrate(pts, bidx)
    pipe.load(pts, bidx, gt, unc)
    pipe.step()
    torch.cuda.synchronize()
    pipe.check()
    pipe.capture()
    before = opt.flat_param.clone()
    for _ in range(3):
        pipe.step()
    torch.cuda.synchronize()
    pipe.check()
    moved = (opt.flat_param - before).abs()
    assert bool(torch.isfinite(opt.flat_param).all()) and float(moved.max()) > 0
    pipe.step()
    torch.cuda.synchronize()
    # the step that was just replayed, again from its inputs: momentum, gradients and parameters of the recorded update
    want = opt.exp_avg.clone()
    p0 = opt.flat_param.clone()
    opt.step(packed=True)
    torch.cuda.synchronize()
    assert int(opt.step_count) == 6 and not torch.equal(want, opt.exp_avg) and not torch.equal(p0, opt.flat_param)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (2, 2), (3, 801), (801, 3), (4, 4), (16, 16), (16, 17), (15, 64), (16, 8192), (8192, 16), (16, 8193)])
def test_few_rows(dev, shape, dtype):
    """Up to 16 x 8192 all arithmetic is in 64 bits: the result's rounding, and its step through fp32, are all that is left."""
    from glenet_amd.optim import orthogonalize
    g = _gradient(*shape, 5, dev, dtype)
    wide = torch.full((shape[0] + 2, shape[1] + 3), float("nan"), device=dev, dtype=dtype)
    wide[1:-1, 1:-2] = g
    o, want = orthogonalize(wide[1:-1, 1:-2]), _exact(g)
    if max(shape) <= 8192:
        assert bool(((o.double() - want).abs() <= (HALF[dtype] + 2.0 ** -23) * want.abs() + (6e-8 if dtype == torch.float16 else 1e-30)).all())
        for steps in (1, 12):
            assert _off(orthogonalize(g, steps=steps), _exact(g, steps)) < HALF[dtype] + 2.0 ** -23
    else:
        assert _off(o, want) < LIMIT[dtype] + HALF[dtype]
    zero = torch.zeros(shape, device=dev, dtype=dtype)
    assert not orthogonalize([zero, g])[0].any()
    assert torch.equal(orthogonalize([zero, g, torch.cat([g, g])])[1], orthogonalize(g))


def test_a_matrix_of_few_rows_may_be_overwritten(dev):
    from glenet_amd.optim import _check_steps, _orthogonalize
    steps, coeffs, eps = _check_steps("test", 5, COEFFS, 1e-7)
    for shape in ((16, 1500), (700, 9), (40, 300)):
        g = _gradient(*shape, 8, dev)
        want, buf = _exact(g), g.clone()
        _orthogonalize([buf], steps, coeffs, eps, [buf])
        assert _off(buf, want) < LIMIT[torch.float32]


def test_a_list_beyond_one_workspace_runs_in_groups(dev):
    """17 matrices of 2100 x 2100 need more than 1 GiB side by side; between them small and wide ones, in place and not."""
    from glenet_amd import _lib
    from glenet_amd.optim import _Matrix, _check_steps, _orthogonalize, orthogonalize
    shapes = ([(2100, 2100)] * 5 + [(12, 300), (150, 900)]) * 3 + [(2100, 2100)] * 2
    mats = [_gradient(r, c, i, dev) for i, (r, c) in enumerate(shapes)]
    table = (_Matrix * len(shapes))(*[_Matrix(64, 64, c, c, r, c) for r, c in shapes])
    one = _lib.query("glx_orthogonalize_workspace_bytes", (_Matrix * 1)(_Matrix(64, 64, 2100, 2100, 2100, 2100)), 1, 0, 5)
    assert _lib.query("glx_orthogonalize_workspace_bytes", table, len(shapes), 0, 5) <= 1 << 30 < 17 * one
    alone = [orthogonalize(m) for m in mats]
    for got in (orthogonalize(mats), orthogonalize(mats)):
        assert all(torch.equal(a, b) for a, b in zip(got, alone))
    steps, coeffs, eps = _check_steps("test", 5, COEFFS, 1e-7)
    _orthogonalize(mats, steps, coeffs, eps, mats)
    assert all(torch.equal(a, b) for a, b in zip(mats, alone))


@pytest.mark.parametrize("size", [1e-27, 1e-30, 1e-33, 1e-35])
def test_gradients_that_vanish_beside_eps(dev, size):
    """A = X X^T is below 2^-100 there and a step multiplies X by 3.4445: five products of operands of 22 bits, each off by two
    operands' 2^-22 and the sum's 2^-24, and the division.  Without eps the result does not depend on the size."""
    from glenet_amd.optim import orthogonalize
    for shape in ((60, 90), (150, 400), (900, 150), (200, 200)):
        m = _gradient(*shape, 1, dev) * size
        off = _off(orthogonalize(m), _exact(m))
        assert off < 5 * (2 * 2.0 ** -22 + 2.0 ** -24) + 2.0 ** -22, shape
        assert _off(orthogonalize(m, eps=0.0), _exact(m, eps=0.0)) < LIMIT[torch.float32], shape
