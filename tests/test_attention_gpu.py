"""glenet_amd.attention.cross_attention (csrc/glx_attention.hip, glx_attention_bwd.hip) against the formulas in 64 bits.

Tolerances, computed per output element from the inputs (u = 2^-24, h = half a step of the inputs' type, 2^-24 for fp32):
  a product over D terms is off by (D + 8) u sum |terms|; a score s in base 2 by es = that + 4 u |s|, a probability by a relative
  ep = 2 es + 16 u + the row's own sum (depth N: N u).
  O:  (2 ep + N u + h) sum p |v| + h |O|            (h: p rounded in front of its product; the second one: the result)
  dP, delta: (D + 8) u sum |terms|, delta also h sum |dO O| (from the rounded O);  dS: eds = p (edp + edelta) + (ep + h) |dS|
  dQ: scale (sum eds |k| + N u sum |dS k|) + h |dQ|, dK alike over the M rows, dV: sum (ep + h + M u) p |dO| + h |dV|
  fp16: p below 2^-14 of its scale loses up to 2^-25: + 2^-25 sum |v| / l forward; backward P carries 2^12, dS 2^8 over a tile's
  largest value: + 2^-24 max |dS| sum |k|.  Nothing below half a subnormal step of the result's type is asked for."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUB = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}

# q lengths, k lengths, heads, key heads, dim, mask, padded
CASES = [
    ([1], [1], 1, 1, 8, False, True),
    ([1, 1], [7, 7], 4, 2, 16, True, True),
    ([1, 1, 1], [2000, 2000, 2000], 8, 2, 64, False, True),
    ([33, 33], [65, 65], 3, 3, 40, True, True),
    ([130], [300], 2, 1, 128, False, True),
    ([5, 0, 200, 17], [64, 90, 0, 1301], 4, 4, 32, False, False),
    ([64, 1, 129], [63, 257, 128], 6, 2, 72, True, False),
    ([31, 100], [1, 2], 7, 1, 20, False, False),
    ([300], [500], 2, 2, 100, True, False),
    ([4, 4], [3000, 900], 2, 1, 96, True, False),
    ([700, 650], [40, 33], 4, 2, 64, False, False),
    ([9, 3], [50, 70], 3, 1, 1, False, False),
    ([50, 37], [140, 260], 6, 2, 32, True, False),             # three heads share one: tiles hold whole queries
    ([3, 7], [200, 31], 70, 1, 16, False, False),              # more heads share one than a tile has rows
    ([1], [129], 128, 2, 128, False, True),
]


def _frames(ql, kl):
    q0 = k0 = 0
    for a, b in zip(ql, kl):
        yield q0, a, k0, b
        q0, k0 = q0 + a, k0 + b


def _inputs(case, dtype, seed, dev, tail=0):
    ql, kl, h, hk, d, masked, padded = case
    g = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g).to(dtype).to(dev)

    q, k, v, go = normal(sum(ql) + tail, h, d), normal(sum(kl) + tail, hk, d), normal(sum(kl) + tail, hk, d), normal(sum(ql) + tail, h, d)
    mask = None
    if masked:
        mask = (torch.rand(sum(kl) + tail, generator=g) < 0.7).to(dev)
        mask[:kl[0]] = False                                  # a frame without a state
        if len(kl) > 1 and kl[1] > 2:
            mask[kl[0]:kl[0] + kl[1]] = False
            mask[kl[0] + kl[1] - 1] = True                    # one state, the last
    cnts = None
    if padded:
        b = len(ql)
        q, go = q.view(b, -1, h, d), go.view(b, -1, h, d)
        k, v = k.view(b, -1, hk, d), v.view(b, -1, hk, d)
        mask = mask.view(b, -1) if mask is not None else None
    else:
        cnts = tuple(torch.tensor(x, dtype=torch.int32, device=dev) for x in (ql, kl))
    return q, k, v, go, mask, cnts


def _reference(q, k, v, go, mask, case, dtype, scale=None):
    """{name: (value, limit)} in 64 bits, on stacked rows."""
    ql, kl, h, hk, d, _, _ = case
    q, go = (t.detach().reshape(-1, h, d).double() for t in (q, go))
    k, v = (t.detach().reshape(-1, hk, d).double() for t in (k, v))
    mask = mask.reshape(-1) if mask is not None else torch.ones(k.shape[0], dtype=torch.bool, device=q.device)
    scale = 1 / math.sqrt(d) if scale is None else scale
    h_ = HALF[dtype]
    fp16 = dtype == torch.float16
    out = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    for q0, lq, k0, lk in _frames(ql, kl):
        live = torch.arange(k0, k0 + lk, device=q.device)[mask[k0:k0 + lk]]
        if lq == 0 or live.numel() == 0:
            continue
        n = live.numel()
        for j in range(h):
            jk = j // (h // hk)
            qq, gg, kk, vv = q[q0:q0 + lq, j], go[q0:q0 + lq, j], k[live, jk], v[live, jk]
            s = qq @ kk.t() * scale
            p = torch.softmax(s, 1)
            o = p @ vv
            dp = gg @ vv.t()
            de = (gg * o).sum(1, keepdim=True)
            ds = p * (dp - de)
            es = ((d + 8) * U * (qq.abs() @ kk.abs().t()) * abs(scale) + 4 * U * s.abs()).amax(1, keepdim=True) * 1.5
            ep = 2 * es + (16 + n) * U
            tiny = 2.0 ** -25 * vv.abs().sum(0) if fp16 else 0.0
            eo = (2 * ep + n * U + h_) * (p @ vv.abs()) + tiny
            edp = (d + 8) * U * (gg.abs() @ vv.abs().t())
            ede = (gg.abs() * ((d + 8) * U * o.abs() + eo + h_ * o.abs())).sum(1, keepdim=True)
            eds = p * (edp + ede) + (ep + h_) * ds.abs()
            if fp16:
                eds = eds + 2.0 ** -24 * ds.abs().max()
            out["o"][0][q0:q0 + lq, j] = o
            out["o"][1][q0:q0 + lq, j] = eo
            out["dq"][0][q0:q0 + lq, j] = scale * ds @ kk
            out["dq"][1][q0:q0 + lq, j] = abs(scale) * (eds @ kk.abs() + n * U * (ds.abs() @ kk.abs()))
            out["dk"][0][live, jk] += scale * ds.t() @ qq
            out["dk"][1][live, jk] += abs(scale) * (eds.t() @ qq.abs() + h * lq * U * (ds.abs().t() @ qq.abs()))
            out["dv"][0][live, jk] += p.t() @ gg
            out["dv"][1][live, jk] += ((ep + h_ + h * lq * U) * p).t() @ gg.abs() + (2.0 ** -37 * gg.abs().sum(0) if fp16 else 0.0)
    return out


def _check(got, ref, name, dtype):
    want, lim = ref[name]
    got = got.detach().reshape(want.shape).double()
    lim = lim + HALF[dtype] * want.abs() + SUB[dtype]
    off = (got - want).abs()
    assert bool((off <= lim).all()), "%s: %d of %d off, worst %.3g of its limit, nan %d" % (
        name, int((~(off <= lim)).sum()), off.numel(), float((off / lim).nan_to_num(0).max()), int(torch.isnan(got).sum()))


def _run(q, k, v, go, mask, cnts, **kw):
    from glenet_amd.attention import cross_attention
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    a = cnts if cnts is not None else (None, None)
    o = cross_attention(*leaves, *a, key_mask=mask, **kw)
    return [o] + list(torch.autograd.grad(o, leaves, go))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("index", range(len(CASES)))
def test_cross_attention_and_its_gradients(dev, index, dtype):
    from glenet_amd.attention import cross_attention
    case = CASES[index]
    q, k, v, go, mask, cnts = _inputs(case, dtype, index, dev)
    outs = _run(q, k, v, go, mask, cnts)
    ref = _reference(q, k, v, go, mask, case, dtype)
    for t, n, like in zip(outs, ("o", "dq", "dk", "dv"), (q, q, k, v)):
        assert t.shape == like.shape and t.dtype == dtype
        _check(t, ref, n, dtype)
    a = cnts if cnts is not None else (None, None)
    assert torch.equal(cross_attention(q, k, v, *a, key_mask=mask), outs[0])            # the inference call
    for x, y in zip(_run(q, k, v, go, mask, cnts), outs):
        assert torch.equal(x, y)                                                       # fixed summation orders


def test_cross_attention_gradients_equal_differences(dev):
    """Central differences of the 64-bit formula; truncation h^2 of a third derivative of order 10, the kernel ~1e-5."""
    case = ([3], [5], 2, 1, 4, False, False)
    q, k, v, go, mask, cnts = _inputs(case, torch.float32, 1, dev)
    grads = _run(q, k, v, go, mask, cnts)[1:]

    def value(q, k, v):
        s = torch.einsum("mhd,nd->hmn", q, k[:, 0]) / 2.0
        return float((torch.einsum("hmn,nd->mhd", torch.softmax(s, 2), v[:, 0]) * go.double()).sum())

    base = [t.double() for t in (q, k, v)]
    h = 1e-5
    for i, g in enumerate(grads):
        for e in range(0, base[i].numel(), 3):
            up, down = [t.clone() for t in base], [t.clone() for t in base]
            up[i].view(-1)[e] += h
            down[i].view(-1)[e] -= h
            assert abs(float(g.reshape(-1)[e]) - (value(*up) - value(*down)) / (2 * h)) < 2e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_what_masked_and_trailing_states_hold_does_not_matter(dev, dtype):
    """NaN, infinities and the type's lowest value in masked states and behind the last frame; trailing queries give zeros."""
    case = ([40, 21], [90, 133], 4, 2, 48, True, False)
    q, k, v, go, mask, cnts = _inputs(case, dtype, 3, dev, tail=9)
    want = _run(q, k, v, go, mask, cnts)
    k2, v2, q2, go2 = k.clone(), v.clone(), q.clone(), go.clone()
    dead = torch.nonzero(~mask).flatten()
    for i, bad in enumerate((float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min)):
        k2[dead[i::4]] = bad
        v2[dead[i::4]] = bad
    k2[-9:], v2[-9:], q2[-9:] = float("nan"), float("inf"), float("nan")
    go2[-9:] = float("nan")
    got = _run(q2, k2, v2, go2, mask, cnts)
    for w, g in zip(want, got):
        assert torch.equal(w, g)
    o, dq, dk, dv = got
    for t in (o[-9:], dq[-9:], dk[-9:], dv[-9:], dk[dead], dv[dead], o[:40], dq[:40]):
        assert not bool(t.any())
    # an unmasked broken state breaks its own frame alone
    k3 = k.clone()
    k3[90 + 132, 0] = float("nan")
    assert bool(mask[90 + 132])
    o3 = _run(q, k3, v, go, mask, cnts)[0]
    assert torch.equal(o3[:40], want[0][:40]) and bool(torch.isnan(o3[40:61, :2]).all()) and torch.equal(o3[:, 2:], want[0][:, 2:])


def test_large_scores_and_equal_scores(dev):
    """Scores of +-1e4: the maximum is taken out before the exponential; equal scores give the mean."""
    from glenet_amd.attention import cross_attention
    q = torch.zeros(1, 2, 1, 8, device=dev)
    q[0, 0] = 100.0
    k = torch.randn(1, 700, 1, 8, device=dev) * 30
    v = torch.randn(1, 700, 1, 8, device=dev)
    o = cross_attention(q, k, v, scale=1.0)
    best = int((k[0, :, 0].double().sum(1)).argmax())
    assert torch.equal(o[0, 0, 0], v[0, best, 0])
    assert float((o[0, 1, 0].double() - v[0, :, 0].double().mean(0)).abs().max()) < 700 * U
    o = cross_attention(q, k, v, scale=0.0)
    assert float((o[0, 0, 0].double() - v[0, :, 0].double().mean(0)).abs().max()) < 700 * U


@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_fp16_gradients_keep_their_range(dev, size):
    """fp16 with a loss scale that puts dS far below or at the edge of fp16's range: both inner products carry their own scale."""
    case = ([70], [900], 2, 1, 64, False, False)
    q, k, v, go, mask, cnts = _inputs(case, torch.float16, 8, dev)
    go = (go.double() * size).clamp(-6e4, 6e4).half()
    outs = _run(q, k, v, go, mask, cnts)
    ref = _reference(q, k, v, go, mask, case, torch.float16)
    for t, n in zip(outs, ("o", "dq", "dk", "dv")):
        _check(t, ref, n, torch.float16)


def test_strides(dev):
    """Views of packed projections, transposed head / row orders, expanded gradients."""
    g = torch.Generator().manual_seed(5)
    kv = torch.randn(2, 50, 2, 3, 32, generator=g).to(dev)                # frames, states, k | v, heads, dim
    qt = torch.randn(2, 6, 20, 32, generator=g).to(dev).transpose(1, 2)   # heads in front of rows
    k, v = kv[:, :, 0], kv[:, :, 1]
    go = torch.randn(2, 20, 6, 32, generator=g).to(dev)
    want = _run(qt.contiguous(), k.contiguous(), v.contiguous(), go, None, None)
    for w, t in zip(want, _run(qt, k, v, go, None, None)):
        assert torch.equal(w, t)
    odd = torch.randn(2, 20, 6, 33, generator=g).to(dev)
    for w, t in zip(_run(odd[..., 1:].contiguous(), k.contiguous(), v.contiguous(), go, None, None), _run(odd[..., 1:], k, v, go, None, None)):
        assert torch.equal(w, t)
    every = qt.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)      # the head dimension strided
    assert torch.equal(_run(every, k, v, go, None, None)[0], want[0])
    one = torch.ones((), device=dev).expand(2, 20, 6, 32)
    for w, t in zip(_run(qt, k, v, one.contiguous(), None, None), _run(qt, k, v, one, None, None)):
        assert torch.equal(w, t)
    cnt = torch.tensor([20, 20], device=dev), torch.tensor([50, 50], device=dev)      # int64 counts, the same frames stacked
    st = _run(qt.reshape(40, 6, 32), k.reshape(100, 3, 32), v.reshape(100, 3, 32), go.reshape(40, 6, 32), None, cnt)
    for w, t in zip(want, st):
        assert torch.equal(w.reshape(t.shape), t)


def test_one_side_needs_a_gradient(dev):
    from glenet_amd.attention import cross_attention
    case = ([40, 30], [60, 80], 4, 2, 32, False, False)
    q, k, v, go, mask, cnts = _inputs(case, torch.float32, 3, dev)
    full = _run(q, k, v, go, mask, cnts)[1:]
    for i in range(3):
        ts = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        g, = torch.autograd.grad(cross_attention(*ts, *cnts), ts[i], go)
        assert torch.equal(g, full[i])


def test_counts_that_do_not_fit_are_cut(dev):
    from glenet_amd.attention import cross_attention
    case = ([10, 20], [30, 40], 2, 1, 16, False, False)
    q, k, v, go, _, cnts = _inputs(case, torch.float32, 3, dev)
    want = _run(q, k, v, go, None, cnts)
    wild = torch.tensor([10, 2 ** 31 - 1], dtype=torch.int32, device=dev), torch.tensor([30, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    for w, t in zip(want, _run(q, k, v, go, None, wild)):
        assert torch.equal(w, t)
    neg = torch.tensor([-5, 10, 20, -1], dtype=torch.int32, device=dev), torch.tensor([-3, 30, 40, 7], dtype=torch.int32, device=dev)
    for w, t in zip(want, _run(q, k, v, go, None, neg)):
        assert torch.equal(w, t)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    for t in _run(q, k, v, go, None, (none, none)):
        assert not bool(t.any())
    many = torch.ones(200, dtype=torch.int32, device=dev)                # more frames than a wave has lanes
    q, k, v = torch.randn(200, 2, 16, device=dev), torch.randn(200, 1, 16, device=dev), torch.randn(200, 1, 16, device=dev)
    o = cross_attention(q, k, v, many, many)
    assert torch.equal(o, v.expand(200, 2, 16))


def test_nothing_on_one_side(dev):
    for ql, kl in ((0, 5), (5, 0), (0, 0)):
        q = torch.randn(2, ql, 4, 16, device=dev)
        k, v = torch.randn(2, kl, 2, 16, device=dev), torch.randn(2, kl, 2, 16, device=dev)
        for t, like in zip(_run(q, k, v, torch.ones_like(q), None, None), (q, q, k, v)):
            assert t.shape == like.shape and not bool(t.any())
    k = torch.randn(0, 3, 2, 16, device=dev)
    assert _run(torch.randn(0, 3, 4, 16, device=dev), k, k, torch.randn(0, 3, 4, 16, device=dev), None, None)[0].shape == (0, 3, 4, 16)


def test_captured_graphs_and_another_stream(dev):
    """Forward + backward of two sizes in two graphs, replayed in turn with other inputs and counts, beside eager calls."""
    from glenet_amd import _lib
    from glenet_amd.attention import cross_attention
    sets = []
    for seed, case in enumerate([([20, 60], [700, 900], 4, 2, 64, True, False), ([2, 1], [3000, 2000], 8, 2, 32, False, False)]):
        q, k, v, go, mask, cnts = _inputs(case, torch.bfloat16, seed, dev)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]

        def step(leaves=leaves, go=go, mask=mask, cnts=cnts):
            o = cross_attention(*leaves, *cnts, key_mask=mask)
            return [o.detach()] + list(torch.autograd.grad(o, leaves, go))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        for x, y in zip(step(), other):
            assert torch.equal(x, y)
        graph = _lib.new_graph()
        with torch.cuda.graph(graph):
            outs = step()
        sets.append((graph, step, outs, leaves, go, cnts))
    for it in range(4):
        for _, _, _, leaves, go, cnts in sets:
            with torch.no_grad():
                for t in leaves + [go]:
                    t.copy_(torch.randn(t.shape, device=dev))
                cnts[1][0] -= 13
        for graph, *_ in sets:
            graph.replay()
        torch.cuda.synchronize()
        for _, step, outs, *_ in sets:
            for x, y in zip(outs, step()):
                assert torch.equal(x, y)


def test_a_long_sequence_with_offsets_beyond_32_bits(dev):
    """States whose last rows lie more than 2^31 elements into their buffer: 70 frames' worth of one wide packed tensor."""
    rows, width = 40000, 56000                                           # 2.24e9 elements of bf16, 4.5 GB
    big = torch.empty(rows, width, dtype=torch.bfloat16, device=dev)
    k, v = big[:, :64].view(rows, 1, 64), big[:, 64:128].view(rows, 1, 64)
    k.copy_(torch.randn(rows, 1, 64, device=dev))
    v.copy_(torch.randn(rows, 1, 64, device=dev))
    q = torch.randn(2, 1, 64, dtype=torch.bfloat16, device=dev)
    go = torch.randn(2, 1, 64, dtype=torch.bfloat16, device=dev)
    cnts = torch.tensor([1, 1], dtype=torch.int32, device=dev), torch.tensor([39000, 1000], dtype=torch.int32, device=dev)
    for x, y in zip(_run(q, k, v, go, None, cnts), _run(q, k.contiguous(), v.contiguous(), go, None, cnts)):
        assert torch.equal(x, y)


def test_an_attention_block_trained_with_muon(dev):
    """The operators as they are used together: tokens normalised, proposals attending to their frame's points, the block's
    matrices updated with orthogonalised steps.  Every parameter gets the gradient that 64-bit autograd gives."""
    from glenet_amd.attention import cross_attention
    from glenet_amd.norm import LayerNorm
    from glenet_amd.optim import FlatMuon
    torch.manual_seed(0)

    class Block(torch.nn.Module):
        def __init__(self, c, heads):
            super().__init__()
            self.norm, self.heads = LayerNorm(c), heads
            self.wq, self.wkv, self.wo = (torch.nn.Linear(c, n * c, bias=False) for n in (1, 2, 1))

        def forward(self, x, states, x_cnt, s_cnt):
            c = x.shape[1]
            q = self.wq(self.norm(x)).view(-1, self.heads, c // self.heads)
            kv = self.wkv(states).view(states.shape[0], 2, self.heads, c // self.heads)
            return x + self.wo(cross_attention(q, kv[:, 0], kv[:, 1], x_cnt, s_cnt).reshape(-1, c))

    net = Block(64, 4).to(dev)
    opt = FlatMuon(net.parameters(), lr=1e-3)
    x, states = torch.randn(24, 64, device=dev), torch.randn(300, 64, device=dev)
    x_cnt, s_cnt = (torch.tensor(c, dtype=torch.int32, device=dev) for c in ([10, 14], [180, 120]))
    go = torch.randn(24, 64, device=dev)
    y = net(x, states, x_cnt, s_cnt)
    y.backward(go)
    got = {n: p.grad.clone() for n, p in net.named_parameters()}
    ref = {n: p.detach().double().requires_grad_(True) for n, p in net.named_parameters()}
    xd, sd = x.double(), states.double()
    xn = (xd - xd.mean(1, keepdim=True)) / (xd.var(1, correction=0, keepdim=True) + 1e-5).sqrt() * ref["norm.weight"] + ref["norm.bias"]
    outs = []
    for q0, lq, k0, lk in _frames([10, 14], [180, 120]):
        kv = (sd[k0:k0 + lk] @ ref["wkv.weight"].t()).view(lk, 2, 4, 16)
        q = (xn[q0:q0 + lq] @ ref["wq.weight"].t()).view(lq, 4, 16)
        o = [torch.softmax(q[:, j] @ kv[:, 0, j].t() / 4, 1) @ kv[:, 1, j] for j in range(4)]
        outs.append(torch.cat(o, 1))
    want = xd + torch.cat(outs) @ ref["wo.weight"].t()
    # products over 64 and 300 terms behind each other: a few hundred roundings of values of order 1 .. 10
    assert float((y.double() - want).abs().max()) < 500 * U * 10
    grads = torch.autograd.grad(want, list(ref.values()), go.double())
    for (n, g), w in zip(got.items(), grads):
        assert float((g.double() - w).norm()) < 500 * U * 10 * float(w.norm()), n
    before = {n: p.detach().clone() for n, p in net.named_parameters()}
    opt.step()
    for n, p in net.named_parameters():
        assert bool(torch.isfinite(p).all()) and not torch.equal(p, before[n])


def test_negative_scale_and_64_bit_counts(dev):
    case = ([25, 40], [70, 300], 4, 2, 24, True, False)
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, go, mask, cnts = _inputs(case, dtype, 6, dev)
        outs = _run(q, k, v, go, mask, cnts, scale=-0.3)
        ref = _reference(q, k, v, go, mask, case, dtype, scale=-0.3)
        for t, n in zip(outs, ("o", "dq", "dk", "dv")):
            _check(t, ref, n, dtype)
        wide = tuple(c.long() for c in cnts)
        wide[1][1] += 1 << 32                                 # beyond 32 bits: cut at the tensor's end, not wrapped
        for a, b in zip(_run(q, k, v, go, mask, wide, scale=-0.3), outs):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hk,d", [(4, 2, 16), (2, 2, 128), (14, 2, 72)])
def test_rows_with_one_key_have_no_score_gradient(dev, h, hk, d, dtype):
    """softmax of one score is 1 whatever the score: dq is 0, and dk (frames of one key), to the bit; o and dv are v and sum go."""
    case = ([5, 300, 40], [1, 1, 20], h, hk, d, False, False)
    q, k, v, go, _, cnts = _inputs(case, dtype, 9, dev)
    mask = torch.ones(k.shape[0], dtype=torch.bool, device=dev)
    mask[2:] = False
    mask[11] = True                                           # the third frame: one of 20
    o, dq, dk, dv = _run(q, k, v, go, mask, cnts)
    assert not dq.any() and not dk.any()
    at = torch.tensor([0] * 5 + [1] * 300 + [11] * 40, device=dev)
    assert torch.equal(o, v[at].repeat_interleave(h // hk, 1))
    for i, (a, b) in {0: (0, 5), 1: (5, 305), 11: (305, 345)}.items():
        want = go[a:b].double().view(b - a, hk, h // hk, d)
        # (P is 1 to the rounding of s and lse: |s| a few units)
        lim = (HALF[dtype] + (40 + 300) * U) * want.abs().sum((0, 2)) + SUB[dtype]
        assert bool(((dv[i].double() - want.sum((0, 2))).abs() <= lim).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lk", [20, 700])
def test_gradients_of_rows_that_one_key_dominates(dev, lk, dtype):
    """One key's weight is 1 - 1e-3: dS is a thousandth of P dP, so what o loses to its type must not reach delta = sum go o.  The
    p's roundings move delta by h sum |dS| (o is divided by their own sum), o's by h^2 sum |go o| (its rest is kept)."""
    g = torch.Generator().manual_seed(lk)
    d, lq, h = 64, 50, 2
    k, v, go = (torch.randn(n, h, d, generator=g).to(dtype).to(dev) for n in (lk, lk, lq))
    near = torch.randint(0, lk, (lq,), generator=g).to(dev)
    top = math.log(1000.0 * lk)
    q = (k[near].double() * (top * math.sqrt(d) / (k[near].double() ** 2).sum(-1, keepdim=True))).to(dtype)
    cnts = tuple(torch.tensor([n], dtype=torch.int32, device=dev) for n in (lq, lk))
    _, dq, _, _ = _run(q, k, v, go, None, cnts)
    u, scale = HALF[dtype], 1 / math.sqrt(d)
    for j in range(h):
        qq, kk, vv, gg = (t[:, j].double() for t in (q, k, v, go))
        p = torch.softmax(qq @ kk.t() * scale, 1)
        o = p @ vv
        ds = p * (gg @ vv.t() - (gg * o).sum(1, keepdim=True))
        want = scale * ds @ kk
        low = 1.1 * u * ds.abs().sum(1, keepdim=True) + 1.1 * u * u * (gg.abs() * o.abs()).sum(1, keepdim=True)
        # (fp32 sums and scores: the limits of the general test, without its rounding of o)
        es = (2 * d + 40) * U * (qq.abs() @ kk.abs().t()).amax(1, keepdim=True) * scale * 3
        fine = (2 * d + 40) * U * (gg.abs() @ vv.abs().t() + (gg.abs() * o.abs()).sum(1, keepdim=True)) + 2 * es * (gg @ vv.t()).abs().amax(1, keepdim=True)
        lim = scale * ((1.1 * u * ds.abs() + p * (low + fine) + 2 * es * ds.abs()) @ kk.abs()) + u * want.abs() + SUB[dtype]
        if dtype == torch.float16:
            lim = lim + scale * 2.0 ** -24 * ds.abs().max() * kk.abs().sum(0)
        assert bool(((dq[:, j].double() - want).abs() <= lim).all())


@pytest.mark.parametrize("lk", [[20, 3], [200, 20]])
def test_gradients_of_the_keys_alone(dev, lk):
    """dk and dv without dq: delta comes from the same launch, which then writes nothing else."""
    from glenet_amd.attention import cross_attention
    case = ([70, 33], lk, 4, 2, 32, True, False)
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, go, mask, cnts = _inputs(case, dtype, 12, dev)
        _, _, dk, dv = _run(q, k, v, go, mask, cnts)
        kk, vv = k.clone().requires_grad_(True), v.clone().requires_grad_(True)
        o = cross_attention(q, kk, vv, *cnts, key_mask=mask)
        a, b = torch.autograd.grad(o, [kk, vv], go)
        assert torch.equal(a, dk) and torch.equal(b, dv)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [32, 40, 128])
def test_masked_states_have_no_gradient_whatever_the_queries_gradients_hold(dev, d, dtype):
    """A loss takes the logarithm of rows without a state (0) and hands back infinities and NaN: nothing of that reaches the
    gradients of masked states, of trailing ones or of other frames."""
    from glenet_amd.attention import cross_attention
    g = torch.Generator().manual_seed(d)
    ql, kl, h, hk = [40, 70, 3, 2], [50, 150, 0, 40], 4, 2

    def normal(*s):
        return torch.randn(*s, generator=g).to(dtype).to(dev)

    q, k, v, go = normal(sum(ql) + 1, h, d), normal(sum(kl) + 9, hk, d), normal(sum(kl) + 9, hk, d), normal(sum(ql) + 1, h, d)
    mask = (torch.rand(sum(kl) + 9, generator=g) < 0.7).to(dev)
    mask[:50] = False                                         # frame 0 has no state left, frame 2 has none at all
    cnts = tuple(torch.tensor(x, dtype=torch.int32, device=dev) for x in (ql, kl))
    want = _run(q, k, v, go, mask, cnts)
    none = torch.cat([torch.arange(40), torch.arange(110, 113), torch.arange(sum(ql), sum(ql) + 1)]).to(dev)      # rows without a state
    for bad in (float("nan"), float("inf"), -float("inf")):
        broken, odd = go.clone(), q.clone()
        broken[none] = bad
        odd[none] = bad
        for got in (_run(q, k, v, broken, mask, cnts), _run(odd, k, v, go, mask, cnts), _run(odd, k, v, broken, mask, cnts)):
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    broken = go.clone()
    broken[60] = float("nan")                                 # a row of frame 1: its masked states and other frames stay clean
    _, dq, dk, dv = _run(q, k, v, broken, mask, cnts)
    off = ~mask
    off[200:] = True
    for a, b in ((dk, want[2]), (dv, want[3])):
        assert torch.equal(a[off], b[off]) and bool(torch.isnan(a[50:200][mask[50:200]]).any())
    rows = torch.arange(sum(ql) + 1, device=dev) != 60
    assert torch.equal(dq[rows], want[1][rows])


@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("queries,keys", [(8192, 131072), (1, 131072), (40, 700)])
def test_fp16_rows_that_one_key_dominates_keep_the_others_weight(dev, queries, keys, first):
    """One key's weight is 2^25.4 times each of the others', which together add keys 2^-25.4 to the row: 3e-3 of it at 131 072 keys.
    They carry the values 1, the one key 0, so that the row IS what they add.

    A weight is rounded to fp16 at 2^11 times its size, the largest of a row's between 2^11 and 2^15: what rounds to a subnormal is
    off by 2^-25 2^-11, the others by 2^-11 of themselves; the weights' exponents by 4 2^-24 25.4 and the sums by keys 2^-24 relative
    at most; the result is rounded to 2^-11 or half a subnormal step."""
    from glenet_amd.attention import cross_attention
    h, d = 8 if queries > 1 else 2, 8
    q, k, v = (torch.zeros(n, h, d, device=dev, dtype=torch.float16) for n in (queries, keys, keys))
    at = 0 if first else keys - 1
    q[:, :, 0], k[at, :, 0] = 4.195, 4.195
    v.fill_(1.0)
    v[at] = 0.0
    other = math.exp(-float(q[0, 0, 0].double() * k[at, 0, 0].double()))
    want = (keys - 1) * other / (1 + (keys - 1) * other)
    limit = (keys - 1) * 2.0 ** -36 + want * (2 * 2.0 ** -11 + keys * U + 120 * U) + 2.0 ** -25
    for o in (cross_attention(q[None], k[None], v[None], scale=1.0),
              cross_attention(q.clone().requires_grad_()[None], k[None], v[None], scale=1.0)):
        off = float((o.detach().double() - want).abs().max())
        assert off < limit


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("frames,lq,lk,h,hk,d", [(4, 1, 5000, 8, 2, 128), (1, 1, 700, 4, 4, 64), (2, 3, 900, 6, 3, 40), (3, 20, 130, 2, 2, 96)])
def test_few_rows_are_rounded_once(dev, frames, lq, lk, h, hk, d, dtype):
    """Rows of up to one tile a frame: weights go into their product as two 16-bit numbers, off by (half a step)^2 of themselves
    (fp16, whose exponents end: or by 2^-36 of the row's largest), and the result is rounded once.  Scores as in the limits above."""
    from glenet_amd.attention import cross_attention
    g = torch.Generator().manual_seed(lk)
    q, k, v = (torch.randn(frames, n, j, d, generator=g).to(dtype).to(dev) for n, j in ((lq, h), (lk, hk), (lk, hk)))
    kk, vv = (t.double().repeat_interleave(h // hk, 2).permute(0, 2, 1, 3) for t in (k, v))
    qq = q.double().permute(0, 2, 1, 3)
    s = torch.stack([a @ b.transpose(-1, -2) for a, b in zip(qq, kk)]) / math.sqrt(d)
    p = torch.softmax(s, -1)
    es = (d + 8) * U * qq.norm(dim=-1)[..., None] * kk.norm(dim=-1).amax(-1)[..., None, None] / math.sqrt(d) * 1.5 + 4 * U * s.abs().amax()
    mass = torch.stack([a @ b.abs() for a, b in zip(p, vv)])
    want = torch.stack([a @ b for a, b in zip(p, vv)])
    small = 2 * (2 * es + (16 + lk) * U) + HALF[dtype] ** 2
    tiny = 2.0 ** -36 * vv.abs().sum(2, keepdim=True) if dtype == torch.float16 else 0.0
    limit = HALF[dtype] * want.abs() + small * mass + tiny + SUB[dtype]
    for o in (cross_attention(q, k, v), cross_attention(q.clone().requires_grad_(), k, v)):
        off = (o.detach().double().permute(0, 2, 1, 3) - want).abs()
        worst = float((off / limit).max())
        assert worst <= 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [16, 20, 32, 40, 72, 96, 128])
def test_a_score_of_minus_infinity_is_a_weight_of_zero(dev, d, dtype):
    """A state whose product with every query is -infinity weighs nothing, without a mask and at any number of channels."""
    from glenet_amd.attention import cross_attention
    g = torch.Generator().manual_seed(d)
    for lq, lk in ((5, 300), (700, 90)):
        q, k, v = (torch.randn(1, n, 2, d, generator=g).to(dtype).to(dev) for n in (lq, lk, lk))
        q[..., 0] = q[..., 0].abs() + 0.5
        mask = torch.ones(1, lk, dtype=torch.bool, device=dev)
        mask[0, lk // 3] = mask[0, 0] = False
        want = cross_attention(q, k, v, key_mask=mask)
        k[:, lk // 3, :, 0] = k[:, 0, :, 0] = -float("inf")
        got = cross_attention(q, k, v)
        assert bool(torch.isfinite(got).all()) and torch.equal(got, want)
