"""Forms of the operators' kernels that only larger sizes take: which one a size takes is read from the launches themselves, so a
changed rule cannot leave a form without its test.  Limits: those of test_attention_gpu, test_layer_norm_gpu and
test_orthogonal_gpu, and, for the orthogonaliser, what the same formula leaves in plain fp32 products."""
import math
import re

import pytest
import torch

import test_attention_gpu as xa
import test_layer_norm_gpu as ln
import test_orthogonal_gpu as ns

pytestmark = pytest.mark.gpu

NAMES = {torch.float32: "float", torch.bfloat16: "__bf16", torch.float16: "_Float16"}


def _kernel(name):
    """name<template arguments> of a kernel of these operators, None of others.  Names with 16-bit types come as the linker has them."""
    m = re.match(r"_Z\d+(k_(?:xa|ln|ns)_[a-z_]+)I((?:f|DF16b|DF16_|Li\d+E|Lb[01]E)+)E", name)
    if m:
        words = {"f": "float", "DF16b": "__bf16", "DF16_": "_Float16", "Lb0E": "false", "Lb1E": "true"}
        args = re.findall(r"DF16b|DF16_|Li\d+E|Lb[01]E|f", m.group(2))
        return "%s<%s>" % (m.group(1), ",".join(words.get(a) or a[2:-1] for a in args))
    m = re.search(r"\b(k_(?:xa|ln|ns)_\w+(?:<[^>]*>)?)", name)
    return m.group(1).replace(" ", "") if m else None


def _launched(f):
    """f's result and the kernels of these operators that it launched."""
    from torch.profiler import ProfilerActivity, profile
    with profile(activities=[ProfilerActivity.CUDA, ProfilerActivity.CPU]) as p:
        out = f()
        torch.cuda.synchronize()
    return out, {_kernel(e.name) for e in p.events()} - {None}


def test_launches_are_seen(dev):
    from glenet_amd.norm import layer_norm
    for dtype, lanes in ((torch.float32, 16), (torch.bfloat16, 8), (torch.float16, 8)):
        x = torch.randn(5, 64, device=dev).to(dtype)
        assert _launched(lambda: layer_norm(x))[1] == {"k_ln_forward<%s,%d,1>" % (NAMES[dtype], lanes)}
    assert _kernel("_Z13k_ln_backwardIDF16bLi256ELi4ELb1EEv6LnArgs") == "k_ln_backward<__bf16,256,4,true>"


# ---------------------------------------------------------------------------------------------- cross attention: four row tiles a block
# q lengths, k lengths, heads, key heads, mask, padded; splits over the keys
FOUR = [
    ([700, 0, 300, 3201], [333, 20, 100, 2500], 8, 4, True, False, 1),         # frame 0 has no state left, frame 1 no query, frame 2 one state
    ([1009, 985], [333, 1290], 8, 4, False, False, 2),                          # 3988 rows a key head: 128 blocks and two splits
    ([217] * 6, [1531] * 6, 12, 6, True, True, 2),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [32, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("index", range(len(FOUR)))
def test_attention_with_four_row_tiles_a_block(dev, index, d, dtype):
    ql, kl, h, hk, masked, padded, splits = FOUR[index]
    if index == 0:
        d = d if d != 40 else 20                              # (a row that is no whole chunk)
    case = (ql, kl, h, hk, d, masked, padded)
    q, k, v, go, mask, cnts = xa._inputs(case, dtype, index * 131 + d, dev)
    got, names = _launched(lambda: xa._run(q, k, v, go, mask, cnts))
    wide = (d + 31) // 32 * 32
    two = splits > 1 and not (dtype == torch.float32 and d > 64 and index == 2)
    if index == 2 and dtype == torch.float32 and d > 64:
        assert "k_xa_forward<float,%d,2>" % wide in names     # 144 blocks would fill a card of one block a compute unit too little
    else:
        for kernel in ("k_xa_forward", "k_xa_dq"):
            assert "%s<%s,%d,4>" % (kernel, NAMES[dtype], wide) in names, names
    assert ("k_xa_join<%s>" % NAMES[dtype] in names) == two, names
    with torch.no_grad():
        ref = xa._reference(q, k, v, go, mask, case, dtype)
        for t, n in zip(got, ("o", "dq", "dk", "dv")):
            xa._check(t, ref, n, dtype)
    for a, b in zip(xa._run(q, k, v, go, mask, cnts), got):
        assert torch.equal(a, b)                              # fixed summation orders, dq's among them


# ---------------------------------------------------------------------------------------------- layer norm: blocks that visit rows in turn
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,width,kernel", [(700, 2500, "forward"), (700, 4090, "backward"), (9001, 2060, "forward"), (9001, 4100, "forward_long")])
def test_layer_norm_blocks_visit_many_rows(dev, rows, width, kernel, dtype, wdtype):
    """Rows of a block each: beyond 256 rows a backward block takes several, beyond 8192 a forward one too."""
    from glenet_amd.norm import layer_norm
    if dtype != torch.float32:
        width = width * 2 - 1                                 # eight values a vector: the same forms
    x, w, b, gy = ln._inputs(rows, width, dtype, wdtype, rows + width, dev)
    for t in (x, w, b):
        t.requires_grad_(True)

    def run():
        y = layer_norm(x, w, b, 1e-3)
        return (y,) + torch.autograd.grad(y, (x, w, b), gy)

    (y, dx, dw, db), names = _launched(run)
    form = r"<%s>$" % NAMES[dtype] if kernel == "forward_long" else r"<%s,256,[24](,true)?>$" % NAMES[dtype]
    assert any(re.search("k_ln_%s%s" % (kernel, form), n) for n in names), names
    with torch.no_grad():
        ry, rdx, rdw, rdb, mean, sd, xh = ln._formula(x, w, b, gy, 1e-3)
        ey, edx, edw, edb = ln._limits(x, w, gy, mean, sd, xh)
        ln._check(y, ry, ey + ln.HALF[torch.float32] * ry.abs(), dtype, "y")
        ln._check(dx, rdx, edx, dtype, "dx")
        ln._check(dw, rdw, edw, wdtype, "dw")
        ln._check(db, rdb, edb, wdtype, "db")
    for p, q in zip(run(), (y, dx, dw, db)):
        assert torch.equal(p, q)


# ---------------------------------------------------------------------------------------------- orthogonaliser
def _plain(m):
    """The same steps in fp32 products, rounded once."""
    x = m.float()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + 1e-7)
    a, b, c = ns.COEFFS
    for _ in range(5):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.t() if tall else x).to(m.dtype)


def _flat(r, c, seed, dev, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(r, c, generator=g).to(dev).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("r,c", [(2500, 2601), (1100, 4500), (1500, 1100), (2900, 1100), (2501, 3300), (10300, 2500)])
def test_large_matrices(dev, r, c, dtype):
    """128-wide tiles for X (200 tiles of it: 1100 x 2900) and for the symmetric products (200 on and below the diagonal: 2433 rows),
    in segments of one step and of several."""
    from glenet_amd.optim import orthogonalize
    m, n = min(r, c), max(r, c)
    x = ns._gradient(r, c, r + c, dev, dtype)
    o, names = _launched(lambda: orthogonalize(x))
    wide, across = -(-m // 128), -(-n // 128)
    # (the fewest products of a pair of operands that the type's steps take, and which tiles)
    for tile in {128 if wide * (wide + 1) // 2 >= 200 else 64, 128 if wide * across >= 200 else 64}:
        assert any(s.startswith("k_ns_gemm<%d," % tile) for s in names), names
    assert any("k_ns_gemm<128," in s for s in names) == (wide * across >= 200)
    want = ns._exact(x)
    assert ns._off(o, want) < ns.LIMIT[dtype] + ns.HALF[dtype]
    assert torch.equal(o, orthogonalize(x))
    off, plain, once = ns._off(o, want), ns._off(_plain(x), want), ns._off(want.to(dtype), want)
    assert off < {torch.float32: 2 * plain, torch.bfloat16: 1.4 * once, torch.float16: 1.05 * once}[dtype], (off, plain, once)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [ns._gradient, _flat])
@pytest.mark.parametrize("r,c", [(20, 24), (24, 360), (40, 5001), (64, 64), (128, 1300), (129, 1032), (700, 160), (192, 1000), (200, 300),
                                 (200, 790), (300, 500), (700, 777), (256, 1111), (1500, 300), (500, 2100)])
def test_no_further_off_than_plain_products(dev, r, c, kind, dtype):
    """Operands carry 22 bits, an rms of 2^-23 / sqrt 3 of their size; sums of K >= 64 terms in fp32 leave about 2^-25 sqrt K, so
    that in segments of one step -- fp32 up to 192 rows, and wider matrices up to 4 : 1 -- the error is that of fp32 products or
    less.  Segments of three multiply what the Gram matrix lost in its smallest directions: up to twice.  16-bit results: their own
    rounding, in bfloat16 with up to its equal from five steps on one Gram matrix (1 + 1 in squares)."""
    from glenet_amd.optim import orthogonalize
    m, n = min(r, c), max(r, c)
    sums = torch.zeros(3, dtype=torch.float64)
    for seed in range(4):
        x = kind(r, c, seed, dev, dtype)
        want = ns._exact(x)
        sums += torch.tensor([ns._off(t, want) ** 2 for t in (orthogonalize(x), _plain(x), want.to(dtype))])
    off, plain, once = (sums / 4).sqrt().tolist()
    limit = {torch.float32: plain if m <= 192 or n < 4 * m else 2 * plain, torch.bfloat16: math.sqrt(2) * once, torch.float16: 1.05 * once}[dtype]
    assert off <= limit, (off, plain, once)
