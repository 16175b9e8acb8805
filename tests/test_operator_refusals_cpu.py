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


def test_orthogonalize_refuses():
    from glenet_amd import _lib
    from glenet_amd.optim import orthogonalize
    m = torch.zeros(4, 6)
    with pytest.raises(_lib.GlxError, match="no CPU path"):
        orthogonalize(m)
    with pytest.raises(_lib.GlxError, match="no CPU path"):
        orthogonalize([m, m])
    assert orthogonalize([]) == []
    for bad in (torch.zeros(5), m.double(), [m, m.half()], [torch.zeros(2, 3, 4)], [3.0], torch.zeros(0, 3), [torch.zeros(2, 0)]):
        with pytest.raises(ValueError):
            orthogonalize(bad)
    for kw in (dict(steps=0), dict(steps=65), dict(steps=2.5), dict(coefficients=(1.0, 2.0)),
               dict(coefficients=(float("nan"), 0.0, 0.0)), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            orthogonalize(m, **kw)


def test_orthogonalize_c_entry_refuses():
    """The C entry's own checks, on the host: shapes, steps, coefficients that diverge, workspaces that are too small."""
    import ctypes

    from glenet_amd import _lib
    from glenet_amd.optim import _Matrix
    lib = _lib.load()

    def call(rows=4, cols=6, ld=6, dtype=0, steps=5, coeffs=(3.4445, -4.775, 2.0315), eps=1e-7, ws=16, nbytes=0, src=64):
        t = (_Matrix * 1)(_Matrix(src, 64, ld, 6, rows, cols))
        rc = lib.glx_orthogonalize(t, 1, dtype, steps, (ctypes.c_double * 3)(*coeffs), ctypes.c_double(eps), ctypes.c_void_p(ws),
                                   ctypes.c_size_t(nbytes), ctypes.c_void_p(0))
        return rc, lib.glx_last_error().decode()

    assert call()[0] == -3 and "workspace" in call()[1]                       # every other check passed
    for kw in (dict(rows=0), dict(cols=1 << 21, ld=1 << 21), dict(rows=40000, cols=40000, ld=40000), dict(dtype=3), dict(steps=0),
               dict(steps=65), dict(eps=-1.0), dict(ld=5), dict(src=0)):
        assert call(**kw)[0] == -1, kw
    for coeffs in ((50.0, 0.0, 0.0), (3.4445, -4.775, 9.0), (float("nan"), 0.0, 0.0), (float("inf"), 0.0, 0.0)):
        rc, msg = call(coeffs=coeffs)
        assert rc == -1 and "range" in msg, (coeffs, rc, msg)
    assert call(coeffs=(1.875, -1.25, 0.375), steps=64)[0] == -3
    assert call(steps=64)[0] == -3
    t = (_Matrix * 1)(_Matrix(64, 64, 6, 6, 4, 6))
    assert lib.glx_orthogonalize_workspace_bytes(t, 1, 0, 5) > 0 and lib.glx_orthogonalize_workspace_bytes(t, 1, 7, 5) == 0


def test_cross_attention_refuses():
    from glenet_amd import _lib
    from glenet_amd.attention import cross_attention
    q, k = torch.zeros(2, 5, 4, 16), torch.zeros(2, 7, 2, 16)
    c = torch.tensor([5, 5], dtype=torch.int32)
    with pytest.raises(_lib.GlxError, match="no CPU path"):
        cross_attention(q, k, k)
    with pytest.raises(_lib.GlxError, match="no CPU path"):
        cross_attention(q.view(10, 4, 16), k.view(14, 2, 16), k.view(14, 2, 16), c, c)
    bad = [(q.double(), k.double(), k.double()), (q, k.half(), k), (q, k, k.half()), (q[0], k[0], k[0]), (q, k, k[:, :6]),
           (q, k[..., :8], k[..., :8]), (q[:1], k, k), (q[:, :, :3], k, k), (torch.zeros(1, 2, 1, 129),) + (torch.zeros(1, 3, 1, 129),) * 2,
           (torch.zeros(1, 2, 1, 0),) + (torch.zeros(1, 3, 1, 0),) * 2, (q, k[:, :, :0], k[:, :, :0])]
    for args in bad:
        with pytest.raises(ValueError):
            cross_attention(*args)
    for kw in (dict(key_mask=torch.ones(2, 7)), dict(key_mask=torch.ones(2, 5, dtype=torch.bool)), dict(scale=float("nan")),
               dict(q_batch_cnt=c), dict(q_batch_cnt=c, k_batch_cnt=c)):
        with pytest.raises(ValueError):
            cross_attention(q, k, k, **kw)
    q3, k3 = q.view(10, 4, 16), k.view(14, 2, 16)
    for a, b in ((c, None), (None, c), (c, c[:1]), (c.float(), c), (c, c.view(2, 1))):
        with pytest.raises(ValueError):
            cross_attention(q3, k3, k3, a, b)


def test_attention_c_entry_refuses():
    import ctypes

    from glenet_amd import _lib
    lib = _lib.load()

    class _Attention(ctypes.Structure):        # glx_attention
        _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "out", "out_rest", "lse", "key_mask", "q_cnt", "k_cnt")]
                    + [(n, ctypes.c_int64) for n in ("q_rows", "k_rows", "q_len", "k_len", "q_stride", "q_head_stride", "k_stride",
                                                     "k_head_stride", "v_stride", "v_head_stride")]
                    + [(n, ctypes.c_int32) for n in ("frames", "heads", "kv_heads", "dim", "dtype")] + [("scale", ctypes.c_float)])


    def call(backward=False, **kw):
        d = _Attention(q=64, k=64, v=64, out=64, lse=64, q_rows=2000, k_rows=8000, q_len=1000, k_len=4000, q_stride=64, q_head_stride=16,
                       k_stride=32, k_head_stride=16, v_stride=32, v_head_stride=16, frames=2, heads=4, kv_heads=2, dim=16, dtype=1,
                       scale=0.25)
        for n, x in kw.items():
            setattr(d, n, x)
        size0, null = ctypes.c_size_t(0), ctypes.c_void_p(0)
        if backward:
            p = ctypes.c_void_p(64)
            return lib.glx_attention_backward(ctypes.byref(d), p, ctypes.c_int64(64), ctypes.c_int64(16), p, p, p, null, size0, null)
        return lib.glx_attention_forward(ctypes.byref(d), null, size0, null)

    for kw in (dict(dtype=9), dict(dim=129), dict(dim=0), dict(heads=3), dict(kv_heads=0), dict(frames=-1), dict(q_len=999), dict(k_rows=1),
               dict(q=0), dict(out=0), dict(v=0), dict(q_cnt=64), dict(k_cnt=64), dict(q_rows=1 << 40)):
        assert call(**kw) == -1 and call(True, **kw) == -1, kw
    assert call(True, lse=0) == -1
    assert call(True) == -3                                          # every other check passed
    assert call(q_rows=2, q_len=1) == -3                             # few rows: split over the keys, a workspace
    assert lib.glx_attention_forward(None, None, ctypes.c_size_t(0), None) == -1


def test_workspace_of_the_orthogonaliser():
    """Of one matrix m x n, rows padded to 64 (above 1024: 128) elements and 64 more: X once, its transpose twice, A and P (longer
    segments: also H, a second P and two Qs) as two 16-bit planes, sums and split products beside them; of a list at most 1 GiB and
    one matrix."""
    import ctypes

    from glenet_amd import _lib
    from glenet_amd.optim import _Matrix
    lib = _lib.load()

    def need(shapes, dtype=1, steps=5):
        t = (_Matrix * len(shapes))(*[_Matrix(64, 64, c, c, r, c) for r, c in shapes])
        return lib.glx_orthogonalize_workspace_bytes(t, len(shapes), dtype, steps)

    small = 1 << 16
    assert need([(4096, 4096)]) <= 4 * 5 * 4096 * 4160 + small
    assert need([(4096, 4096)], steps=1) <= 4 * 4 * 4096 * 4160 + small
    assert need([(8192, 8192)], dtype=0) <= 4 * 5 * 8192 * 8256 + small
    for dtype in range(3):
        wide = 4 * (2 * 1280 * 5184 + 5120 * 1344 + 6 * 1280 * 1344)
        assert need([(1200, 5000)], dtype) <= wide + 4 * 5120 * 1344 + small
    one = need([(4096, 4096)])
    assert one <= need([(4096, 4096)] * 3) <= 3 * one
    assert need([(4096, 4096)] * 300) <= (1 << 30) + small and need([(100, 4096)] * 3000) <= (1 << 30) + small
    assert need([(20000, 20000)] * 4) == need([(20000, 20000)])             # one of them is beyond it already: one by one
    assert need([(4096, 4096)] + [(16, 100)] * 50) == one and need([(3, 5)] * 9) <= small


def test_orthogonalize_c_entry_asks_for_the_workspace_it_names():
    import ctypes

    from glenet_amd import _lib
    from glenet_amd.optim import _Matrix
    lib = _lib.load()
    for shapes in ([(4096, 4096)] * 9, [(900, 140)], [(140, 900), (3, 4), (2500, 2500)], [(16, 16)] + [(20000, 20000)]):
        t = (_Matrix * len(shapes))(*[_Matrix(64, 64, c, c, r, c) for r, c in shapes])
        named = lib.glx_orthogonalize_workspace_bytes(t, len(shapes), 1, 5)
        for coeffs in ((3.4445, -4.775, 2.0315), (4.5, -14.58, 9.44784)):
            rc = lib.glx_orthogonalize(t, len(shapes), 1, 5, (ctypes.c_double * 3)(*coeffs), ctypes.c_double(1e-7), ctypes.c_void_p(256),
                                       ctypes.c_size_t(0), ctypes.c_void_p(0))
            asked = int(lib.glx_last_error().decode().split("<")[1].split()[0])
            assert rc == -3 and asked <= named < asked + 1024


def test_orthogonalize_c_entry_refuses_coefficients_of_an_empty_list():
    import ctypes

    from glenet_amd import _lib
    lib = _lib.load()
    for coeffs, want in (((3.4445, -4.775, 2.0315), 0), ((50.0, 0.0, 0.0), -1), ((3.4445, -4.775, 9.0), -1)):
        assert lib.glx_orthogonalize(None, 0, 0, 5, (ctypes.c_double * 3)(*coeffs), ctypes.c_double(1e-7), None, ctypes.c_size_t(0), None) == want
