"""What the training operators cost: layer norm, Newton-Schulz orthogonalisation and stacked cross attention.

`own = False` computes them with elementary torch operations in 32 bits, `own = True` with glenet_amd's kernels; both take what
`prepare` makes.  `exact` is the definition in 64 bits, written apart from both.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
STEPS, COEFFS, NS_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LN_EPS = 1e-5

# the matrices of the GLENet-VR detector's parameters, as (rows, columns) of the memory they lie in
DETECTOR = ([(108, 16), (432, 16), (432, 32), (864, 32), (864, 32), (864, 64)] + [(1728, 64)] * 5 + [(192, 128), (64, 2304)]
            + [(64, 576)] * 5 + [(128, 576)] + [(128, 1152)] * 5 + [(64, 128), (128, 512), (14, 256), (32, 32), (32, 64),
                                                                   (256, 20736)] + [(256, 256)] * 5)


def listed():
    return [
        # layer norm behind the RoI head's shared layers, one frame's 128 proposals: the call is all latency
        dict(name="ln_roi", op="ln", rows=128, width=256, dtype="fp32", train=True, affine=True),
        # ... over the non-empty voxels of a batch of four frames, rows of 64 channels
        dict(name="ln_voxels", op="ln", rows=58733, width=64, dtype="fp32", train=True, affine=True),
        # ... over the pooled RoI grid laid flat (216 grid points of 96 channels), inference
        dict(name="ln_grid", op="ln", rows=512, width=20736, dtype="fp32", train=False, affine=True),
        # ... over a long batch of tokens in mixed precision: bandwidth
        dict(name="ln_tokens", op="ln", rows=131072, width=1024, dtype="bf16", train=True, affine=True),
        # the update of one 256-wide head layer
        dict(name="ns_layer", op="ns", shapes="256x256", dtype="fp32"),
        # the update of the whole detector: every weight matrix of it, in one call
        dict(name="ns_detector", op="ns", shapes=_text(DETECTOR), dtype="fp32"),
        # two odd-sized half-precision gradients, one of them tall
        dict(name="ns_odd", op="ns", shapes="777x1411,1411x777", dtype="fp16"),
        # a wide projection's gradient in bfloat16: matrix products
        dict(name="ns_large", op="ns", shapes="4096x4096", dtype="bf16"),
        # every proposal of four frames attends to its frame's keypoints, training
        dict(name="xa_rois", op="xa", q_lens="128,128,128,128", k_lens="2048,1773,1290,2011", heads=4, kv_heads=4, dim=64,
             dtype="fp32", train=True, mask=False, padded=False),
        # one query token per sequence against a long encoder output, heads shared four to one
        dict(name="xa_token", op="xa", q_lens="1,1,1,1", k_lens="32768,32768,32768,32768", heads=32, kv_heads=8, dim=128,
             dtype="bf16", train=False, mask=False, padded=True),
        # a padded batch whose mask says which encoder states are real (one frame has none), odd sizes
        dict(name="xa_padded", op="xa", q_lens="217,217,217,217,217,217", k_lens="1531,1531,1531,1531,1531,1531", heads=6,
             kv_heads=3, dim=40, dtype="fp16", train=False, mask=True, padded=True),
        # long queries and longer encoder states, training in mixed precision: matrix products
        dict(name="xa_long", op="xa", q_lens="4096,4096", k_lens="16384,16384", heads=8, kv_heads=2, dim=128, dtype="bf16",
             train=True, mask=False, padded=True),
    ]


def _text(shapes):
    return ",".join("%dx%d" % s for s in shapes)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _lens(text):
    return [int(v) for v in text.split(",")]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["ln", "ns", "xa"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "ln":
        width = _log_int(rng, 1, 20736)
        rows = _log_int(rng, 1, max(1, min(131072, (1 << 26) // width)))
        return dict(op="ln", rows=rows, width=width, dtype=dtype, train=rng.random() < 0.7, affine=rng.random() < 0.8)
    if op == "ns":
        shapes, cost = [], 0.0
        for _ in range(_log_int(rng, 1, 24)):
            r, c = _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
            cost += min(r, c) * float(r * c)
            if shapes and cost > 2e10:
                break
            shapes.append((r, c))
        return dict(op="ns", shapes=_text(shapes), dtype=dtype)
    kv_heads, group, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 7]), rng.choice([8, 16, 20, 32, 40, 64, 72, 96, 128])
    frames, padded = rng.randint(1, 6), rng.random() < 0.5
    pairs = 2.0e8 / frames / (kv_heads * group)          # query-key pairs a frame and head may have
    lq = _log_int(rng, 1, 4096)
    lk = _log_int(rng, 1, max(1, min(65536, int(pairs / lq))))
    q_lens = [lq] * frames if padded else [rng.randint(0, lq) for _ in range(frames - 1)] + [lq]
    k_lens = [lk] * frames if padded else [rng.randint(0, lk) for _ in range(frames - 1)] + [lk]
    return dict(op="xa", q_lens=",".join(map(str, q_lens)), k_lens=",".join(map(str, k_lens)), heads=kv_heads * group,
                kv_heads=kv_heads, dim=dim, dtype=dtype, train=rng.random() < 0.5, mask=rng.random() < 0.5, padded=padded)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "ln":
        rows, width = case["rows"], case["width"]
        # features behind a residual path: a common offset and a few channels of larger spread
        x = (normal(rows, width) * (1.0 + 2.0 * (normal(width) > 1.5)) + 0.5 * normal(rows, 1)).to(t)
        st = dict(case=case, x=x, weight=None, bias=None)
        if case["affine"]:
            st["weight"] = (1.0 + 0.1 * normal(width)).to(t)
            st["bias"] = (0.1 * normal(width)).to(t)
        if case["train"]:
            st["gy"] = (normal(rows, width) / math.sqrt(rows)).to(t)
            for k in ("x", "weight", "bias"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
        return st
    if case["op"] == "ns":
        mats = []
        for r, c in _shapes(case):
            # a layer's gradient: errors x activations summed over samples, channels of unequal scale
            s = max(64, min(r, c))
            err = normal(s, r) * torch.exp(0.7 * normal(r))
            act = normal(s, c) * torch.exp(0.7 * normal(c))
            mats.append((err.t() @ act * (1e-2 / s)).to(t))
        return dict(case=case, mats=mats)
    ql, kl = _lens(case["q_lens"]), _lens(case["k_lens"])
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = normal(sum(ql), h, d), normal(sum(kl), hk, d), normal(sum(kl), hk, d)
    st = dict(case=case)
    mask = None
    if case["mask"]:
        mask = torch.rand(sum(kl), generator=g, device="cuda") < 0.8
        mask[:kl[0]] = False                                   # a frame that has no real state
        if len(kl) > 1:
            mask[kl[0] + kl[1] // 2:kl[0] + kl[1]] = False     # padding behind half of the states
    if case["padded"]:
        b = len(ql)
        q, k, v = q.view(b, -1, h, d), k.view(b, -1, hk, d), v.view(b, -1, hk, d)
        mask = mask.view(b, -1) if mask is not None else None
    else:
        st["q_cnt"] = torch.tensor(ql, dtype=torch.int32, device="cuda")
        st["k_cnt"] = torch.tensor(kl, dtype=torch.int32, device="cuda")
    st.update(q=q.to(t).contiguous(), k=k.to(t).contiguous(), v=v.to(t).contiguous(), mask=mask)
    if case["train"]:
        st["go"] = normal(*q.shape).to(t)
        for name in ("q", "k", "v"):
            st[name].requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return dict(ln=_run_ln, ns=_run_ns, xa=_run_xa)[case["op"]](state, case)


def _run_ln(st, case):
    x, w, b = st["x"], st["weight"], st["bias"]
    if own:
        from glenet_amd import norm
        if not case["train"]:
            return norm.layer_norm(x, w, b, eps=LN_EPS)
        y = norm.layer_norm(x, w, b, eps=LN_EPS)
        leaves = [x] if w is None else [x, w, b]
        return [y.detach()] + list(torch.autograd.grad(y, leaves, st["gy"]))
    with torch.no_grad():
        xf = x.float()
        centred = xf - xf.mean(1, keepdim=True)
        rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + LN_EPS)
        xhat = centred * rstd
        y = (xhat if w is None else xhat * w.float() + b.float()).to(x.dtype)
        if not case["train"]:
            return y
        gy = st["gy"].float()
        gx = gy if w is None else gy * w.float()
        dx = rstd * (gx - gx.mean(1, keepdim=True) - xhat * (gx * xhat).mean(1, keepdim=True))
        out = [y, dx.to(x.dtype)]
        if w is not None:
            out += [(gy * xhat).sum(0).to(w.dtype), gy.sum(0).to(b.dtype)]
        return out


def _run_ns(st, case):
    if own:
        from glenet_amd import optim
        return optim.orthogonalize(st["mats"], steps=STEPS, coefficients=COEFFS, eps=NS_EPS)
    a, b, c = COEFFS
    out = []
    for m in st["mats"]:
        x = m.float()
        tall = x.shape[0] > x.shape[1]
        if tall:
            x = x.t()
        x = x / (torch.sqrt((x * x).sum()) + NS_EPS)
        for _ in range(STEPS):
            s = x @ x.t()
            x = a * x + (b * s + c * (s @ s)) @ x
        out.append((x.t() if tall else x).to(m.dtype).contiguous())
    return out


def _frames(case):
    q0 = k0 = 0
    for lq, lk in zip(_lens(case["q_lens"]), _lens(case["k_lens"])):
        yield q0, lq, k0, lk
        q0, k0 = q0 + lq, k0 + lk


def _run_xa(st, case):
    if own:
        from glenet_amd import attention
        out = attention.cross_attention(st["q"], st["k"], st["v"], st.get("q_cnt"), st.get("k_cnt"), key_mask=st["mask"])
        if not case["train"]:
            return out
        return [out.detach()] + list(torch.autograd.grad(out, [st["q"], st["k"], st["v"]], st["go"]))
    with torch.no_grad():
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        scale = 1.0 / math.sqrt(d)
        q, k, v = (st[n].reshape(-1, n_h, d) for n, n_h in (("q", h), ("k", hk), ("v", hk)))
        mask = st["mask"].reshape(-1) if st["mask"] is not None else None
        names = ["o"] + (["q", "k", "v"] if case["train"] else [])
        out = dict(o=torch.zeros_like(q))
        if case["train"]:
            go = st["go"].reshape(-1, h, d)
            out.update(q=torch.zeros_like(q), k=torch.zeros_like(k), v=torch.zeros_like(v))
        for q0, lq, k0, lk in _frames(case):
            if lq == 0 or lk == 0:
                continue
            # (kv heads, query heads of the group x queries, channels)
            qf = q[q0:q0 + lq].float().view(lq, hk, -1, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
            kf = k[k0:k0 + lk].float().permute(1, 0, 2).contiguous()
            vf = v[k0:k0 + lk].float().permute(1, 0, 2).contiguous()
            s = torch.matmul(qf, kf.transpose(1, 2).contiguous()) * scale
            if mask is not None:
                s = s.masked_fill(~mask[k0:k0 + lk], float("-inf"))
            top = s.amax(2, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            total = p.sum(2, keepdim=True)
            p = p / torch.where(total == 0, torch.ones_like(total), total)
            o = torch.matmul(p, vf)

            def rows(t):
                return t.view(hk, -1, lq, d).permute(2, 0, 1, 3).reshape(lq, h, d).to(q.dtype)

            out["o"][q0:q0 + lq] = rows(o)
            if not case["train"]:
                continue
            gf = go[q0:q0 + lq].float().view(lq, hk, -1, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
            dp = torch.matmul(gf, vf.transpose(1, 2).contiguous())
            ds = p * (dp - (gf * o).sum(2, keepdim=True)) * scale
            out["q"][q0:q0 + lq] = rows(torch.matmul(ds, kf))
            out["k"][k0:k0 + lk] = torch.matmul(ds.transpose(1, 2).contiguous(), qf).permute(1, 0, 2).to(q.dtype)
            out["v"][k0:k0 + lk] = torch.matmul(p.transpose(1, 2).contiguous(), gf).permute(1, 0, 2).to(q.dtype)
        res = [out[n].view(st["q" if n == "o" else n].shape) for n in names]
        return res if case["train"] else res[0]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "ln":
        n, w = case["rows"] * case["width"], case["width"] * (2 if case["affine"] else 0)
        if case["train"]:
            return dict(bytes=e * (4 * n + 2 * w), flops=20 * n)
        return dict(bytes=e * (2 * n + w), flops=8 * n)
    if case["op"] == "ns":
        nbytes = flops = 0
        for r, c in _shapes(case):
            m, n = min(r, c), max(r, c)
            nbytes += 2 * e * m * n
            # the definition (symmetric products once per pair), or the same polynomial taken on the Gram matrix alone
            flops += min(STEPS * (3 * m * m * n + m ** 3), 3 * m * m * n + 4 * STEPS * m ** 3)
        return dict(bytes=nbytes, flops=flops)
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    nq, nk = sum(_lens(case["q_lens"])), sum(_lens(case["k_lens"]))
    pairs = sum(lq * lk for _, lq, _, lk in _frames(case)) * h
    nbytes = e * d * (2 * nq * h + 2 * nk * hk) + (nk if case["mask"] else 0)
    flops = 4 * pairs * d
    if case["train"]:
        nbytes += e * d * (2 * nq * h + 2 * nk * hk)
        flops += 10 * pairs * d
    return dict(bytes=nbytes, flops=flops)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ln":
            return _exact_ln(st, case)
        if case["op"] == "ns":
            return [_exact_ns(m.double()) for m in st["mats"]]
        return _exact_xa(st, case)


def _exact_ln(st, case):
    outs = [[] for _ in range(2)]
    w = st["weight"].double() if st["weight"] is not None else None
    b = st["bias"].double() if st["bias"] is not None else None
    dw = db = 0.0
    for r0 in range(0, case["rows"], 16384):
        x = st["x"][r0:r0 + 16384].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sd = torch.sqrt(var + LN_EPS)
        z = (x - mean) / sd
        outs[0].append(z if w is None else torch.addcmul(b, z, w))
        if case["train"]:
            gy = st["gy"][r0:r0 + 16384].double()
            gz = gy if w is None else gy * w
            # the Jacobian of z: (I - 1 1'/n - z z'/n) / sd
            n = case["width"]
            outs[1].append((gz - (gz.sum(1, keepdim=True) + z * (z * gz).sum(1, keepdim=True)) / n) / sd)
            dw, db = dw + (gy * z).sum(0), db + gy.sum(0)
    if not case["train"]:
        return torch.cat(outs[0])
    return [torch.cat(outs[0]), torch.cat(outs[1])] + ([dw, db] if w is not None else [])


def _exact_ns(m):
    if m.shape[0] > m.shape[1]:
        return _exact_ns(m.t().contiguous()).t().contiguous()
    a, b, c = COEFFS
    x = m / (torch.linalg.vector_norm(m) + NS_EPS)
    eye = torch.eye(m.shape[0], dtype=m.dtype, device=m.device)
    for _ in range(STEPS):
        s = x.mm(x.t())
        x = (a * eye + s.mm(b * eye + c * s)).mm(x)
    return x


def _exact_xa(st, case):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    flat = {n: st[n].reshape(-1, st[n].shape[-2], d) for n in ("q", "k", "v")}
    mask = st["mask"].reshape(-1) if st["mask"] is not None else None
    out = torch.zeros(flat["q"].shape, dtype=torch.float64, device="cuda")
    gq, gk, gv = (torch.zeros(flat[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v"))
    for q0, lq, k0, lk in _frames(case):
        live = torch.arange(k0, k0 + lk, device="cuda")
        if mask is not None:
            live = live[mask[k0:k0 + lk]]
        if lq == 0 or live.numel() == 0:
            continue
        for j in range(h):
            kk, vv = flat["k"][live, j // (h // hk)].double(), flat["v"][live, j // (h // hk)].double()
            for r0 in range(q0, q0 + lq, 2048):
                r1 = min(r0 + 2048, q0 + lq)
                qq = flat["q"][r0:r1, j].double()
                p = torch.softmax(qq.mm(kk.t()) / math.sqrt(d), dim=1)
                o = p.mm(vv)
                out[r0:r1, j] = o
                if case["train"]:
                    go = st["go"].reshape(-1, h, d)[r0:r1, j].double()
                    gp = go.mm(vv.t())
                    gs = p * (gp - (p * gp).sum(1, keepdim=True)) / math.sqrt(d)
                    gq[r0:r1, j] = gs.mm(kk)
                    gk[:, j // (h // hk)].index_add_(0, live, gs.t().mm(qq))
                    gv[:, j // (h // hk)].index_add_(0, live, p.t().mm(go))
    res = [out.view(st["q"].shape)]
    if not case["train"]:
        return res[0]
    return res + [t.view(st[n].shape) for t, n in ((gq, "q"), (gk, "k"), (gv, "v"))]
