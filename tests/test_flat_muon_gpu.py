"""glenet_amd.optim.FlatMuon inside the recorded training step and with a gradient exchange: the update that was recorded is the
update that runs eagerly, to the bit (test_orthogonal_gpu.py holds the eager one against its formulas)."""
import json
import os
import socket
import subprocess
import sys

import pytest
import torch

from test_orthogonal_gpu import _params

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _state(opt):
    return [opt.flat_param, opt.exp_avg, opt.exp_avg_sq, opt.step_count, opt.grad_norm]


@pytest.mark.parametrize("split,buckets", [(False, 1), (True, 1), (True, 2)])
def test_the_recorded_update_is_the_eager_one(dev, split, buckets):
    """Every replay, again from its own gradients and the state in front of it."""
    from glenet_amd import glenet_vr as gvr
    from glenet_amd.optim import FlatMuon
    from test_train_step_gpu import JIT, _batch, _small_model
    model = _small_model(dev)
    pts, bidx, gt, unc = _batch(dev, [52, 53], 6000)
    opt = FlatMuon(model.parameters(), lr=1e-3, max_norm=10.0)
    if split:
        opt.grad_scale = 0.5                                  # what an exchange between two ranks sets in front of the capture
    pipe = gvr.StaticTrainStep(model, 2, pts.shape[0] + 700, max_gt=gt.shape[1], optimizer=opt, seed_rois_with_gt=JIT)
    pipe.calibrate(pts, bidx)
    pipe.load(pts, bidx, gt, unc)
    pipe.capture(split=split, buckets=buckets)
    matrices = torch.zeros(opt.n, dtype=torch.bool, device=dev)
    for p, o, rc in zip(opt.params, opt.offsets, opt.matrix_shapes):
        matrices[o:o + p.numel()] = rc is not None
    for it in range(3):
        opt.set_lr(1e-3 / (it + 1))
        before = [t.clone() for t in _state(opt)]
        pipe.step()
        torch.cuda.synchronize()
        pipe.check()
        after = [t.clone() for t in _state(opt)]
        grad = opt.flat_grad.clone()
        assert bool(torch.isfinite(grad).all()) and bool(grad.any()) and int(opt.step_count) == it + 1
        moved = (after[0] != before[0])
        assert float(moved[matrices].float().mean()) > 0.5 and bool(moved[~matrices].any())
        for t, b in zip(_state(opt), before):
            t.copy_(b)
        opt.update.fill_(float("nan"))                        # (nothing of the last update is read)
        opt.step(packed=True)
        torch.cuda.synchronize()
        assert torch.equal(opt.flat_grad, grad)
        for t, a in zip(_state(opt), after):
            assert torch.equal(t, a)


def test_a_scale_of_the_gradients_is_their_multiple(dev):
    """grad_scale, what an exchange leaves to the update: a half of doubled gradients, clipped or not."""
    from glenet_amd.optim import FlatMuon
    for max_norm in (None, 0.3):
        a, b = (FlatMuon(_params(dev), lr=1e-2, max_norm=max_norm) for _ in range(2))
        a.grad_scale = 0.5
        for _ in range(3):
            g = torch.randn(a.n, device=dev)
            a.flat_grad.copy_(g * 2)
            b.flat_grad.copy_(g)
            a.step(packed=True)
            b.step(packed=True)
            for s, t in zip(_state(a), _state(b)):
                assert torch.equal(s, t)


@pytest.mark.parametrize("buckets", [1, 2])
def test_two_ranks_make_the_update_of_one_on_both_gradients(dev, buckets):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs = []
    for r in range(2):
        env = dict(os.environ, RANK=str(r), LOCAL_RANK=str(r), WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port),
                   MUON_BUCKETS=str(buckets))
        env.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")
        procs.append(subprocess.Popen([sys.executable, os.path.join(ROOT, "tests", "_muon_exchange_worker.py")], env=env,
                                      stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True))
    outs = [p.communicate(timeout=100) for p in procs]
    for p, (_, err) in zip(procs, outs):
        assert p.returncode == 0, err[-3000:]
    got = [json.loads(line[5:]) for out, _ in outs for line in out.splitlines() if line.startswith("MUON ")]
    assert sorted(d["rank"] for d in got) == [0, 1]
    for d in got:
        assert d["equal"] and d["scale"] == 0.5 and d["steps"] == 3, d


def test_coefficients_are_refused_before_anything_moves(dev):
    from glenet_amd import _lib
    from glenet_amd.optim import FlatMuon
    for coeffs in ((50.0, 0.0, 0.0), (3.4445, -4.775, 9.0)):
        with pytest.raises(_lib.GlxError, match="range"):
            FlatMuon(_params(dev), coefficients=coeffs)
