"""One rank of tests/test_flat_muon_gpu.py's exchange: FlatMuon's gradients over gloo (host copies; the ranks share the GPU), whole
or in two buckets, against one process that was handed both ranks' gradients."""
import json
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))


def main():
    import torch.distributed as dist
    from glenet_amd.optim import FlatMuon
    from test_orthogonal_gpu import _params
    rank, world, buckets = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"]), int(os.environ["MUON_BUCKETS"])
    dev = torch.device("cuda", 0)
    dist.init_process_group("gloo")
    kw = dict(lr=1e-2, weight_decay=0.02, max_norm=0.7)
    mine, alone = _params(dev), _params(dev)
    with torch.no_grad():
        for p in mine:
            p.add_(0.01 * rank)                               # rank 1 starts elsewhere: the broadcast repairs that
    opt, ref = FlatMuon(mine, **kw), FlatMuon(alone, **kw)
    opt.broadcast_state_(0)
    ref.grad_scale = 1.0 / world
    equal = True
    for it in range(3):
        grads = [[torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * it + 10 * r + i)).to(dev) for i, p in enumerate(mine)]
                 for r in range(world)]
        for i, p in enumerate(mine):
            p.grad = grads[rank][i].clone(memory_format=torch.preserve_format)
        for i, p in enumerate(alone):
            p.grad = sum(g[i] for g in grads)
        if buckets == 1:
            opt.pack_grads()
            opt.allreduce_()
        else:
            early, late, ei, li = opt.buckets(mine[2:5])
            opt.pack_grads(only=ei, bump=False)
            opt.allreduce_ranges_(early)
            opt.pack_grads(only=li)
            opt.allreduce_ranges_([late])
        opt.step(packed=True)
        ref.step()
        torch.cuda.synchronize()
        equal = equal and all(torch.equal(a, b) for a, b in ((opt.flat_param, ref.flat_param), (opt.exp_avg, ref.exp_avg),
                                                             (opt.exp_avg_sq, ref.exp_avg_sq), (opt.grad_norm, ref.grad_norm)))
    print("MUON " + json.dumps(dict(rank=rank, equal=bool(equal), scale=opt.grad_scale, steps=int(opt.step_count))), flush=True)
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
