"""Two processes on one card, a replica of the weights each: gradients averaged on the host over gloo (they are copied there
and back), then Muon's step.  The replicas have to hold the same bits after every step.  (Replicas on several cards run the
same kernels with the same sizes; what a card of their own adds is the exchange, which is RCCL's there.)"""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

pytestmark = pytest.mark.gpu
SHAPES = [(256, 256, 3, 3)] * 4 + [(135, 256, 3, 3), (45, 256, 3, 3), (64, 64), (300, 513), (135,), (45,)]


def worker(rank, world, port):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    from r3det.dist_train import Muon
    dist.init_process_group("gloo")
    dev = torch.device("cuda", 0)
    elsewhere = torch.empty(1 + 12345 * rank, device=dev)  # (the ranks' tensors lie at different addresses)
    g = torch.Generator().manual_seed(7)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g).to(dev)) for s in SHAPES]
    ps[1].data = ps[1].data.contiguous(memory_format=torch.channels_last)
    opt = Muon([dict(params=[p for p in ps if p.dim() > 1], weight_decay=0.01),
                dict(params=[p for p in ps if p.dim() < 2], orthogonal=False, lr=0.01)])
    own = torch.Generator().manual_seed(100 + rank)
    for _ in range(3):
        for p in ps:
            mean = torch.randn(p.shape, generator=own)
            dist.all_reduce(mean)
            p.grad = (mean / world).to(dev)
        opt.step()
        mine = torch.cat([t.detach().reshape(-1).cpu() for p in ps for t in (p, opt.state[p]["momentum_buffer"])])
        all_of = [torch.empty_like(mine) for _ in range(world)]
        dist.all_gather(all_of, mine)
        assert all(torch.equal(a.view(torch.int32), mine.view(torch.int32)) for a in all_of)
        assert bool(torch.isfinite(mine).all())
    del elsewhere
    dist.barrier()
    dist.destroy_process_group()


def test_replicas_with_the_same_gradients_stay_equal():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(worker, args=(2, port), nprocs=2, join=True)
