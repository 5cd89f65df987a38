"""The host-memory form of the collectives (what device tensors take under gloo), two gloo ranks on the CPU: same results in place."""
import os

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from immunostruct_amd import distributed as D


def _rank(rank, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2")
    dist.init_process_group("gloo", rank=rank, world_size=2)
    D._through_host = lambda t: True      # (a CPU tensor through the path of a device tensor)
    t = torch.arange(5.0) + 10 * rank
    assert D.all_reduce(t, async_op=True) is None      # synchronous: there is no handle to wait for
    m = torch.tensor([1.0 + rank, 5.0 - rank])
    D.all_reduce(m, op=dist.ReduceOp.MAX)
    p = torch.nn.Parameter(torch.full((3,), float(rank + 1)))
    with torch.no_grad():
        D.broadcast(p, src=1)
    out[rank] = (t.tolist(), m.tolist(), p.tolist())
    dist.destroy_process_group()


def test_host_form_of_the_collectives():
    with mp.Manager() as manager:
        out = manager.dict()
        mp.spawn(_rank, args=(29683, out), nprocs=2)
        want = ([10.0, 12.0, 14.0, 16.0, 18.0], [2.0, 5.0], [2.0, 2.0, 2.0])
        assert out[0] == want and out[1] == want
