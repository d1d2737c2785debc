"""Collectives of device tensors over gloo go through host memory (here forced for CPU tensors): the same sums, in
place, brought back once."""
import os
import tempfile

import pytest
import torch
import torch.multiprocessing as mp

from mx_rcnn_amd.parallel import dist as pdist
from tests.test_dist import _free_port


def _worker(rank, world, port, out_dir):
    os.environ.update({'MASTER_ADDR': '127.0.0.1', 'MASTER_PORT': str(port), 'RANK': str(rank),
                       'WORLD_SIZE': str(world), 'LOCAL_RANK': str(rank)})
    import torch.distributed as dist
    pdist.init_distributed(backend='gloo')
    pdist._through_host = lambda t: True
    a = torch.arange(5.0) + rank
    w = pdist.all_reduce(a, async_op=True)
    before = a.clone()
    w.wait()
    summed = a.clone()
    a.zero_()
    w.wait()  # (the optimizer stream and the end of the step both wait)
    b = torch.full((3,), float(rank), dtype=torch.bfloat16)
    assert pdist.all_reduce(b) is None
    c = torch.full((2,), float(rank))
    pdist.all_reduce(c, op=dist.ReduceOp.MAX)
    d = torch.full((2, 2), 5.0 + rank)
    pdist.broadcast(d, 1)
    m = pdist.all_reduce_max(3.0 + rank, 'cpu')
    torch.save({'before': before, 'sum': summed, 'a': a, 'b': b, 'c': c, 'd': d, 'm': torch.tensor(m)},
               os.path.join(out_dir, 'r%d.pt' % rank))
    pdist.barrier()
    pdist.destroy()


def test_two_ranks():
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_worker, args=(2, _free_port(), d), nprocs=2, join=True)
        for r in range(2):
            g = torch.load(os.path.join(d, 'r%d.pt' % r), weights_only=True)
            assert torch.equal(g['before'], torch.arange(5.0) + r)
            assert torch.equal(g['sum'], 2 * torch.arange(5.0) + 1) and bool((g['a'] == 0).all())
            assert g['b'].tolist() == [1.0] * 3 and g['c'].tolist() == [1.0] * 2
            assert bool((g['d'] == 6).all()) and float(g['m']) == 4.0


@pytest.mark.gpu
def test_device_tensors_are_staged(cuda):
    import torch.distributed as dist
    dist.init_process_group('gloo', init_method='tcp://127.0.0.1:%d' % _free_port(), rank=0, world_size=1)
    try:
        t = torch.arange(7.0, device=cuda)
        assert pdist._through_host(t) and not pdist._through_host(t.cpu())
        w = pdist.all_reduce(t, async_op=True)
        assert not w.host.is_cuda
        w.wait()
        assert torch.equal(t.cpu(), torch.arange(7.0)) and pdist.all_reduce_max(2.5, cuda) == 2.5
    finally:
        dist.destroy_process_group()
