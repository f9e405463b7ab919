"""gloo is given host memory only: the bucket and the parameters of a GPU engine go through a copy of them, with the sums of the direct collectives
(distributed.py:24-57, :71-74).  Two ranks on the CPU, the copying switched on by hand."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from tests.test_host_logic import _FakeEngine


class _Recording:
    """torch.distributed, noting the storage of every tensor that a collective is called with."""
    ReduceOp = dist.ReduceOp

    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        call = getattr(dist, name)
        if name not in ('all_reduce', 'broadcast'):
            return call

        def recorded(t, *args, **kw):
            self.seen.append((name, t.untyped_storage().data_ptr(), t.device.type, t.numel()))
            return call(t, *args, **kw)
        return recorded


def _worker(rank, world, port, tmp, overlap):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    dist.init_process_group('gloo', rank=rank, world_size=world)
    from dotaclient_amd import distributed as D
    D._lib.ptr = lambda t: t
    D._lib.stream_ptr = lambda: None
    D._lib.check = lambda code, what='': None
    D.dist = rec = _Recording()
    out = {}
    for over_host in (False, True):
        eng = _FakeEngine([1, 1, 1, 1, 1 if rank == 0 else 0])
        red = D.FlatGradAllReducer(eng, overlap=overlap)
        assert red.over_host is False                    # CPU tensors need no copy
        red.over_host = over_host
        eng.reducer = red
        eng.params.fill_(float(rank + 1))
        del rec.seen[:]
        red.sync_parameters()
        eng.grads.copy_(torch.randn(eng.total, generator=torch.Generator().manual_seed(100 + rank)))
        if overlap:
            red.start_upper(eng)
            red.finish(eng)
        else:
            red(eng)
        own = {eng.params.untyped_storage().data_ptr(), red.bucket.untyped_storage().data_ptr()}
        assert len(rec.seen) == (3 if overlap else 2)
        assert all((ptr in own) != over_host and dev == 'cpu' for _, ptr, dev, _ in rec.seen)
        assert torch.all(eng.params == 1.0)
        out[over_host] = red.bucket.clone()
    assert torch.equal(out[False], out[True])
    torch.save(out[True], os.path.join(tmp, 'r%d.pt' % rank))
    dist.destroy_process_group()


@pytest.mark.parametrize('overlap', [False, True])
def test_collectives_over_host_equal_the_direct_ones(tmp_path, overlap):
    world, port = 2, 31200 + (os.getpid() + int(overlap)) % 2000
    mp.spawn(_worker, args=(world, port, str(tmp_path), overlap), nprocs=world, join=True)
    a, b = (torch.load(os.path.join(str(tmp_path), 'r%d.pt' % r)) for r in range(world))
    assert torch.equal(a, b)


@pytest.mark.parametrize('device,backend,want', [('cuda', 'gloo', True), ('cuda', 'nccl', False), ('cpu', 'gloo', False), ('cuda', None, False)])
def test_only_gpu_tensors_under_gloo_are_copied(monkeypatch, device, backend, want):
    from dotaclient_amd import distributed as D
    monkeypatch.setattr(torch.distributed, 'is_initialized', lambda: backend is not None)
    monkeypatch.setattr(torch.distributed, 'get_backend', lambda group=None: backend)
    assert D.over_host(torch.device(device)) is want
