"""CPU: AdapterBank's host logic (layout, indexes, storing adapters), the facade's clipping argument, and the flat SUM exchange of
adapter training over gloo with two ranks."""
import os
import types

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_parallel_gloo import _free_port
from yolo_amd import parallel
from yolo_amd.adapters import AdapterBank
from yolo_amd.keras_facade import Adam


def _model(K=50, units=13):
    return types.SimpleNamespace(K=K, units=units, device=torch.device('cpu'))


def test_layout_and_first_values():
    bank = AdapterBank(_model(), 3, 4, scale=0.5)
    assert bank.a.shape == (3, 4, 50) and bank.b.shape == (3, 4, 13) and bank.b.stride() == (64, 16, 1)
    assert bank.flat.numel() == 600 + 3 * 4 * 16 and bank.b.data_ptr() % 16 == 0
    assert int(bank.b.count_nonzero()) == 0 and 0 < float(bank.a.abs().max()) <= 50 ** -0.5 and bool((bank.scale == 0.5).all())
    bank.flat.fill_(7.0)
    assert bool((bank.a == 7).all()) and bool((bank.b == 7).all())
    a, b = bank.views(torch.arange(bank.flat.numel(), dtype=torch.float32))
    assert int(a[2, 3, 49]) == 599 and int(b[0, 0, 0]) == 600 and int(b[2, 3, 12]) == 600 + 11 * 16 + 12


@pytest.mark.parametrize('count, rank', [(0, 4), (4097, 1), (1, 0), (1, 129)])
def test_sizes_refused(count, rank):
    with pytest.raises(ValueError, match='adapters of rank'):
        AdapterBank(_model(), count, rank)


def test_index_on_the_host():
    bank = AdapterBank(_model(), 3, 2)
    want = torch.tensor([0, -1, 2, -1], dtype=torch.int32)
    for which in ([0, None, 2, -1], (0, -1, 2, -1), np.array([0, -1, 2, -1]), torch.tensor([0, -1, 2, -1])):
        got = bank.index(which)
        assert got.dtype == torch.int32 and torch.equal(got, want)
    for bad in ([3], [-2], [0.5], ['0']):
        with pytest.raises(ValueError, match='adapter'):
            bank.index(bad)


def test_set_and_get():
    bank = AdapterBank(_model(), 2, 4)
    rng = np.random.default_rng(0)
    a, b = rng.standard_normal((3, 50)).astype(np.float32), rng.standard_normal((3, 13)).astype(np.float32)
    bank.set(1, a, b, scale=2.0)
    ga, gb, scale = bank.get(1)
    assert np.array_equal(ga[:3], a) and np.array_equal(gb[:3], b) and not ga[3].any() and not gb[3].any() and scale == 2.0
    assert bank.get(0)[2] == 1.0
    for bad in ((a[:, :9], b), (a, b[:2]), (np.zeros((5, 50)), np.zeros((5, 13)))):
        with pytest.raises(ValueError):
            bank.set(0, *bad)
    for i in (-1, 2):
        with pytest.raises(IndexError):
            bank.get(i)


def test_facade_clipping_argument():
    assert Adam(global_clipnorm=2.5).global_clipnorm == 2.5 and Adam().global_clipnorm is None
    for bad in (0, -1.0, float('nan')):
        with pytest.raises(ValueError):
            Adam(global_clipnorm=bad)


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    dist.init_process_group('gloo', rank=rank, world_size=world)
    try:
        flat = torch.arange(5, dtype=torch.float32) * (rank + 1)
        got = parallel.allreduce_flat(flat)
        q.put((rank, got is flat and torch.equal(flat, torch.arange(5, dtype=torch.float32) * 3)))
    finally:
        dist.destroy_process_group()


def test_allreduce_flat_two_ranks():
    alone = torch.ones(3)
    assert parallel.allreduce_flat(alone) is alone and bool((alone == 1).all())
    ctx = mp.get_context('spawn')
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = sorted(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=60)
    assert got == [(0, True), (1, True)]
