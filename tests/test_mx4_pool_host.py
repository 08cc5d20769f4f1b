"""What reading a 4-bit pool's rows does, on the CPU: a stand-in for the unpacking call
records what is asked of it."""
import contextlib

import pytest
import torch

from specgrove_amd import cache as cache_mod
from specgrove_amd import ops

LAYERS, HKV, CAP, DIM = 3, 2, 8, 64


@pytest.fixture
def pool(monkeypatch):
    """A pool over CPU tensors whose reads are recorded: (which, layer, current device)."""
    pool = cache_mod.Mx4RequestCachePool.__new__(cache_mod.Mx4RequestCachePool)
    pool.capacity, pool.lengths, pool.num_layers = CAP, [5, 3], LAYERS
    pool.device = torch.device("cuda", 1)
    for name, width in (("codes", DIM // 2), ("scales", DIM // 32)):
        for which in "kv":
            setattr(pool, f"{which}_{name}", [
                torch.zeros((HKV, 2 * CAP, width), dtype=torch.uint8) for _ in range(LAYERS)])
    pool.caches = tuple(cache_mod.PersistentRequestCache(pool, i) for i in range(2))
    pool.reads, current = [], [torch.device("cuda", 0)]

    @contextlib.contextmanager
    def use(device):
        before, current[0] = current[0], device
        yield
        current[0] = before

    def load(codes, scales):
        where = [(w, i) for w in "kv" for i in range(LAYERS)
                 if getattr(pool, f"{w}_codes")[i].data_ptr()
                 <= codes.data_ptr() < getattr(pool, f"{w}_codes")[i].data_ptr()
                 + getattr(pool, f"{w}_codes")[i].numel()]
        pool.reads.append((*where[0], current[0]))
        return torch.zeros((*codes.shape[:-1], DIM), dtype=torch.bfloat16)

    monkeypatch.setattr(torch.cuda, "device", use)
    monkeypatch.setattr(ops, "kv_load_mx4", load)
    return pool


def test_a_read_unpacks_its_own_rows_on_the_pools_device(pool):
    layer = pool.caches[0].layers[1]
    assert layer.keys.shape == (1, HKV, 5, DIM)
    assert pool.reads == [("k", 1, pool.device)]
    assert pool.caches[1].layers[2].values.shape == (1, HKV, 3, DIM)
    assert pool.reads[1:] == [("v", 2, pool.device)]


def test_a_pool_made_of_a_4_bit_one_reads_every_row_once(pool):
    cache_mod.PersistentRequestCachePool(pool.caches, CAP)
    # Each cache's K and V of every layer, and the first keys for their shape.
    assert len(pool.reads) == 2 * LAYERS * 2 + 1
