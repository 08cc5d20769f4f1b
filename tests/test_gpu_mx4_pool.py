"""A 4-bit pool's prefills: launches by the prompts' lengths, each source row read once."""
import pytest
import torch

from specgrove_amd import ops
from specgrove_amd.cache import Mx4RequestCachePool, PersistentRequestCachePool
from tests.test_gpu_mx4_serving import _source

pytestmark = pytest.mark.gpu


def test_a_prompts_launch_covers_its_rows_and_not_its_slot(device, monkeypatch):
    lengths, started = [5, 0, 33, 1, 70], []
    caches = [_source(device, L, 2, 2, 64, "plain", i) for i, L in enumerate(lengths)]
    call = ops.PreparedCall.__call__

    def record(self):
        started.append((self._args.keep_stride, self._args.capacity))
        return call(self)

    monkeypatch.setattr(ops.PreparedCall, "__call__", record)
    pool = Mx4RequestCachePool(caches, 4096)
    pool.check_status()
    assert started == [(L, 4096) for L in lengths if L]


def test_pools_made_of_a_4_bit_pool_hold_its_values(device, monkeypatch):
    lengths = [9, 0, 40]
    caches = [_source(device, L, 2, 2, 64, "tokens", 7 + i) for i, L in enumerate(lengths)]
    first = Mx4RequestCachePool(caches, 64)
    reads = []
    load = ops.kv_load_mx4
    monkeypatch.setattr(ops, "kv_load_mx4", lambda *a, **k: reads.append(0) or load(*a, **k))
    again = Mx4RequestCachePool(first.caches, 80)
    assert len(reads) == 2 * 2 * 3 + 1
    monkeypatch.undo()
    wide = PersistentRequestCachePool(first.caches, 80)
    for a, b, c in zip(first.caches, again.caches, wide.caches):
        for x, y, z in zip(a.layers, b.layers, c.layers):
            # (Packing what was packed gives the same values.)
            assert torch.equal(x.keys, y.keys) and torch.equal(x.keys, z.keys)
            assert torch.equal(x.values, y.values) and torch.equal(x.values, z.values)
    again.check_status()


def test_more_rows_than_the_bound_are_refused(device):
    tree = torch.randn((2, 40, 2, 64), device=device).to(torch.bfloat16)
    codes = torch.zeros((2, 2, 64, 32), dtype=torch.uint8, device=device)
    scales = torch.zeros((2, 2, 64, 2), dtype=torch.uint8, device=device)

    def at(t):
        return ops.pointer_array([t], device)

    def i32(*v):
        return torch.tensor(v, dtype=torch.int32, device=device)

    lengths, status = i32(0), i32(0)
    call = ops.prepare_kv_commit_mx4(
        at(codes[0]), at(scales[0]), at(codes[1]), at(scales[1]), at(tree[0]), at(tree[1]),
        num_kv_heads=2, head_dim=64, code_head_stride=codes.stride(1),
        code_token_stride=codes.stride(2), scale_head_stride=scales.stride(1),
        scale_token_stride=scales.stride(2), tree_row_stride=tree.stride(1),
        tree_head_stride=tree.stride(2), row_offset=i32(0, 40), keep_rows=None,
        keep_len=i32(40), prefix_start=torch.zeros(1, dtype=torch.int64, device=device),
        lengths=lengths, capacity=64, status=status)
    call.set(keep_stride=39)()
    assert int(status.item()) == -2 and int(lengths.item()) == 0 and not codes.any()
    call.set(keep_stride=40)()
    assert int(lengths.item()) == 40
    assert torch.equal(ops.kv_load_mx4(codes[0], scales[0])[:, 40:],
                       torch.zeros((2, 24, 64), dtype=torch.bfloat16, device=device))
