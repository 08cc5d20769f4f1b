"""The 4-bit cache's commit and load against the format's definition on the CPU:
codes, scales and values bit for bit, and everything else left as it was."""
import numpy as np
import pytest
import torch

from specgrove_amd import ops
from tests import mx4_cases as M

pytestmark = pytest.mark.gpu


def _rows(shape, seed):
    """bf16 rows over the whole range of the type, ties of the grid among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    kind = torch.randint(0, 6, shape[:-1], generator=g)[..., None]
    x = torch.where(kind == 1, (x * 8).round() / 4, x)            # ties
    x = torch.where(kind == 2, x * 2.0 ** 100, x)
    x = torch.where(kind == 3, x * 2.0 ** -126, x)                # subnormal results
    x = torch.where(kind == 4, torch.zeros_like(x), x)
    x = torch.where(kind == 5, x.sign() * torch.tensor(3.3895e38), x)
    return x.to(torch.bfloat16)


def _call(dev, tree, codes, scales, **kw):
    """kv_commit_mx4 of tree [2, layers, Hkv, R, D] into codes/scales [2, layers, ...]."""
    p = [ops.pointer_array(list(t[i].unbind(0)), dev)
         for i in (0, 1) for t in (codes, scales)]
    p += [ops.pointer_array(list(tree[i].unbind(0)), dev) for i in (0, 1)]
    ops.kv_commit_mx4(*p, num_kv_heads=tree.shape[2], head_dim=tree.shape[4],
                      code_head_stride=codes.stride(2), code_token_stride=codes.stride(3),
                      scale_head_stride=scales.stride(2), scale_token_stride=scales.stride(3),
                      tree_row_stride=tree.stride(3), tree_head_stride=tree.stride(2), **kw)


def _dev(a, device, dtype=torch.int32):
    return torch.tensor(a, dtype=dtype, device=device)


@pytest.mark.parametrize("layers,hkv,dim,rows,keeps,lens", [
    (1, 1, 32, 1, [[0]], [0]),
    (1, 2, 64, 5, [[0, 3, 4], []], [2, 1]),
    (3, 8, 128, 40, [[0, 1, 2, 5, 39], [0], list(range(33)), []], [7, 0, 1, 3]),
    (2, 3, 96, 20, [list(range(17)), [19, 0, 0]], [0, 30]),
])
def test_commit_packs_the_kept_rows_and_nothing_else(device, layers, hkv, dim, rows, keeps, lens):
    n, cap = len(keeps), 48
    tree = _rows((2, layers, hkv, n * rows, dim), dim + layers).to(device)
    g = torch.Generator().manual_seed(1)
    shape = (2, layers, hkv, n * cap)
    codes = torch.randint(0, 256, (*shape, dim // 2), generator=g).to(torch.uint8)
    scales = torch.randint(0, 256, (*shape, dim // 32), generator=g).to(torch.uint8)
    want_codes, want_scales = codes.clone(), scales.clone()
    packed, by = M.pack(tree.cpu())
    for i, keep in enumerate(keeps):
        for t, k in enumerate(keep):
            at, src = i * cap + lens[i] + t, i * rows + k
            want_codes[:, :, :, at] = packed[:, :, :, src]
            want_scales[:, :, :, at] = by[:, :, :, src]
    stride = max(1, max(len(k) for k in keeps))
    codes, scales = codes.to(device), scales.to(device)
    lengths = _dev(lens, device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    _call(device, tree, codes, scales, row_offset=_dev([rows * i for i in range(n + 1)], device),
          keep_rows=_dev([k + [-1] * (stride - len(k)) for k in keeps], device),
          keep_len=_dev([len(k) for k in keeps], device),
          prefix_start=_dev([cap * i for i in range(n)], device, torch.int64),
          lengths=lengths, capacity=cap, status=status)
    assert torch.equal(codes.cpu(), want_codes) and torch.equal(scales.cpu(), want_scales)
    assert lengths.tolist() == [a + len(k) for a, k in zip(lens, keeps)]
    assert int(status.item()) == 0


@pytest.mark.parametrize("rows,lens", [([1, 50, 16], [0, 0, 0]), ([33], [5])])
def test_commit_of_whole_prompts(device, rows, lens):
    n, cap, dim = len(rows), 64, 128
    offset = np.concatenate([[0], np.cumsum(rows)]).tolist()
    tree = _rows((2, 2, 2, offset[-1], dim), 9).to(device)
    codes = torch.zeros((2, 2, 2, n * cap, dim // 2), dtype=torch.uint8, device=device)
    scales = torch.zeros((2, 2, 2, n * cap, dim // 32), dtype=torch.uint8, device=device)
    lengths = _dev(lens, device)
    _call(device, tree, codes, scales, row_offset=_dev(offset, device), keep_rows=None,
          keep_len=_dev(rows, device),
          prefix_start=_dev([cap * i for i in range(n)], device, torch.int64),
          lengths=lengths, capacity=cap)
    packed, by = M.pack(tree.cpu())
    for i, r in enumerate(rows):
        at = slice(i * cap + lens[i], i * cap + lens[i] + r)
        assert torch.equal(codes[:, :, :, at].cpu(), packed[:, :, :, offset[i]:offset[i + 1]])
        assert torch.equal(scales[:, :, :, at].cpu(), by[:, :, :, offset[i]:offset[i + 1]])
    assert lengths.tolist() == [a + r for a, r in zip(lens, rows)]


def test_infinities_and_nans_make_their_block_nan(device):
    x = torch.randn((2, 1, 1, 4, 128), generator=torch.Generator().manual_seed(3))
    x[0, 0, 0, 1, 40] = float("inf")
    x[1, 0, 0, 2, 127] = float("nan")
    x[1, 0, 0, 3, 0] = -float("inf")
    tree = x.to(torch.bfloat16).to(device)
    codes = torch.zeros((2, 1, 1, 4, 64), dtype=torch.uint8, device=device)
    scales = torch.zeros((2, 1, 1, 4, 4), dtype=torch.uint8, device=device)
    _call(device, tree, codes, scales, row_offset=_dev([0, 4], device), keep_rows=None,
          keep_len=_dev([4], device), prefix_start=_dev([0], device, torch.int64),
          lengths=_dev([0], device), capacity=4)
    packed, by = M.pack(tree.cpu())
    assert torch.equal(codes.cpu(), packed) and torch.equal(scales.cpu(), by)
    got = ops.kv_load_mx4(codes, scales).cpu()
    bad = torch.isnan(got)
    assert int(bad.sum()) == 3 * 32
    assert bad[0, 0, 0, 1, 32:64].all() and bad[1, 0, 0, 2, 96:].all() and bad[1, 0, 0, 3, :32].all()


@pytest.mark.parametrize("keep,lens,capacity,code", [
    ([[0, 7], [1, 2]], [0, 0], 16, -1),      # row 7 of a 6-row request
    ([[0, -1], [1, 2]], [0, 0], 16, -1),
    ([[0, 1], [1, 2]], [15, 0], 16, -2),     # no room
    ([[0, 1], [1, 2]], [-1, 0], 16, -2),
])
def test_a_bad_request_is_left_alone_and_reported(device, keep, lens, capacity, code):
    tree = _rows((2, 2, 1, 12, 64), 4).to(device)
    codes = torch.zeros((2, 2, 1, 2 * capacity, 32), dtype=torch.uint8, device=device)
    scales = torch.zeros((2, 2, 1, 2 * capacity, 2), dtype=torch.uint8, device=device)
    lengths, status = _dev(lens, device), torch.zeros(1, dtype=torch.int32, device=device)
    _call(device, tree, codes, scales, row_offset=_dev([0, 6, 12], device),
          keep_rows=_dev(keep, device), keep_len=_dev([2, 2], device),
          prefix_start=_dev([0, capacity], device, torch.int64), lengths=lengths,
          capacity=capacity, status=status)
    assert int(status.item()) == code
    assert lengths.tolist() == [lens[0], 2]
    assert not codes[:, :, :, :capacity].any() and not scales[:, :, :, :capacity].any()
    packed, _ = M.pack(tree.cpu())
    assert torch.equal(codes[:, :, :, capacity:capacity + 2].cpu(), packed[:, :, :, [7, 8]])


def test_load_of_every_code_and_scale_and_of_views(device):
    byte = torch.arange(256, dtype=torch.uint8)
    codes = byte.repeat(16, 1).view(256, 16).to(device)           # [tokens, 16] of D = 32
    for s in (1, 2, 7, 100, 127, 128, 251, 252, 255):
        scales = torch.full((256, 1), s, dtype=torch.uint8, device=device)
        got = ops.kv_load_mx4(codes, scales).double().cpu()
        assert torch.equal(torch.nan_to_num(got, nan=-77.0),
                           torch.nan_to_num(M.values(codes, scales), nan=-77.0)), s
    g = torch.Generator().manual_seed(8)
    codes = torch.randint(0, 256, (3, 2, 50, 64), generator=g).to(torch.uint8).to(device)
    scales = torch.randint(100, 140, (3, 2, 50, 4), generator=g).to(torch.uint8).to(device)
    want = M.values(codes, scales)
    assert torch.equal(ops.kv_load_mx4(codes, scales).double().cpu(), want)
    span = ops.kv_load_mx4(codes[1, :, 7:30], scales[1, :, 7:30])
    assert torch.equal(span.double().cpu(), want[1, :, 7:30])
    out = torch.full((3, 2, 50, 128), 9.0, dtype=torch.bfloat16, device=device)
    ops.kv_load_mx4(codes[0, :, :1], scales[0, :, :1], out=out[0, :, :1])
    assert torch.equal(out[0, :, :1].double().cpu(), want[0, :, :1])
    assert (out[0, :, 1:] == 9).all() and (out[1:] == 9).all()
    assert ops.kv_load_mx4(codes[:, :, :0], scales[:, :, :0]).shape == (3, 2, 0, 128)
    with pytest.raises(ValueError):
        ops.kv_load_mx4(codes[:, :, 5:9], scales[:, :, 5:8])
    with pytest.raises(ValueError):
        ops.kv_load_mx4(codes[::2].transpose(0, 1), scales[::2].transpose(0, 1))
