"""Refusals of the 4-bit cache's and the e4m3 projections' entry points, by the host
checks alone (no GPU: nothing is launched)."""
import ctypes

import pytest
import torch

from specgrove_amd import _lib, ops, target
from specgrove_amd.cache import Mx4RequestCachePool, RequestCache

EINVAL = -1


def _code(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    assert (rc == 0) or lib.sg_last_error()
    return rc


def _commit(**fields):
    a = _lib.SgKvCommitMx4Args()
    good = dict(num_layers=2, num_requests=3, num_kv_heads=2, head_dim=64,
                k_code_layers_dev=256, k_scale_layers_dev=256, v_code_layers_dev=256,
                v_scale_layers_dev=256, code_head_stride=3200, code_token_stride=32,
                scale_head_stride=200, scale_token_stride=2, k_tree_layers_dev=256,
                v_tree_layers_dev=256, tree_row_stride=128, tree_head_stride=64,
                row_offset_dev=256, keep_rows_dev=256, keep_stride=4, keep_len_dev=256,
                prefix_start_dev=256, lengths_dev=256, capacity=100, status_dev=256)
    for name, value in {**good, **fields}.items():
        setattr(a, name, value)
    return _code("sg_kv_commit_mx4", ctypes.byref(a), None)


@pytest.mark.parametrize("fields", [
    dict(num_layers=-1), dict(num_requests=-1), dict(num_kv_heads=0), dict(head_dim=48),
    dict(head_dim=0), dict(capacity=0), dict(keep_stride=0), dict(tree_row_stride=60),
    dict(tree_head_stride=4), dict(code_token_stride=30), dict(code_head_stride=3201),
    dict(num_requests=65536), dict(num_layers=65536), dict(k_code_layers_dev=0),
    dict(v_scale_layers_dev=0), dict(k_tree_layers_dev=0), dict(row_offset_dev=0),
    dict(keep_len_dev=0), dict(prefix_start_dev=0), dict(lengths_dev=0),
    dict(num_kv_heads=1 << 28)])
def test_commit_refusals(fields):
    assert _commit(**fields) == EINVAL


def test_commit_of_nothing_is_nothing():
    assert _commit(num_layers=0) == 0 and _commit(num_requests=0) == 0
    assert _code("sg_kv_commit_mx4", None, None) == EINVAL


def _load(codes=256, ch=3200, ct=32, scales=256, sh=200, st=2, outer=2, tokens=100, dim=64,
          out=256, oh=6400, ot=64):
    return _code("sg_kv_load_mx4", codes, ch, ct, scales, sh, st, outer, tokens, dim, out, oh,
                 ot, None)


@pytest.mark.parametrize("fields", [
    dict(codes=0), dict(scales=0), dict(out=0), dict(dim=48), dict(dim=0), dict(outer=-1),
    dict(tokens=-1), dict(codes=258), dict(ct=30), dict(ch=3201), dict(out=264),
    dict(ot=60), dict(oh=6404)])
def test_load_refusals(fields):
    assert _load(**fields) == EINVAL


def test_load_of_nothing_is_nothing():
    assert _load(outer=0) == 0 and _load(tokens=0) == 0


def _rows_out(**fields):
    out = _lib.SgFp8RowsOut(256, 256, 256, 4)
    for name, value in fields.items():
        setattr(out, name, value)
    return out


@pytest.mark.parametrize("x,stride,rows,columns,out", [
    (0, 256, 4, 256, {}), (264, 256, 4, 256, {}), (256, 252, 4, 256, {}), (256, 248, 4, 256, {}),
    (256, 256, -1, 256, {}), (256, 256, 4, 252, {}), (256, 256, 4, 0, {}),
    (256, 256, 4, 256, dict(codes_dev=0)), (256, 256, 4, 256, dict(scales_dev=0)),
    (256, 256, 4, 256, dict(scale_stride=3)), (256, 256, 4, 256, dict(code_stride=128))])
def test_quantizer_refusals(x, stride, rows, columns, out):
    o = _rows_out(**out)
    assert _code("sg_fp8_quantize_rows", x, stride, rows, columns, ctypes.byref(o),
                 None) == EINVAL
    assert _code("sg_fp8_quantize_rows", 256, 256, 4, 256, None, None) == EINVAL
    assert _code("sg_fp8_quantize_rows", 256, 256, 0, 256, ctypes.byref(_rows_out()), None) == 0


def _matmul(**fields):
    a = _lib.SgFp8MatmulArgs(4, 256, 256, 0, 256, 256, 256, 4, 256, 256, 256, 256, 0, 0)
    for name, value in fields.items():
        setattr(a, name, value)
    return _code("sg_fp8_matmul", ctypes.byref(a), None)


@pytest.mark.parametrize("fields", [
    dict(num_rows=-1), dict(n=0), dict(k=0), dict(n=(1 << 24) + 1), dict(k=(1 << 24) + 1),
    dict(codes_dev=0), dict(scales_dev=0), dict(weight_dev=0), dict(weight_scales_dev=0),
    dict(out_dev=0), dict(scale_stride=3), dict(out_stride=248), dict(out_stride=260),
    dict(code_stride=128), dict(code_stride=(1 << 24) + 16), dict(codes_dev=264), dict(out_dev=264), dict(weight_dev=264)])
def test_matmul_refusals(fields):
    assert _matmul(**fields) == EINVAL


def test_matmul_of_no_rows_is_nothing():
    assert _matmul(num_rows=0, codes_dev=0, scales_dev=0, out_dev=0) == 0


def test_sizes_without_a_gpu():
    lib = _lib.load()
    assert lib.sg_fp8_packed_bytes(256, 256) == 256 * 256
    assert lib.sg_fp8_packed_bytes(0, 256) <= 0 and lib.sg_fp8_packed_bytes(256, -1) <= 0
    assert lib.sg_fp8_matmul_workspace_bytes(0, 256, 256) == 0


def test_tensors_that_are_not_on_the_gpu():
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    codes = torch.zeros((2, 8, 32), dtype=torch.uint8)
    scales = torch.zeros((2, 8, 2), dtype=torch.uint8)
    for call in (lambda: ops.quantize_fp8(x), lambda: target.silu_mul_fp8(x),
                 lambda: target.add_rmsnorm_fp8(x, x[0], 1e-6),
                 lambda: ops.kv_load_mx4(codes, scales),
                 lambda: ops.pack_fp8_weight(*ops.quantize_fp8_weight(x))):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    with pytest.raises(ValueError, match="Fp8Rows"):
        ops.fp8_matmul(x, x)
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16)
    kv = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    plan = ops.plan_attention([0, 4], [8], 4, 2, 64)
    meta = [torch.tensor(v, dtype=d) for v, d in (([0, 4], torch.int32), ([0], torch.int64),
                                                  ([8], torch.int32), ([-1, 0, 1, 2], torch.int32))]
    with pytest.raises(ValueError, match="HIP device"):
        ops.tree_attention_mx4(q, codes, scales, codes, scales, kv, kv, *meta, plan)


def test_the_pool_lives_on_the_gpu():
    cache = RequestCache()
    rows = torch.zeros((1, 2, 5, 64), dtype=torch.bfloat16)
    cache.update(rows, rows, 0)
    with pytest.raises(ValueError, match="GPU"):
        Mx4RequestCachePool([cache], 8)
    with pytest.raises(ValueError, match="At least one"):
        Mx4RequestCachePool([], 8)


def test_a_4_bit_cache_is_a_persistent_one():
    from tests.test_wave_loop_host import _loop, _proposer
    p, _ = _proposer()
    good = dict(tree_budget=12, row_cap=4, row_budget=64)
    _loop(p, **good)    # (the helper's loops are not persistent)
    for bad in (dict(cache_format="fp8"), dict(cache_format="mx4")):
        with pytest.raises(ValueError, match="experiment contract"):
            _loop(p, **{**good, **bad})


def test_weights_quantized_on_the_host():
    """e4m3 codes of a weight's blocks: the largest magnitude at 448, every value within
    a half step (2^-4 of it, or of the least normal value) of the weight, and the
    reciprocal's rounding (2^-23) beside it."""
    g = torch.Generator().manual_seed(3)
    w = torch.randn((200, 333), generator=g) * torch.logspace(-3, 3, 200)[:, None]
    w[130:, 128:256] = 0.0
    codes, scales = ops.quantize_fp8_weight(w)
    assert codes.shape == w.shape and scales.shape == (2, 3)
    grid = scales.repeat_interleave(128, 0).repeat_interleave(128, 1)[:200, :333]
    x = (w / grid).double()
    off = (codes.double() - x).abs()
    assert (off <= x.abs().clamp_min(2.0 ** -6) * 2.0 ** -4 * (1 + 2.0 ** -16)).all()
    for i in range(2):
        for j in range(3):
            block = codes[128 * i:128 * i + 128, 128 * j:128 * j + 128].float()
            assert block.abs().max() in (0.0, 448.0)


def _wave(seed):
    import random
    rng = random.Random(seed)
    n = rng.choice([1, 2, 7, 40])
    longest = rng.choice([40, 700, 9000, 40000])
    lengths = [rng.choice([0, 1, rng.randint(0, longest), longest]) for _ in range(n)]
    rows = [rng.choice([0, 1, 1, 16, 33, 64, 200, 256]) for _ in range(n)]
    hq, hkv = rng.choice([(4, 2), (32, 8), (8, 8), (16, 1), (64, 8)])
    return lengths, rows, hq, hkv, rng.choice([64, 128])


@pytest.mark.parametrize("seed", range(40))
def test_plans_over_a_4_bit_cache_cover_the_wave(seed):
    """Every row tile of every request and kv head sees its whole prefix once, in pieces
    of at least 256 keys, and its tree once; work lists and merge groups are whole."""
    lengths, rows, hq, hkv, dim = _wave(seed)
    offset = [0]
    for r in rows:
        offset.append(offset[-1] + r)
    plan = ops.plan_attention_mx4(offset, lengths, hq, hkv, dim)
    ops.check_plan(plan, offset, lengths)
    header, units, merges, bins = ops.decode_plan(plan)
    assert plan.units == len(bins) - 1 and plan.merges == len(merges)
    if len(units):
        assert bins[0] == 0 and bins[-1] == len(units) and (bins[1:] > bins[:-1]).all()
    full = 128 // (hq // hkv)
    # Rows of a unit: a full row tile, or half of one where the planner cut by rows.
    tile = {int(u[0]): full // 2 if u[7] & 2 else full for u in units}
    pieces, slots = {}, set()
    for u in units.tolist():
        req, head, row, count, begin, end, partial, flags, group, splits, first, _ = u
        rpt = tile[req]
        assert row % rpt == 0 and count == min(rpt, rows[req] - row)
        assert flags & 2 == (2 if rpt < full else 0) and flags < 4
        pieces.setdefault((req, head, row), []).append((begin, end, flags & 1, group, splits))
        if partial >= 0:
            assert partial not in slots and first <= partial < first + splits
            slots.add(partial)
            assert merges[group].tolist()[:6] == [req, head, row, count, first, splits]
        else:
            assert group == -1 and splits == 1
    want = {(i, h, r) for i in range(len(rows)) for h in range(hkv)
            for r in range(0, rows[i], tile.get(i, full))}
    assert set(pieces) == want
    for (req, _, _), p in pieces.items():
        p.sort()
        assert p[0][0] == 0 and p[-1][1] == lengths[req]
        assert all(a[1] == b[0] for a, b in zip(p, p[1:]))
        assert [x[2] for x in p] == [0] * (len(p) - 1) + [1]
        assert all(x[4] == len(p) for x in p)
        assert len(p) == 1 or all(x[1] - x[0] >= 224 for x in p)  # 256 less a 32-key tile
    assert slots == set(range(len(slots)))
    assert plan.workspace_bytes == 4 * 128 * (dim + 2) * len(slots)


def test_a_long_unit_is_cut_for_4_bits_and_refusals():
    plan = ops.plan_attention_mx4([0, 1, 2], [32768, 300], 32, 8, 128)
    assert plan.merges > 0 and plan.in_mx4() is plan
    given = ops.plan_attention([0, 1], [32768], 32, 8, 128, 5)
    assert given.in_mx4() is given
    for bad in (([0, 1], [-1], 32, 8, 128), ([0, 257], [5], 32, 8, 128), ([1, 2], [5], 32, 8, 128),
                ([0, 1], [5], 32, 5, 128), ([0, 1], [5], 32, 8, 96), ([0, 1], [5, 6], 32, 8, 128)):
        with pytest.raises(ValueError):
            ops.plan_attention_mx4(*bad)
    assert ops.plan_attention_mx4([0], [], 32, 8, 128).units == 0


def test_devices_are_compared(monkeypatch):
    class On:
        def __init__(self, index):
            self.device = torch.device("cuda", index)

        def get_device(self):
            return self.device.index

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    ops._check_current(On(1), "x", On(1), None)
    with pytest.raises(ValueError, match="not the current device"):
        ops._check_current(On(0), "x")
    with pytest.raises(ValueError, match="x on cuda:1"):
        ops._check_current(On(1), "x", None, On(0))
