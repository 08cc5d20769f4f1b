"""The e4m3 product's choice of a kernel, on the host."""
from specgrove_amd import _lib
from tests.fp8_shapes import FEW, TILES


def _form(rows, k, n):
    got = _lib.load().sg_fp8_matmul_form(rows, n, k)
    assert got >= 16
    return got % 16, got // 16


def test_the_tested_sizes_reach_every_form():
    few = {_form(*s) for s in FEW}
    assert few == {(f, 1) for f in range(4)}
    tiles = {}
    for s in TILES:
        form, splits = _form(*s)
        tiles.setdefault(form, set()).add(splits > 1)
    assert tiles == {f: {False, True} for f in range(4, 10)}


def test_the_workspace_is_that_of_the_splits():
    lib = _lib.load()
    for rows, k, n in FEW + TILES:
        _, splits = _form(rows, k, n)
        want = 0 if splits == 1 else splits * rows * (-(-n // 128) * 128) * 4
        assert lib.sg_fp8_matmul_workspace_bytes(rows, n, k) == want


def test_sizes_without_a_form():
    lib = _lib.load()
    assert lib.sg_fp8_matmul_form(0, 256, 256) == -1
    assert lib.sg_fp8_matmul_form(-1, 256, 256) == -1
    assert lib.sg_fp8_matmul_form(4, 0, 256) == -1
    assert lib.sg_fp8_matmul_form(4, 256, (1 << 24) + 1) == -1


def test_a_large_weight_is_not_read_twice():
    """33 to 64 rows: the few-rows kernel (forms 0 to 3) up to 48 MiB of weight, whichever
    way the weight is long."""
    for rows in (33, 64):
        for k, n in ((2560, 6144), (4096, 12288), (12288, 4096), (4100, 11900)):
            assert _form(rows, k, n)[0] < 4
        for k, n in ((12288, 6144), (12288, 12288), (4096, 16384), (4096, 12289), (12289, 4096)):
            assert _form(rows, k, n)[0] >= 4
    assert _form(32, 12288, 12288)[0] < 4
