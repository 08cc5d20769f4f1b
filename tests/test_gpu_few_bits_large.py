"""Offsets beyond 32 bits: long 4-bit arenas, many rows, large weights.  Only what the
calls read or write is filled; results are compared at the far end, against the plain
forms and bounds of the operators' own tests."""
import pytest
import torch

from specgrove_amd import ops
from tests import mx4_cases as M
from tests.test_gpu_mx4_attention import Wave

pytestmark = pytest.mark.gpu

FAR = (1 << 32) // 64 + 1000   # tokens of 64 code bytes: 4 GiB and a little


def _arena(device, heads, tokens, dim):
    return (torch.empty((heads, tokens, dim // 2), dtype=torch.uint8, device=device),
            torch.empty((heads, tokens, dim // 32), dtype=torch.uint8, device=device))


def test_attention_at_the_end_of_a_long_arena(device):
    w = Wave(device, [700, 90], [5, 40], 8, 2, 128, seed=31)
    want = w.run()
    for t in range(2):
        codes, scales = _arena(device, 2, FAR + w.codes[t].shape[1], 128)
        codes[:, FAR:], scales[:, FAR:] = w.codes[t], w.scales[t]
        w.codes[t], w.scales[t] = codes, scales
    w.meta[1] += FAR
    assert torch.equal(w.run(), want)


def test_commit_and_load_at_the_end_of_a_long_arena(device):
    rows, dim = 40, 128
    tree = torch.randn((2, rows, 2, dim), generator=torch.Generator().manual_seed(2)).to(
        torch.bfloat16).to(device)
    arenas = [_arena(device, 2, FAR + 64, dim) for _ in range(2)]

    def at(tensors):
        return ops.pointer_array(list(tensors), device)

    codes, scales = arenas[0]
    ops.kv_commit_mx4(
        at([arenas[0][0]]), at([arenas[0][1]]), at([arenas[1][0]]), at([arenas[1][1]]),
        at([tree[0]]), at([tree[1]]), num_kv_heads=2, head_dim=dim,
        code_head_stride=codes.stride(0), code_token_stride=codes.stride(1),
        scale_head_stride=scales.stride(0), scale_token_stride=scales.stride(1),
        tree_row_stride=tree.stride(1), tree_head_stride=tree.stride(2),
        row_offset=torch.tensor([0, rows], dtype=torch.int32, device=device), keep_rows=None,
        keep_len=torch.tensor([rows], dtype=torch.int32, device=device),
        prefix_start=torch.tensor([FAR], device=device),
        lengths=torch.tensor([3], dtype=torch.int32, device=device), capacity=64)
    for (codes, scales), t in zip(arenas, tree):
        packed, by = M.pack(t.transpose(0, 1).cpu())
        span = slice(FAR + 3, FAR + 3 + rows)
        assert torch.equal(codes[:, span].cpu(), packed)
        assert torch.equal(scales[:, span].cpu(), by)
        far = ops.kv_load_mx4(codes[:, span], scales[:, span])
        assert torch.equal(far.cpu(), M.values(packed, by).to(torch.bfloat16))
    # Every token of an arena whose values pass 4 GiB, head by head.
    codes, scales = (torch.zeros((3, (1 << 24) + 7, w), dtype=torch.uint8, device=device)
                     for w in (64, 4))
    g = torch.Generator().manual_seed(5)
    codes[2, -9:] = torch.randint(0, 256, (9, 64), generator=g).to(torch.uint8).to(device)
    scales[2, -9:] = torch.randint(100, 140, (9, 4), generator=g).to(torch.uint8).to(device)
    values = ops.kv_load_mx4(codes, scales)
    assert torch.equal(values[2, -9:].double().cpu(), M.values(codes[2, -9:], scales[2, -9:]))


def _ends(device, rows, n, k, last_rows, last_columns):
    """The product of random rows and weights, and its last rows and columns in 64 bits
    with their bound (that of the products' own tests)."""
    g = torch.Generator(device=device).manual_seed(rows + n)
    x = torch.randn((rows, k), generator=g, device=device, dtype=torch.bfloat16)
    fx = ops.quantize_fp8(x)
    del x
    w = torch.randint(0, 120, (n, k), generator=g, device=device, dtype=torch.uint8)
    w = w.view(torch.float8_e4m3fn)
    ws = torch.rand((-(-n // 128), -(-k // 128)), generator=g, device=device) + 0.5
    got = ops.fp8_matmul(fx, ops.pack_fp8_weight(w, ws))
    xv = ops.Fp8Rows(fx.codes[-last_rows:], fx.scales[-last_rows:]).dequantize().double()
    ws = ws.repeat_interleave(128, 0)[:n][-last_columns:].repeat_interleave(128, 1)[:, :k]
    wv = w[-last_columns:].double() * ws.double()
    want = xv @ wv.T.contiguous()
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -14 * (xv.abs() @ wv.abs().T.contiguous())
    err = (got[-last_rows:, -last_columns:].double() - want).abs()
    return float((err / bound).max())


@pytest.mark.parametrize("rows,n,k", [
    (290000, 136, 16384),      # rows and codes
    (40, 140000, 32768),       # a weight, few rows
    (300, 140000, 32768),      # a weight, tiles
])
def test_products_beyond_32_bits(device, rows, n, k):
    assert _ends(device, rows, n, k, min(rows, 300), min(n, 200)) <= 1.0
