"""e4m3 rows, weights and products against float64.

Tolerances, before any run.  Quantized rows: x * (448 / m) is the same two fp32
roundings on any machine, so codes and scales of given rows are compared bit for
bit; after a norm or SiLU (whose sums and exponentials may round differently) a
value is within half an e4m3 step of the float64 result, 2^-4 of it or 2^-10 of the
scale, plus 2^-18 of it for the fp32 arithmetic.  Products: the result's rounding
is 2^-8 of it; the matrix instruction adds 128 products with less than fp32's
precision (an error of up to 2.3e-5 of the sum of their magnitudes was seen over
e4m3's whole range), so 2^-14 of sum |x w| is allowed for sums.
"""
import numpy as np
import pytest
import torch

from specgrove_amd import ops, target

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _quantized(x):
    """codes and scales of fp32 rows on the CPU, columns padded to 128."""
    b = torch.nn.functional.pad(x, (0, -x.shape[1] % 128)).unflatten(1, (-1, 128))
    m = b.abs().amax(2, keepdim=True).clamp_min(2.0 ** -100)
    r = torch.full_like(m, 448) / m  # (a number over a tensor is a product with 1 / m)
    return (b * r).to(F8).flatten(1), (m / 448).squeeze(2)


def _rows(rows, k, seed):
    x = torch.randn((rows, k), generator=_gen(seed))
    return (x * (1 + 30 * (torch.rand(k, generator=_gen(seed + 1)) < 0.02))).to(torch.bfloat16)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("rows,k", [(1, 8), (3, 128), (2, 136), (5, 2048), (4, 2056), (7, 4096),
                                    (300, 1000), (2, 12288)])
def test_quantized_rows_bit_for_bit(device, rows, k):
    wide = _rows(rows, k + 16, k)
    wide[0, 8:16] = 0
    if rows > 1:
        wide[1] = 0                                    # a row of zeros
        wide[-1, 8:] *= 2.0 ** 100
    if rows > 2:
        wide[2] = (wide[2].float() * 2.0 ** -120).to(torch.bfloat16)
    x = wide[:, 8:8 + k]
    got = ops.quantize_fp8(wide.to(device)[:, 8:8 + k])
    codes, scales = _quantized(x.float())
    assert got.shape == (rows, k)
    padded = got.codes.as_strided((rows, codes.shape[1]), (codes.shape[1], 1))
    assert torch.equal(_bytes(padded.cpu()), _bytes(codes))
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.dequantize().cpu(),
                       (codes.float() * scales.repeat_interleave(128, 1))[:, :k])


def test_infinities_and_nans_stay_in_their_block(device):
    x = _rows(4, 384, 1)
    x[1, 130] = float("inf")
    x[2, 3] = float("nan")
    rows = ops.quantize_fp8(x.to(device))
    bad = ~torch.isfinite(rows.dequantize().cpu())
    assert bad[1, 128:256].any() and bad[2, :128].any()
    bad[1, 128:256] = False
    bad[2, :128] = False
    assert not bad.any()
    w, ws = ops.quantize_fp8_weight(torch.randn((130, 384), generator=_gen(2)))
    out = ops.fp8_matmul(rows, ops.pack_fp8_weight(w.to(device), ws.to(device)))
    assert not torch.isfinite(out[1:3]).any() and torch.isfinite(out[[0, 3]]).all()


def _close_rows(got, want, what):
    """Half an e4m3 step of the float64 rows `want`."""
    want = want.double()
    s = got.scales.double().cpu().repeat_interleave(128, 1)[:, :want.shape[1]]
    err = (got.dequantize().double().cpu() - want).abs()
    bound = want.abs() * (2.0 ** -4 + 2.0 ** -18) + s * 2.0 ** -10
    assert bool((err <= bound).all()), (what, float((err / bound).max()))


@pytest.mark.parametrize("rows,hidden", [(1, 8), (3, 256), (5, 2040), (2, 2048), (2, 2560),
                                         (300, 4096), (2, 8192)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_add_rmsnorm_fp8(device, rows, hidden, with_residual):
    x = (torch.randn((rows, hidden), generator=_gen(hidden)) * 3).to(torch.bfloat16)
    res = torch.randn((rows, hidden), generator=_gen(1)).to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(hidden, generator=_gen(2))).to(torch.bfloat16)
    total = (x + res) if with_residual else x
    f = total.double()
    want = f / (f.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    got, kept = target.add_rmsnorm_fp8(x.to(device), w.to(device), 1e-6,
                                       res.to(device) if with_residual else None, want_sum=True)
    assert torch.equal(kept.cpu(), total)
    _close_rows(got, want, "norm")
    again = target.add_rmsnorm_fp8(x.to(device), w.to(device), 1e-6,
                                   res.to(device) if with_residual else None)
    assert torch.equal(_bytes(again.codes), _bytes(got.codes))


@pytest.mark.parametrize("rows,inter", [(1, 8), (3, 768), (2, 2056), (77, 9728), (2, 12288)])
def test_silu_mul_fp8(device, rows, inter):
    gu = (torch.randn((rows, 2 * inter), generator=_gen(inter)) * 4).to(torch.bfloat16)
    gate, up = gu.double().chunk(2, 1)
    _close_rows(target.silu_mul_fp8(gu.to(device)), gate * torch.sigmoid(gate) * up, "silu")


def _product(device, rows, k, n, seed):
    x = _rows(rows, k, seed)
    w = torch.randn((n, k), generator=_gen(seed + 2)) * (1 + torch.rand((n, 1), generator=_gen(3)))
    wq, ws = ops.quantize_fp8_weight(w)
    fx = ops.quantize_fp8(x.to(device))
    packed = ops.pack_fp8_weight(wq.to(device), ws.to(device))
    xv = fx.dequantize().double()
    wv = wq.to(device).double() * ws.to(device).double().repeat_interleave(
        128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want = xv @ wv.T.contiguous()
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -14 * (xv.abs() @ wv.abs().T.contiguous())
    return fx, packed, want, bound


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 129, 257, 600])
@pytest.mark.parametrize("k,n", [(128, 128), (8, 1), (264, 130), (1000, 777), (4096, 4096)])
def test_products(device, rows, k, n):
    fx, packed, want, bound = _product(device, rows, k, n, rows + k)
    got = ops.fp8_matmul(fx, packed)
    assert got.shape == (rows, n) and got.dtype == torch.bfloat16
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    assert torch.equal(got, ops.fp8_matmul(fx, packed))


@pytest.mark.parametrize("rows,k,n", [(2048, 4096, 6144), (1500, 12288, 2560), (4096, 1024, 4096),
                                      (300, 2568, 50257), (1, 12288, 4096), (40, 4096, 24576)])
def test_large_products(device, rows, k, n):
    fx, packed, want, bound = _product(device, rows, k, n, 5)
    err = (ops.fp8_matmul(fx, packed).double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def test_out_is_written_where_it_is_and_nowhere_else(device):
    fx, packed, want, bound = _product(device, 37, 256, 203, 9)
    wide = torch.full((39, 240), 3.0, dtype=torch.bfloat16, device=device)
    out = wide[1:38, 16:219]
    assert ops.fp8_matmul(fx, packed, out=out).data_ptr() == out.data_ptr()
    assert bool(((out.double() - want).abs() <= bound).all())
    wide[1:38, 16:219] = 3.0
    assert (wide == 3).all()
    none = ops.quantize_fp8(torch.empty((0, 256), dtype=torch.bfloat16, device=device))
    assert ops.fp8_matmul(none, packed).shape == (0, 203)


def test_rows_of_rows_streams_and_graphs(device):
    fx, packed, want, bound = _product(device, 96, 2560, 1024, 11)
    some = ops.Fp8Rows(fx.codes[32:], fx.scales[32:])      # rows of a larger wave
    got = ops.fp8_matmul(some, packed)
    assert bool(((got.double() - want[32:]).abs() <= bound[32:]).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = ops.fp8_matmul(fx, packed)
    side.synchronize()
    here = ops.fp8_matmul(fx, packed)
    assert torch.equal(there, here)
    # A captured step: norm, product, SiLU, product; two graphs of one memory pool.
    x = _rows(19, 256, 12).to(device)
    norm = torch.ones(256, dtype=torch.bfloat16, device=device)
    wide = ops.pack_fp8_weight(*(t.to(device) for t in ops.quantize_fp8_weight(
        torch.randn((1536, 256), generator=_gen(13)) / 16)))
    down = ops.pack_fp8_weight(*(t.to(device) for t in ops.quantize_fp8_weight(
        torch.randn((256, 768), generator=_gen(14)) / 28)))

    def step():
        h, total = target.add_rmsnorm_fp8(x, norm, 1e-6, want_sum=True)
        return total + ops.fp8_matmul(target.silu_mul_fp8(ops.fp8_matmul(h, wide)), down)

    step()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            outs.append(step())
    for k in range(3):
        x.copy_(_rows(19, 256, 20 + k).to(device))
        eager = step()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager), k


def test_weight_quantization(device):
    w = torch.randn((200, 300), generator=_gen(15))
    w[:, 140] *= 50
    codes, scales = ops.quantize_fp8_weight(w)
    assert codes.shape == (200, 300) and scales.shape == (2, 3)
    back = codes.double() * scales.double().repeat_interleave(128, 0)[:200].repeat_interleave(
        128, 1)[:, :300]
    err = (back - w.double()).abs()
    step = scales.double().repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :300]
    assert bool((err <= w.double().abs() * (2.0 ** -4 + 2.0 ** -20) + step * 2.0 ** -10).all())
    on_gpu = ops.quantize_fp8_weight(w.to(device))
    assert torch.equal(_bytes(on_gpu[0].cpu()), _bytes(codes))


def test_refusals(device):
    fx, packed, _, _ = _product(device, 4, 256, 64, 16)
    x = _rows(4, 256, 1).to(device)
    other, _, _, _ = _product(device, 4, 128, 64, 17)
    for call in (lambda: ops.quantize_fp8(x.float()),
                 lambda: ops.quantize_fp8(x[:, :100]),
                 lambda: ops.quantize_fp8(x[:, 1:9]),
                 lambda: ops.quantize_fp8(x.T),
                 lambda: target.silu_mul_fp8(x[:, :24]),
                 lambda: target.add_rmsnorm_fp8(x, x[0, :128], 1e-6),
                 lambda: target.add_rmsnorm_fp8(x, x[0], 1e-6, x[:, :128]),
                 lambda: ops.fp8_matmul(other, packed),
                 lambda: ops.fp8_matmul(x, packed),
                 lambda: ops.fp8_matmul(ops.Fp8Rows(fx.codes, fx.scales[:, :1]), packed),
                 lambda: ops.fp8_matmul(ops.Fp8Rows(fx.codes, fx.scales.contiguous()), packed),
                 lambda: ops.fp8_matmul(fx, packed, out=x[:, :32]),
                 lambda: ops.fp8_matmul(fx, packed, out=torch.empty(
                     (4, 64), dtype=torch.float32, device=device)),
                 lambda: ops.pack_fp8_weight(fx.codes, fx.scales.T),
                 lambda: ops.quantize_fp8_weight(torch.zeros(0, 4))):
        with pytest.raises(ValueError):
            call()
    thin = torch.empty((4, 250), dtype=F8, device=device)  # no padded columns behind a row
    odd = ops.pack_fp8_weight(*(t.to(device) for t in ops.quantize_fp8_weight(
        torch.randn((64, 250), generator=_gen(1)))))
    with pytest.raises(ValueError):
        ops.fp8_matmul(ops.Fp8Rows(thin, fx.scales), odd)
