"""Scores of the attention over a 4-bit cache where they are hardest: outlier columns,
large scores, wide ranges inside a block of 32 columns, and values that are no numbers.

Tolerance.  Three things put a score s = scale * sum_c k_c q_c off.  q is held as two
e4m3 values: exactly from 2^-14 of its block's largest value on, else within 2^-22 of
that.  The matrix instruction adds the products of 8 columns cut to multiples of
2^(e - 13), e the largest sum of a column's exponents: a product that has it is exact and
at least 2^e, so 8 products are off by at most 7 * 2^-13 of their largest, and a sum of
them by less than 2^-10 of sum |k q|, for each of the two terms (the second one's products
are 2^-4 of the first one's); nothing is cut where the products of 8 columns have sums of
exponents less than 2^5 apart (their last bit is 2^-7 of that at least).  fp32 sums of the
parts: 2^-20 of sum |k q| at most.  With a score off by at most D everywhere a probability
is off by a factor within exp(+-2 D), so an output by (exp(2 D) - 1) sum(p |v|), beside
what the attention's other tests allow.
"""
import pytest
import torch

from tests import mx4_cases as M
from tests.test_gpu_mx4_attention import Wave

pytestmark = pytest.mark.gpu


def _set_k(w, change):
    """Repack the prefix's K after change(values [Hkv, tokens, D])."""
    behind = w.scales[0].cpu() == 255
    k = torch.nan_to_num(M.values(w.codes[0], w.scales[0]))
    k = change(k).to(torch.bfloat16)
    codes, scales = M.pack(k)
    scales[behind] = 255
    w.codes[0], w.scales[0] = codes.to(w.device), scales.to(w.device)


def _worst(w, out, cut=2.0 ** -10):
    """The largest error against its bound, and the largest D."""
    worst, most = 0.0, 0.0
    for i in range(len(w.lengths)):
        a, b = int(w.offset[i]), int(w.offset[i + 1])
        want, bound = w.reference(i)
        at = slice(int(w.start[i]), int(w.start[i]) + int(w.lengths[i]))
        k = torch.cat([M.values(w.codes[0][:, at], w.scales[0][:, at]),
                       w.tree[0][a:b].double().cpu().transpose(0, 1)], 1)
        v = torch.cat([M.values(w.codes[1][:, at], w.scales[1][:, at]),
                       w.tree[1][a:b].double().cpu().transpose(0, 1)], 1)
        group = w.hq // w.hkv
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        q = w.q[a:b].double().cpu().transpose(0, 1)
        blocks = q.abs().unflatten(2, (-1, 32))
        most_q = blocks.amax(3, keepdim=True)
        lost = torch.where(blocks < 2.0 ** -14 * most_q, 2.0 ** -22 * most_q, 0.0).flatten(2)
        off = ((cut * (1 + 2.0 ** -4) + 2.0 ** -20) * (q.abs() @ k.abs().transpose(1, 2))
               + lost @ k.abs().transpose(1, 2)) * w.dim ** -0.5
        d = off.amax(2).transpose(0, 1)[..., None]
        # sum(p |v|) again, from the bound: it is (bound - 2^-8 |out|) / (2^-8 + 2^-12).
        mass = (bound - 2.0 ** -8 * want.abs()) / (2.0 ** -8 + 2.0 ** -12)
        bound = bound + torch.expm1(2 * d) * mass
        err = (out[a:b].double().cpu() - want).abs()
        assert torch.isfinite(out[a:b]).all()
        worst = max(worst, float((err / bound).max()))
        most = max(most, float(d.max()))
    return worst, most


@pytest.mark.parametrize("ratio", [10, 13, 14, 17, 20])
@pytest.mark.parametrize("dim,rows", [(64, [3, 40]), (128, [1, 7]), (128, [16, 33])])
def test_one_large_q_channel_that_meets_no_key(device, ratio, dim, rows):
    """Every block of q has a channel 2^ratio times the others' least magnitude; all
    keys are 0 there, so the scores are the other channels' alone."""
    w = Wave(device, [300, 129], rows, 8, 2, dim, seed=ratio + dim)
    lone = torch.arange(5, dim, 32)
    g = torch.Generator().manual_seed(ratio)
    q = (1 + torch.rand(w.q.shape, generator=g)) * torch.randn(w.q.shape, generator=g).sign()
    q = q.to(torch.bfloat16)
    q[..., lone] = 2.0 ** ratio
    w.q = q.to(device)

    def clear(k):
        k[..., lone] = 0
        return k

    _set_k(w, clear)
    w.tree[0][..., lone.to(device)] = 0
    # |q| in [1, 2) and keys of 1/2 to 6 times their scale: nothing is cut.
    worst, most = _worst(w, w.run(), cut=0.0)
    assert worst <= 1.0
    assert ratio > 14 or most < 0.001  # the bound itself says something


@pytest.mark.parametrize("dim,rows", [(64, [5, 40]), (128, [1, 16]), (128, [33, 64])])
@pytest.mark.parametrize("kind", ["keys", "queries", "both", "large", "wide"])
def test_outliers_and_large_scores(device, kind, dim, rows):
    w = Wave(device, [700, 95], rows, 8, 2, dim, seed=dim + len(kind))
    lone = torch.tensor([3, 40])
    g = torch.Generator().manual_seed(7)
    if kind in ("keys", "both"):        # a few columns far larger, as keys have them
        def grow(k):
            k[..., lone] *= 30
            return k
        _set_k(w, grow)
    if kind in ("queries", "both"):
        w.q[..., lone.to(device)] *= 20.0 if kind == "queries" else 4.0
    if kind == "large":                 # scores of some tens
        w.q *= 8.0
    if kind == "wide":                  # 2^-16 to 1 of the block's largest, everywhere
        w.q *= torch.exp2(torch.randint(-16, 1, w.q.shape, generator=g)).to(w.q)
        _set_k(w, lambda k: k * torch.exp2(torch.randint(-6, 1, k.shape, generator=g)))
    worst, _ = _worst(w, w.run())
    assert worst <= 1.0


@pytest.mark.parametrize("rows", [[1, 3], [16, 3], [33, 3]])
def test_a_cached_key_that_is_no_number_reaches_its_heads_rows(device, rows):
    w = Wave(device, [70, 40], rows, 8, 2, 128, seed=3)
    clean = w.run()
    w.scales[0][1, 11, 2] = 255          # K of token 11 of request 0, kv head 1
    got = w.run()
    assert torch.isnan(got[:rows[0], 4:]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[:rows[0], 4:] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("rows", [[4, 3], [16, 3], [33, 3]])
def test_a_query_that_is_no_number_gives_its_own_vector(device, rows, bad):
    w = Wave(device, [70, 40], rows, 8, 2, 128, seed=4)
    clean, bound = (torch.cat(t) for t in zip(*(w.reference(i) for i in range(2))))
    w.q[2, 5, 77] = bad
    got = w.run()
    assert torch.isnan(got[2, 5]).all()
    keep = torch.ones(got.shape, dtype=torch.bool)
    keep[2, 5] = False
    err = (got.double().cpu() - clean).abs()
    assert bool((err <= bound)[keep].all())
