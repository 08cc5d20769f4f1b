"""Tree attention over a 4-bit cache against a float64 restatement.

Tolerance, before any run: the probabilities are rounded to bf16 for the matrix
product and the result once more, each by at most 2^-8 of the value, so an output
is off by at most 2^-8 sum(p |v|) + 2^-8 |out|; the fp32 products, sums and
exponentials before that (relative errors of 2^-24 over a few hundred terms, scores
below 2^7) stay below 2^-12 sum(p |v|).
"""
import numpy as np
import pytest
import torch

from specgrove_amd import ops
from specgrove_amd import workloads as W
from tests import mx4_cases as M

pytestmark = pytest.mark.gpu


class Wave:
    """A wave's inputs on the device, its cache packed into 4 bits; what lies
    behind a request's last token is NaN."""

    def __init__(self, device, lengths, rows, hq, hkv, dim, seed=0, tree="random", capacity=None):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.lengths = np.asarray(lengths, np.int32)
        self.parents = [list(range(-1, r - 1)) if tree == "chain" else
                        W.random_parent_tree(r, rng, max_depth=16) for r in rows]
        self.offset = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.cap = capacity or int(max(lengths)) + 5
        self.hq, self.hkv, self.dim = hq, hkv, dim
        total, n = int(self.offset[-1]), len(rows)
        self.start = np.arange(n, dtype=np.int64) * self.cap

        def rand(*shape, scale=1.0):
            return (torch.randn(shape, generator=g) * scale).to(torch.bfloat16)

        self.q = rand(total, hq, dim, scale=1.5).to(device)
        self.tree = [rand(total, hkv, dim).to(device) for _ in range(2)]
        behind = np.concatenate([np.arange(self.cap) >= L for L in self.lengths])
        self.codes, self.scales = [], []
        for _ in range(2):
            c, s = M.pack(rand(hkv, n * self.cap, dim))
            s[:, torch.from_numpy(behind)] = 255
            self.codes.append(c.to(device))
            self.scales.append(s.to(device))
        self.meta = [torch.from_numpy(np.ascontiguousarray(a)).to(device) for a in (
            self.offset, self.start, self.lengths,
            np.concatenate([np.asarray(p, np.int32) for p in self.parents]))]
        self.device = device

    def plan(self, target=0):
        return ops.plan_attention(self.offset, self.lengths, self.hq, self.hkv, self.dim,
                                  target).to(self.device)

    def run(self, plan=None, **kw):
        return ops.tree_attention_mx4(self.q, self.codes[0], self.scales[0], self.codes[1],
                                      self.scales[1], *self.tree, *self.meta,
                                      plan or self.plan(), **kw)

    def reference(self, i, scale=None):
        """(out, bound) of request i, [rows, Hq, D] float64."""
        a, b = int(self.offset[i]), int(self.offset[i + 1])
        at = slice(int(self.start[i]), int(self.start[i]) + int(self.lengths[i]))
        k, v = (torch.cat([M.values(self.codes[t][:, at], self.scales[t][:, at]),
                           self.tree[t][a:b].double().cpu().transpose(0, 1)], 1)
                for t in range(2))
        group = self.hq // self.hkv
        q = self.q[a:b].double().cpu().transpose(0, 1)
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        seen = torch.eye(b - a, dtype=torch.bool)
        for r, p in enumerate(self.parents[i]):
            if p >= 0:
                seen[r] |= seen[p]
        seen = torch.cat([torch.ones((b - a, int(self.lengths[i])), dtype=torch.bool), seen], 1)
        s = (q @ k.transpose(1, 2)) * (scale or self.dim ** -0.5)
        p = torch.softmax(s.masked_fill(~seen, -torch.inf), 2)
        out, mass = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
        return out, (2.0 ** -8 + 2.0 ** -12) * mass + 2.0 ** -8 * out.abs() + 1e-30

    def check(self, out, requests=None, scale=None):
        for i in (range(len(self.lengths)) if requests is None else requests):
            a, b = int(self.offset[i]), int(self.offset[i + 1])
            want, bound = self.reference(i, scale)
            err = (out[a:b].double().cpu() - want).abs()
            assert bool((err <= bound).all()), (i, float((err / bound).max()))


@pytest.mark.parametrize("hq,hkv,dim", [(4, 2, 64), (8, 2, 128), (32, 8, 128), (2, 2, 128),
                                        (16, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("lengths,rows", [
    ([0, 1, 31, 32, 33], [1, 2, 3, 16, 33]),
    ([63, 64, 65, 127, 128, 129], [5, 1, 17, 8, 64, 2]),
    ([1000, 0, 640], [31, 64, 130]),
    ([300], [256]),
])
def test_lengths_rows_and_heads(device, hq, hkv, dim, lengths, rows):
    w = Wave(device, lengths, rows, hq, hkv, dim, seed=sum(lengths) + hq)
    w.check(w.run())


@pytest.mark.parametrize("rows", [1, 2, 7, 33, 64])
@pytest.mark.parametrize("target", [0, 3, 700])
def test_split_and_packed_plans(device, rows, target):
    w = Wave(device, [900, 2000, 130], [rows, 1, rows], 8, 2, 128, seed=rows)
    plan = w.plan(target)
    w.check(w.run(plan))


def test_single_token_steps_and_prompt_chunks(device):
    w = Wave(device, [500 + 37 * i for i in range(24)], [1] * 24, 32, 8, 128, seed=5)
    w.check(w.run(), requests=range(0, 24, 5))
    w = Wave(device, [0, 77, 600], [256, 200, 256], 32, 8, 128, seed=6, tree="chain")
    w.check(w.run())


def test_equals_the_bf16_kernel_on_the_unpacked_cache(device):
    # The same values through another kernel: each is within its own bound.
    w = Wave(device, [700, 64, 1500], [16, 40, 9], 32, 8, 128, seed=7)
    k, v = (ops.kv_load_mx4(c, s) for c, s in zip(w.codes, w.scales))
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    full = ops.tree_attention(w.q, k, v, *w.tree, *w.meta, w.plan())
    got = w.run()
    w.check(got)
    assert (got.float() - full.float()).abs().max() <= 2e-2


def test_scale_out_strides_and_arena_views(device):
    w = Wave(device, [200, 65], [9, 20], 8, 2, 128, seed=8)
    arena = [torch.zeros((2, *c.shape[:2], 96), dtype=torch.uint8, device=device)
             for c in w.codes]
    for t, (big, c) in enumerate(zip(arena, w.codes)):
        big[1, :, :, :64] = c
        w.codes[t] = big[1, :, :, :64]                      # token stride 96 bytes
    arena = [torch.zeros((*s.shape[:2], 7), dtype=torch.uint8, device=device) for s in w.scales]
    for t, (big, s) in enumerate(zip(arena, w.scales)):
        big[:, :, 3:] = s
        w.scales[t] = big[:, :, 3:]                         # unaligned, stride 7
    wide = torch.full((29, 8, 132), 5.0, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError):
        w.run(out=wide[:, :, :128])                         # rows of 264 bytes
    wide = torch.full((29, 8, 136), 5.0, dtype=torch.bfloat16, device=device)
    got = w.run(out=wide[:, :, :128], scale=0.05)
    w.check(got, scale=0.05)
    assert (wide[:, :, 128:] == 5).all()


def test_values_that_are_no_numbers_stay_with_the_rows_that_see_them(device):
    # A chain of 0, 1, 2 with branches 3 (under 0) and 4 (under 1), then one far row.
    for bad in (float("nan"), float("inf")):
        w = Wave(device, [70, 40], [40, 3], 8, 2, 128, seed=9)
        w.parents[0] = [-1, 0, 1, 0, 1] + [3] * 35
        w.meta[3][:40] = torch.tensor(w.parents[0], dtype=torch.int32)
        # The others are held to the clean wave's bounds, not to its bits: all rows
        # of a wave move their softmax reference point when one of them has to (an
        # infinite score is such a move), which rescales fp32 sums.
        clean, bound = (torch.cat(t) for t in zip(*(w.reference(i) for i in range(2))))
        w.tree[0][2, 0, 5] = bad                            # K of row 2, head 0
        w.tree[1][4, 1, 77] = bad                           # V of row 4, head 1
        got = w.run()
        assert torch.isnan(got[2, :4]).any() or bad == float("inf")
        assert not torch.isfinite(got[4, 4:, 77]).any()
        same = torch.ones(got.shape, dtype=torch.bool)
        same[2, :4] = False
        same[4, 4:, 77] = False
        err = (got.double().cpu() - clean).abs()
        assert bool((err <= bound)[same].all())
    # A cached row packed from a NaN reaches its request and no other.
    w = Wave(device, [70, 40], [4, 3], 8, 2, 128, seed=9)
    clean = w.run()
    w.scales[1][0, 11, 2] = 255
    got = w.run()
    assert torch.isnan(got[:4, :4, 64:96]).all()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[:4, :4, 64:96] = False
    assert torch.equal(got[keep], clean[keep])


def test_another_waves_plan_marks_status_and_rows(device):
    w = Wave(device, [200, 100], [4, 5], 8, 2, 64, seed=10)
    plan = w.plan()
    status = torch.zeros(1, dtype=torch.int32, device=device)
    w.meta[2][1] = 90                                       # shorter than planned
    got = w.run(plan, status=status)
    assert int(status.item()) == -1
    assert torch.isnan(got[4:]).all() and torch.isfinite(got[:4]).all()


def test_streams_prepared_calls_and_graphs(device):
    w = Wave(device, [1500, 300], [6, 12], 32, 8, 128, seed=11)
    want = w.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = w.run()
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    call = ops.prepare_tree_attention_mx4(
        w.q, w.codes[0], w.scales[0], w.codes[1], w.scales[1], *w.tree, *w.meta, w.plan(), out=out)
    call()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for k in range(3):
        w.q.mul_(-1.0)
        eager = w.run()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), k


def test_refusals(device):
    w = Wave(device, [40], [3], 8, 2, 128, seed=12)
    plan = w.plan()
    with pytest.raises(ValueError):
        w.run(ops.plan_attention(w.offset, w.lengths, 4, 2, 128).to(device))
    codes = w.codes[0]
    w.codes[0] = codes[:, :, :32]
    with pytest.raises(ValueError):
        w.run(plan)
    w.codes[0] = codes.view(torch.int8)
    with pytest.raises(ValueError):
        w.run(plan)
    w.codes[0] = codes
    scales = w.scales[0]
    w.scales[0] = scales[:, :-1]
    with pytest.raises(ValueError):
        w.run(plan)
    w.scales[0] = scales
    w.q = w.q.float()
    with pytest.raises(ValueError):
        w.run(plan)
