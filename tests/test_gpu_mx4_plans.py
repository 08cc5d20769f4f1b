"""Plans of waves over a 4-bit cache: the wave's own cut, the form that a plan made for
bf16 takes, captures and streams."""
import pytest
import torch

from specgrove_amd import ops
from tests.test_gpu_mx4_attention import Wave

pytestmark = pytest.mark.gpu


def _own_plan(w):
    plan = ops.plan_attention_mx4(w.offset, w.lengths, w.hq, w.hkv, w.dim)
    return plan.to(w.device)


@pytest.mark.parametrize("hq,hkv,dim,lengths,rows", [
    (32, 8, 128, [4000, 300, 9000], [1, 33, 16]),
    (4, 2, 64, [20000], [64]),
    (16, 1, 128, [5000, 0, 2500, 40], [8, 3, 256, 1]),
])
def test_cut_waves(device, hq, hkv, dim, lengths, rows):
    w = Wave(device, lengths, rows, hq, hkv, dim, seed=len(rows) + dim)
    own = _own_plan(w)
    assert own.merges > 0
    got = w.run(own)
    w.check(got)
    # A plan made for bf16 gives the same cut, and the same bits.
    usual = w.plan()
    assert torch.equal(w.run(usual), got)
    assert usual.mx4 is not None and (usual.mx4.host == own.host).all()
    kept = usual.mx4
    assert torch.equal(w.run(usual), got) and usual.mx4 is kept
    other = usual.with_workspace()
    assert other.mx4.workspace.data_ptr() != kept.workspace.data_ptr()
    assert torch.equal(w.run(other), got)


def test_a_capture_needs_the_4_bit_form_first(device):
    w = Wave(device, [3000, 50], [16, 5], 32, 8, 128, seed=4)
    want = w.run(_own_plan(w))
    plan = w.plan()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(ValueError, match="before a capture"):
                w.run(plan)
        w.run(plan)
        out = torch.empty_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            w.run(plan, out=out)
        for seed in range(3):
            w.q.copy_(torch.randn(w.q.shape, generator=torch.Generator().manual_seed(seed)))
            eager = w.run(_own_plan(w))
            out.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(out, eager)
    torch.cuda.current_stream().wait_stream(side)


def test_the_plan_keeps_its_wave(device):
    """What the caller's arrays hold later does not reach the plan."""
    w = Wave(device, [2500, 900], [3, 4], 8, 2, 128, seed=9)
    offset, lengths = w.offset.copy(), w.lengths.copy()
    plan = ops.plan_attention(offset, lengths, w.hq, w.hkv, w.dim).to(device)
    offset[:], lengths[:] = 0, 0
    w.check(w.run(plan))
