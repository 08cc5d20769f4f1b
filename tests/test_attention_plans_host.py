"""Where a plan's tensors live and who keeps them, on the CPU: CPU and meta tensors stand
for two devices, and nothing is launched."""
import copy
import dataclasses
import gc
import pickle
import weakref

import numpy as np
import pytest
import torch

from specgrove_amd import _lib, ops

WAVE = ([0, 1, 2], [32768, 300])


@pytest.fixture(autouse=True)
def tensors_count_as_device_tensors(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)  # get_device() of these


def _plan(device="cpu"):
    return ops.plan_attention(*WAVE, 32, 8, 128).to(device)


def test_a_moved_plan_makes_its_4_bit_form_anew():
    plan = _plan()
    first = plan.in_mx4()
    assert first is not plan and plan.in_mx4() is first
    assert first.device.device.type == "cpu"
    plan.to("meta")
    second = plan.in_mx4()
    assert second is not first
    assert second.device.device.type == second.workspace.device.type == "meta"
    # The device tensor set by hand is a move as well.
    plan.device = torch.from_numpy(plan.host)
    assert plan.in_mx4().device.device.type == "cpu"
    # Copied again to the same device: the old form's memory is the old plan's.
    plan.to("cpu")
    assert plan.mx4 is None


def test_a_replaced_plan_shares_no_workspace_with_the_first_one():
    plan = _plan()
    plan.in_mx4()
    other = dataclasses.replace(plan, workspace=torch.empty_like(plan.workspace))
    assert other.in_mx4().workspace.data_ptr() != plan.mx4.workspace.data_ptr()
    third = plan.with_workspace()
    assert third.mx4.workspace.data_ptr() != plan.mx4.workspace.data_ptr()
    assert third.mx4.device is plan.mx4.device
    plan.device = plan.device.to("meta")
    assert plan.with_workspace().mx4 is None


def test_the_4_bit_form_is_of_the_plans_own_wave():
    plan = _plan()
    other = ops.plan_attention(WAVE[0], [32768, 301], 32, 8, 128)
    mixed = dataclasses.replace(plan, host=other.host)
    with pytest.raises(ValueError):
        mixed.in_mx4()


def _meta_tensors(offset, lengths):
    parents = [k - 1 for n in np.diff(offset) for k in range(n)]
    return [torch.from_numpy(np.asarray(a, t)) for a, t in (
        (offset, np.int32), (np.zeros(len(lengths)), np.int64), (lengths, np.int32),
        (parents, np.int32))]


def _call(plan, **kw):
    """A bound call over small CPU tensors (nothing is launched)."""
    rows = WAVE[0][-1]
    q = torch.zeros((rows, 32, 128), dtype=torch.bfloat16)
    tree = torch.zeros((2, rows, 8, 128), dtype=torch.bfloat16)
    codes = torch.zeros((8, 64, 64), dtype=torch.uint8)
    scales = torch.zeros((8, 64, 4), dtype=torch.uint8)
    return ops.prepare_tree_attention_mx4(q, codes, scales, codes, scales, *tree,
                                          *_meta_tensors(*WAVE), plan, **kw)


@pytest.mark.parametrize("make", [ops.plan_attention, ops.plan_attention_mx4])
def test_a_prepared_call_keeps_the_plans_memory(make):
    plan = make(*WAVE, 32, 8, 128).to("cpu")
    call = _call(plan)
    run = plan.in_mx4()
    attn = call._args.attn
    assert attn.plan_dev == run.device.data_ptr() and attn.workspace_dev
    held = {"plan_dev": weakref.ref(run.device), "workspace_dev": weakref.ref(run.workspace),
            "plan_host": weakref.ref(run.host)}
    plan.to("meta")
    plan.host = np.zeros_like(plan.host)
    del run, plan
    gc.collect()
    assert all(ref() is not None for ref in held.values()), held
    assert held["plan_dev"]().data_ptr() == attn.plan_dev
    assert held["workspace_dev"]().data_ptr() == attn.workspace_dev
    assert held["plan_host"]().ctypes.data == attn.plan_host


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "replace", "assigned"])
@pytest.mark.parametrize("make", [ops.plan_attention, ops.plan_attention_mx4])
def test_copies_of_a_used_plan_read_their_own_host_records(make, how):
    plan = make(*WAVE, 32, 8, 128).to("cpu")
    _call(plan)
    if how == "deepcopy":
        other = copy.deepcopy(plan)
    elif how == "pickle":
        other = pickle.loads(pickle.dumps(plan))
    elif how == "replace":
        other = dataclasses.replace(plan, host=plan.host.copy())
    else:
        other = plan
        plan.host = plan.host.copy()
    assert _call(other)._args.attn.plan_host == other.in_mx4().host.ctypes.data


def test_arguments_that_fit_are_looked_at_once(monkeypatch):
    """The check of one argument at a time is for calls that do not fit, an output or a
    status word given or not: it took longer than the call it stands before."""
    def explain(*args):
        raise AssertionError("looked at again")

    plan = ops.plan_attention_mx4(*WAVE, 32, 8, 128).to("cpu")
    out = torch.zeros((2, 32, 128), dtype=torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32)
    with monkeypatch.context() as patched:
        patched.setattr(ops, "_explain_mx4_attention", explain)
        for kw in ({}, dict(out=out), dict(status=status), dict(out=out, status=status)):
            call = _call(plan, **kw)
            assert call._args.attn.status_dev == (status.data_ptr() if "status" in kw else None)
            assert (call.result is out) == ("out" in kw)
    wide = torch.zeros((2, 32, 136), dtype=torch.bfloat16)
    assert _call(plan, out=wide[:, :, :128])._args.attn.out_head_stride == 136
    for bad in (dict(out=out.float()), dict(out=out[:1]), dict(out=out.transpose(0, 1)),
                dict(out=torch.zeros((2, 32, 132), dtype=torch.bfloat16)[:, :, :128]),
                dict(out=wide[:, :, 4:132]), dict(out=out.to("meta")[:, :1]),
                dict(status=status.long()), dict(out=[1]), dict(status=1)):
        with pytest.raises(ValueError):
            _call(plan, **bad)


@pytest.mark.parametrize("scale", [0.0, -0.1, float("inf"), float("nan")])
def test_scales_that_are_no_scales_are_refused(scale):
    """(An empty wave: nothing would be launched.)"""
    plan = ops.plan_attention_mx4([0], [], 8, 2, 64).to("cpu")
    q, tree = torch.zeros((0, 8, 64)), torch.zeros((0, 2, 64))
    q, tree = q.to(torch.bfloat16), tree.to(torch.bfloat16)
    codes = torch.zeros((2, 16, 32), dtype=torch.uint8)
    scales = torch.zeros((2, 16, 2), dtype=torch.uint8)
    meta = _meta_tensors([0], [])
    for value, code in ((scale, -1), (0.125, 0)):
        call = ops.prepare_tree_attention_mx4(q, codes, scales, codes, scales, tree, tree, *meta,
                                              plan, scale=value)
        assert _lib.load().sg_tree_attn_mx4_fwd(call._ref, None) == code
        assert call.result.shape == (0, 8, 64)
