"""Where a plan's tensors live and who keeps them, on the CPU: CPU and meta tensors stand
for two devices, and nothing is launched."""
import dataclasses

import pytest
import torch

from specgrove_amd import ops

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
