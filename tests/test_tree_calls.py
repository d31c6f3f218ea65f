"""Refusals of the draft-tree calls that need no GPU to be seen."""

from __future__ import annotations

import pytest
import torch

from asrback_b200 import _native, attention, step
from tests.test_tree import P, PLAN, _status


def test_a_step_with_weights_on_another_device_is_refused(monkeypatch):
    """No second GPU is needed: the devices' types differ here."""
    monkeypatch.setattr(attention, "_dtype_code", lambda *tensors: _native.BF16)
    hidden = torch.zeros((3, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="hidden states' device"):
        step.greedy_choose(hidden, torch.zeros((100, 64), dtype=torch.bfloat16, device="meta"))


IN_CACHE = {k: v for k, v in PLAN.items() if k not in ("ancestors", "depths", "live_counts", "status",
                                                       "stream")}
IN_CACHE |= dict(lengths=P, capacity=40, ancestors=P, depths=P, live_counts=P, status=None, stream=None)


@pytest.mark.parametrize("change", [
    dict(batch=0), dict(nodes=65), dict(parents=None), dict(ancestors=None), dict(depths=None),
    dict(live_counts=None), dict(parents_stride=4), dict(capacity=0), dict(capacity=-1)],
    ids=lambda change: "-".join(f"{k}={v}" for k, v in change.items()))
def test_bad_plans_in_a_cache_are_refused(change):
    assert _status("asrback_draft_tree_in_cache", IN_CACHE, **change) == _native.ERR_ARGUMENT
