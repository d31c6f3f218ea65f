"""Refusals of the draft-tree calls that need no GPU to be seen."""

from __future__ import annotations

import pytest
import torch

from asrback_b200 import _native, attention, step


def test_a_step_with_weights_on_another_device_is_refused(monkeypatch):
    """No second GPU is needed: the devices' types differ here."""
    monkeypatch.setattr(attention, "_dtype_code", lambda *tensors: _native.BF16)
    hidden = torch.zeros((3, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="hidden states' device"):
        step.greedy_choose(hidden, torch.zeros((100, 64), dtype=torch.bfloat16, device="meta"))
