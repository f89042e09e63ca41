"""CPU checks of which memory a launch is given after a handle was copied or one of its
tensors replaced: that of the handle's tensors as they are now. The launches are recorded
in place of being made, on tensors in host memory."""

from __future__ import annotations

import copy

import pytest
import torch

from engine import _hip
from engine import kv as kv_module
from engine import rotary as rotary_module
from engine.rotary import Rotary, rotary_embed


@pytest.fixture
def launches(monkeypatch):
    """(name, arguments) of every launch."""
    made = []
    for module in (_hip, kv_module, rotary_module):
        monkeypatch.setattr(module, "call", lambda name, *args: made.append((name, args)))
    monkeypatch.setattr(_hip, "require_gpu", torch.device)
    monkeypatch.setattr(_hip, "stream_of", lambda device: 0)
    return made


def _embed(launches, rot):
    q, k = torch.zeros(1, 2, 3, rot.head_dim), torch.zeros(1, 2, 1, rot.head_dim)
    rotary_embed(q, k, rot, torch.zeros(1, 2, dtype=torch.int32))
    name, args = launches[-1]
    assert name == "spv_rotary"
    return args[8], args[9]  # inv_freq, axis_of


def test_a_copied_rotary_launches_with_its_own_frequencies(launches):
    rot = Rotary(8, "cpu", axis_of=[0, 0, 0, 0])
    assert _embed(launches, rot) == (rot.inv_freq.data_ptr(), rot.axis_of.data_ptr())
    other = copy.deepcopy(rot)
    assert other.inv_freq.data_ptr() != rot.inv_freq.data_ptr()
    assert _embed(launches, other) == (other.inv_freq.data_ptr(), other.axis_of.data_ptr())


def test_replaced_frequencies_are_used(launches):
    rot = Rotary(8, "cpu")
    _embed(launches, rot)
    rot.inv_freq = rot.inv_freq / 8
    assert _embed(launches, rot)[0] == rot.inv_freq.data_ptr()
    rot.factor = 0.5
    _embed(launches, rot)
    assert launches[-1][1][11] == 0.5
