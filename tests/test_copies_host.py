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
from engine.kv import PagedKVCache
from engine.rotary import Rotary, rotary_append, rotary_embed


@pytest.fixture
def launches(monkeypatch):
    """(name, arguments) of every launch."""
    made = []
    for module in (_hip, kv_module, rotary_module):
        monkeypatch.setattr(module, "call", lambda name, *args: made.append((name, args)))
    monkeypatch.setattr(_hip, "require_gpu", torch.device)
    monkeypatch.setattr(_hip, "stream_of", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)  # (asked with replaced frequencies)
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


def _append(launches, kv, rot):
    x = torch.zeros(1, 2, kv.num_kv_heads, kv.head_dim)
    ids = torch.zeros(1, dtype=torch.int32)
    rotary_append(x, x, x, kv, 0, ids, ids, rot)
    name, args = launches[-1]
    assert name == "spv_kv_rotary_append"
    return args[6:15]


def _of(kv):
    a = kv.allocator
    return (kv.k_pool.data_ptr(), kv.v_pool.data_ptr(), kv.tables_dev.data_ptr(), kv._maxb, kv.nblocks_dev.data_ptr(),
            kv.lens_dev.data_ptr(), a.free_stack.data_ptr(), a.free_flag.data_ptr(), a.ctr.data_ptr())


def test_a_copied_cache_is_appended_to_in_its_own_memory(launches):
    kv, rot = PagedKVCache(1, 1, 8, 4, 16, "cpu", torch.float32), Rotary(8, "cpu")
    assert _append(launches, kv, rot) == _of(kv)
    other = copy.deepcopy(kv)
    assert not set(_of(other)) & set(_of(kv)) - {kv._maxb}
    assert _append(launches, other, rot) == _of(other)


@pytest.mark.parametrize("name", ["k_pool", "v_pool", "tables_dev", "nblocks_dev", "lens_dev"])
def test_a_replaced_tensor_of_the_cache_is_used(launches, name):
    kv, rot = PagedKVCache(1, 1, 8, 4, 16, "cpu", torch.float32), Rotary(8, "cpu")
    _append(launches, kv, rot)
    setattr(kv, name, getattr(kv, name).clone())
    assert _append(launches, kv, rot) == _of(kv)
    kv.allocator.free_stack = kv.allocator.free_stack.clone()
    assert _append(launches, kv, rot) == _of(kv)


@pytest.mark.parametrize("bad", [torch.ones(4), torch.ones(3, dtype=torch.float64), torch.ones(8, dtype=torch.float64)[::2],
                                 torch.ones(4, dtype=torch.float64, device="meta"), [1.0] * 4, None])
def test_frequencies_that_a_launch_cannot_read_are_refused(launches, bad):
    """Another type, length, layout or device: the kernels read rotary_dim / 2 float64 in a row."""
    rot = Rotary(8, "cpu")
    with pytest.raises(ValueError):
        rot.inv_freq = bad
    with pytest.raises(ValueError):
        rot.axis_of = bad
    before = _embed(launches, rot)
    assert before == (rot.inv_freq.data_ptr(), rot.axis_of.data_ptr())
    rot.axis_of = torch.zeros(4, dtype=torch.int32)
    assert _embed(launches, rot) == (before[0], rot.axis_of.data_ptr())
