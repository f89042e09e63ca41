"""CPU checks of what rotary_append launches over pools that its one launch does not take."""

from __future__ import annotations

import pytest
import torch

from engine import _hip
from engine import kv as kv_module
from engine import rotary as rotary_module
from engine.kv import PagedKVCache, WritePlan
from engine.rotary import Rotary, rotary_append


@pytest.fixture
def launches(monkeypatch):
    made = []
    for module in (_hip, kv_module, rotary_module):
        monkeypatch.setattr(module, "call", lambda name, *args: made.append(name))
    monkeypatch.setattr(_hip, "require_gpu", torch.device)
    monkeypatch.setattr(_hip, "stream_of", lambda device: 0)
    return made


@pytest.mark.parametrize("alloc", [True, False])
@pytest.mark.parametrize("with_query", [True, False])
@pytest.mark.parametrize("rows,one", [(2 ** 31 - 16, True), (2 ** 31, False)])
def test_pools_of_2_31_rows_are_written_in_two_launches(launches, alloc, with_query, rows, one):
    """As write_block_device takes them: rotated first, then written; smaller pools in one launch."""
    kv, rot = PagedKVCache(1, 1, 8, 4, 16, "cpu", torch.float32), Rotary(8, "cpu")
    kv.allocator.capacity = rows // kv.block_size
    x, ids = torch.zeros(1, 2, 1, 8), torch.zeros(1, dtype=torch.int32)
    del launches[:]
    out = rotary_append(x if with_query else None, x, x, kv, 0, ids, ids, rot, alloc=alloc, plan=WritePlan())
    assert (out is not None) == with_query
    assert launches == (["spv_kv_rotary_append"] if one else ["spv_rotary", "spv_kv_append"])


@pytest.mark.parametrize("shape", [(), (1,), (1, 1)])
def test_one_entry_of_any_shape_over_fp8(launches, shape):
    """Start positions of one entry, however they are shaped, as every other call takes them."""
    kv, rot = PagedKVCache(1, 1, 8, 4, 16, "cpu", torch.float8_e4m3fn), Rotary(8, "cpu")
    x, ids = torch.zeros(1, 2, 1, 8), torch.zeros(shape, dtype=torch.int32)
    del launches[:]
    rotary_append(x, x, x, kv, 0, ids, ids, rot)
    assert launches == ["spv_rotary", "spv_kv_append_fp8"]
