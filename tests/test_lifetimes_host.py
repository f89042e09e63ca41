"""CPU checks that what a handle holds on the device is kept from reuse until the streams
that were given it are done. Launches and streams are recorded in place of being made."""

from __future__ import annotations

import pytest
import torch

from engine import _hip
from engine import attention as attention_module
from engine import kv as kv_module
from engine import rotary as rotary_module
from engine.attention import SharedPrefix, shared_prefix_attention
from engine.kv import PagedKVCache
from engine.rotary import Rotary, rotary_append, rotary_embed


class Streams:
    now, capturing = 0, False

    def __init__(self) -> None:
        self.recorded = []


@pytest.fixture
def streams(monkeypatch):
    s = Streams()
    for module in (_hip, attention_module, kv_module, rotary_module):
        monkeypatch.setattr(module, "call", lambda name, *args: None)
    monkeypatch.setattr(_hip, "require_gpu", torch.device)
    monkeypatch.setattr(_hip, "stream_of", lambda device: s.now)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: s.now)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: s.capturing)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: s.recorded.append((t.data_ptr(), stream)))
    return s


def _calls():
    """{name: (call, tensors of its handle)}"""
    kv = PagedKVCache(1, 1, 8, 4, 16, "cpu", torch.float32)
    fp8 = PagedKVCache(1, 1, 8, 4, 16, "cpu", torch.float8_e4m3fn)
    for cache in (kv, fp8):
        cache.add_sequence(1)
        cache._lens = [2, 16]
    rot, prefix = Rotary(8, "cpu"), SharedPrefix(kv, [1], [16], 2, 1)
    x = torch.zeros(1, 2, 1, 8)
    ids = torch.zeros(1, dtype=torch.int32)
    return {
        "embed": (lambda: rotary_embed(x, x, rot, torch.zeros(1, 2, dtype=torch.int32)), (rot.inv_freq, rot.axis_of)),
        "append": (lambda: rotary_append(x, x, x, kv, 0, ids, ids, rot), (rot.inv_freq, rot.axis_of)),
        "append fp8": (lambda: rotary_append(x, x, x, fp8, 0, ids, ids, rot), (rot.inv_freq, rot.axis_of)),
        "shared": (lambda: shared_prefix_attention(x, kv, 0, ids, ids, 2, prefix), (prefix._dev,)),
    }


@pytest.mark.parametrize("name", ["embed", "append", "append fp8", "shared"])
def test_a_handle_is_kept_for_other_streams(streams, name):
    go, held = _calls()[name]
    go()
    assert not streams.recorded  # the stream it was made on
    streams.now = 7
    go()
    assert set(streams.recorded) == {(t.data_ptr(), 7) for t in held}
    del streams.recorded[:]
    streams.capturing = True  # the caller keeps what a graph uses
    go()
    assert not streams.recorded


def test_replaced_frequencies_are_kept_for_every_stream(streams):
    """They may have been made on any."""
    rot, x = Rotary(8, "cpu"), torch.zeros(1, 2, 1, 8)
    rot.inv_freq = rot.inv_freq * 2
    rotary_embed(x, x, rot, torch.zeros(1, 2, dtype=torch.int32))
    assert set(streams.recorded) == {(rot.inv_freq.data_ptr(), 0), (rot.axis_of.data_ptr(), 0)}
