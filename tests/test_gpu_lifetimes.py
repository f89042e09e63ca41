"""Handles dropped while another stream still works with them."""

from __future__ import annotations

import pytest
import torch

from engine.attention import SharedPrefix, shared_prefix_attention
from engine.kv import PagedKVCache
from engine.rotary import Rotary, rotary_append, rotary_embed

pytestmark = pytest.mark.gpu


def _busy(stream, x):
    with torch.cuda.stream(stream):
        for _ in range(6):
            x = x @ x * 1e-4
    return x


def test_handles_dropped_while_another_stream_works(cuda):
    """The memory of a plan and of frequencies is not handed out while a queued launch still reads
    it: what is allocated on their own stream after the drop, zeros, does not reach the results."""
    g = torch.Generator().manual_seed(3)
    B, C, hq, hkv, d, P = 3, 2, 4, 2, 64, 100
    kv = PagedKVCache(1, hkv, d, 40, 16, cuda, torch.bfloat16, max_seqs=B + 1)
    kv.add_sequence(B)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().to(cuda)  # noqa: E731
    rotary_append(None, rnd(1, P, hkv, d), rnd(1, P, hkv, d), kv, 0, [B], [0], Rotary(d, cuda))
    rotary_append(None, rnd(B, C, hkv, d), rnd(B, C, hkv, d), kv, 0, list(range(B)), [0] * B, Rotary(d, cuda))
    q, pos = rnd(B, C, hq, d), torch.full((B, C), 5, dtype=torch.int32, device=cuda)
    sid, st = torch.arange(B, dtype=torch.int32, device=cuda), torch.zeros(B, dtype=torch.int32, device=cuda)
    make = lambda: (SharedPrefix(kv, [B] * B, [P] * B, C, hq), Rotary(d, cuda))  # noqa: E731
    run = lambda p, r: (shared_prefix_attention(q, kv, 0, sid, st, C, p), rotary_embed(q, q, r, pos)[0])  # noqa: E731
    want = run(*make())
    big = torch.randn(4096, 4096, device=cuda)
    handles = make()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    _busy(other, big)
    with torch.cuda.stream(other):
        got = run(*handles)
    sizes = [t.numel() * t.element_size() for t in (handles[0]._dev, handles[1].inv_freq, handles[1].axis_of)]
    del handles
    filled = [torch.zeros(n, dtype=torch.uint8, device=cuda) for n in sizes for _ in range(8)]
    torch.cuda.synchronize()
    assert filled and all(torch.equal(a, b) for a, b in zip(want, got))
