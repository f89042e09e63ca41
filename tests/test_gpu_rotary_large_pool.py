"""rotary_append into a pool of more than 2^31 token rows."""

from __future__ import annotations

import pytest
import torch

from engine.kv import PagedKVCache, WritePlan
from engine.rotary import Rotary, rotary_append

pytestmark = pytest.mark.gpu


def test_rows_past_31_bits(cuda):
    """The last blocks of a pool of 2^31 + 2^24 rows, in two layers' calls of a round: bit for bit what a
    small pool holds."""
    g = torch.Generator().manual_seed(5)
    B, C, d = 2, 21, 2
    rot = Rotary(d, cuda)
    x = [[torch.randn(B, C, 1, d, generator=g).bfloat16().to(cuda) for _ in range(3)] for _ in range(2)]
    got = []
    for blocks in (16, (1 << 27) + (1 << 20)):
        kv = PagedKVCache(1, 1, d, blocks, 16, cuda, torch.bfloat16, max_seqs=B, max_blocks_per_seq=4)
        kv.allocator.load_free_list(torch.arange(blocks, dtype=torch.int32))  # the last ones first
        kv.add_sequence(B - 1)
        plan = WritePlan()
        q = [rotary_append(*parts, kv, 0, [0, 1], [0, 0], rot, alloc=n == 0, plan=plan) for n, parts in enumerate(x)]
        ids = torch.tensor([b for t in kv.block_tables for b in t], device=cuda)
        assert int(ids.min()) >= blocks - 8 and kv.seq_lengths == [C, C]
        got.append([*q, kv.k_pool[0][ids].clone(), kv.v_pool[0][ids].clone()])
        del kv
    for a, b in zip(*got):
        assert torch.equal(a, b)
