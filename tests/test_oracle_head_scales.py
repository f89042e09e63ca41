"""The oracle's 8-bit pool with head scales, by the bounds that its rule implies."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.kv_fp8 import Fp8PagedKVCache, HeadScaledPagedKVCache, e4m3_decode


def _pair(H, cap=8, bs=4, d=6, layers=2):
    one, many = Fp8PagedKVCache(layers, H, d, cap, bs), HeadScaledPagedKVCache(layers, H, d, cap, bs)
    for kv in (one, many):
        kv.add_sequence(0)
        kv.add_sequence(1)
    return one, many


def test_one_head_is_the_one_scale_pool():
    one, many = _pair(1)
    g = torch.Generator().manual_seed(0)
    for start, n, mag in ((0, 3, 1.0), (3, 4, 5.0), (5, 2, 0.1), (6, 9, 40.0)):
        k, v = (torch.randn(1, n, 1, 6, generator=g) * mag for _ in range(2))
        for kv in (one, many):
            kv.write_block(1, [0], [start], k, v)
    assert torch.equal(one.k, many.k) and torch.equal(one.v, many.v)
    assert np.array_equal(one.scales, many.scales[:, 0])


def test_heads_do_not_touch_each_other():
    """Every head of the pool is what a pool of that head alone holds."""
    H, d, bs = 3, 6, 4
    many = HeadScaledPagedKVCache(1, H, d, 8, bs)
    alone = [HeadScaledPagedKVCache(1, 1, d, 8, bs) for _ in range(H)]
    for kv in (many, *alone):
        kv.add_sequence(0)
    g = torch.Generator().manual_seed(1)
    for start, n in ((0, 3), (2, 5), (7, 6)):
        k, v = (torch.randn(1, n, H, d, generator=g) * torch.tensor([1e-3, 1.0, 1e4])[:, None] for _ in range(2))
        many.write_block(0, [0], [start], k, v)
        for h in range(H):
            alone[h].write_block(0, [0], [start], k[:, :, h:h + 1], v[:, :, h:h + 1])
    for h in range(H):
        assert torch.equal(many.k[:, :, :, h], alone[h].k[:, :, :, 0])
        assert np.array_equal(many.scales[:, h], alone[h].scales[:, 0])


def test_small_heads_keep_their_precision():
    """Half an e4m3 step of each head's own largest value bounds what is lost, whatever the other heads hold."""
    H, d, bs = 2, 8, 16
    kv = HeadScaledPagedKVCache(1, H, d, 4, bs)
    kv.add_sequence(0)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, bs, H, d, generator=g) * torch.tensor([1.0, 1e-6])[:, None]
    kv.write_block(0, [0], [0], x, x)
    got = kv.dequantized().k[0, kv.block_tables[0][0]]
    for h in range(H):
        scale = float(kv.scales[0, h, kv.block_tables[0][0], 0])
        assert scale == float(np.float32(x[0, :, h].abs().max().item()) / np.float32(448.0))
        err = (got[:, h] - x[0, :, h]).abs()
        bound = torch.maximum(2.0 ** -4 * x[0, :, h].abs(), torch.tensor(2.0 ** -10 * scale)) * (1 + 1e-6)
        assert bool((err <= bound).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_is_not_finite(bad):
    kv = HeadScaledPagedKVCache(1, 2, 4, 4, 4)
    kv.add_sequence(0)
    x = torch.ones(1, 2, 2, 4)
    x[0, 1, 0, 2] = bad
    kv.write_block(0, [0], [0], x, x)
    blk = kv.block_tables[0][0]
    assert float(kv.scales[0, 0, blk, 0]) == float(np.float32(1.0) / np.float32(448.0))
    kv.write_block(0, [0], [2], torch.full((1, 1, 2, 4), 9.0), x[:, :1])  # a grown scale
    deq = kv.dequantized().k[0, blk].numpy()
    assert np.isnan(deq[1, 0, 2]) and np.isnan(deq).sum() == 1
    assert np.isnan(e4m3_decode(kv.k.numpy())).sum() == 1


def test_allocation_clears_the_scales():
    _, kv = _pair(2)
    x = torch.full((1, 4, 2, 6), 3.0)
    kv.write_block(0, [0], [0], x, x)
    kv.write_block(1, [0], [0], x * 2, x)
    blk = kv.block_tables[0][0]
    assert (kv.scales[:, :, blk] > 0).all()
    kv.clear(0)
    kv.write_block(0, [1], [0], x[:, :1], x[:, :1])
    assert kv.block_tables[1][0] == blk and (kv.scales[1, :, blk] == 0).all() and (kv.scales[0, :, blk] > 0).all()
