"""The turn itself: rows whose pairs are (1, 0) come back as (cos, sin) of position times frequency."""

from __future__ import annotations

import pytest
import torch

from engine.kv import PagedKVCache
from engine.rotary import Rotary, rotary_append, rotary_embed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [128, 126])  # whole 16-byte pieces, and not
@pytest.mark.parametrize("far", [4096, 1000000])
def test_cos_and_sin_to_their_own_rounding(cuda, d, far):
    """fp32 sin and cos, off by up to 2 steps of 2^-24 (theirs below 1) and by half a step, evenly spread,
    as a rule: 2^-24 / sqrt(12) = 1.7e-8 rms, a quarter more for those that are off by more. The angle's
    rounding to fp32, in steps of 2^-25 turns at most, would by itself add 2 pi 2^-25 / sqrt(12) / sqrt(2)
    = 3.8e-8 where it is largest. (fp64 angles of 10^6 / (2 pi) turns: 2^-36.)"""
    rot = Rotary(d, cuda, base=1e6)
    g = torch.Generator().manual_seed(7)
    pos = torch.randint(0, far, (2, 3001), generator=g).to(torch.int32).to(cuda)
    x = torch.zeros(2, 3001, 1, d, device=cuda)
    x[..., :d // 2] = 1
    q, k = rotary_embed(x, x, rot, pos)
    angle = pos.double()[..., None, None] * rot.inv_freq
    want = torch.cat([angle.cos(), angle.sin()], -1)
    for y in (q, k):
        err = (y.double() - want).abs()
        assert float(err.max()) <= 2.0 ** -23 and float(err.square().mean().sqrt()) <= 1.25 * 2.0 ** -24 / 12 ** 0.5
    kv = PagedKVCache(1, 1, d, 400, 16, cuda, torch.float32, max_seqs=2, max_blocks_per_seq=200)
    kv.add_sequence(1)
    assert torch.equal(rotary_append(x, x, x, kv, 0, [0, 1], [0, 0], rot, pos), q)
