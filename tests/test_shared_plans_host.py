"""CPU check of the tests' own plans: cut as the library cuts, they are the library's, word for word."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch  # noqa: F401

from engine import _hip
from shared_plans import UNIT, cut_plan, segments

I32 = ctypes.c_int32


@pytest.mark.parametrize("seed", range(40))
def test_cut_as_the_library_cuts(seed):
    r = random.Random(seed)
    B, hkv = r.choice([1, 5, 60, 200]), r.choice([1, 2, 4])
    C, hq, d = r.randint(1, 9), hkv * r.randint(1, 8), r.choice([64, 128, 80])
    plens = [r.randint(0, 9000) for _ in range(r.choice([1, 1, 3]))]
    which = [r.randrange(-1, len(plens)) for _ in range(B)]
    ids, lens = [w if w < 0 else 100 + w for w in which], [plens[w] if w >= 0 else 0 for w in which]
    dtype, bs = r.choice([_hip.SPV_F32, _hip.SPV_BF16, _hip.SPV_F16, _hip.SPV_FP8E4M3]), r.choice([16, 16, 7])
    args = ((I32 * B)(*ids), (I32 * B)(*lens), B, C, hq, hkv, d, bs, dtype)
    n = _hip.lib().spv_shared_attn_plan(*args, None, 0)
    plan = (I32 * n)()
    assert _hip.lib().spv_shared_attn_plan(*args, plan, n) == n
    plan = list(plan)
    pers = {}  # units of a prefix -> units of its ranges
    for s in segments(plan):
        if s[6] == 0:
            pers[-(-s[1] // UNIT)] = -(-s[7] // UNIT)
    assert cut_plan(plan, ids, lens, lambda units: pers[units], plan[13]) == plan
