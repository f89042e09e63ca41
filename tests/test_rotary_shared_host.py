"""CPU checks of the rotary and shared-prefix entry points: refusals before
anything touches a GPU, the plan of a shared-prefix batch, and the overlap rules
of rotary outputs."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from engine import _hip
from engine.rotary import Rotary, _apart, _one_place, rotary_embed

I32 = ctypes.c_int32


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_hip.LIB_PATH):
        pytest.fail("libspecverify.so is not built; run __graft_entry__.build()")
    return _hip.lib()


def _plan(lib, ids, lens, C=3, Hq=4, Hkv=2, bs=16, d=128, dtype=_hip.SPV_BF16):
    n = len(ids)
    a, b = (I32 * n)(*ids), (I32 * n)(*lens)
    need = lib.spv_shared_attn_plan(a, b, n, C, Hq, Hkv, d, bs, dtype, None, 0)
    if need < 0:
        return need
    buf = (I32 * need)()
    assert lib.spv_shared_attn_plan(a, b, n, C, Hq, Hkv, d, bs, dtype, buf, need - 1) == _hip.SPV_ERR_WORKSPACE
    assert lib.spv_shared_attn_plan(a, b, n, C, Hq, Hkv, d, bs, dtype, buf, need) == need
    return list(buf)


def _sections(plan):
    """(segments, members, entries) of a plan as lists of records."""
    at = plan[9:12]
    cut = lambda o, n, w: [plan[o + i * w:o + (i + 1) * w] for i in range(n)]  # noqa: E731
    return cut(at[0], plan[7], 8), plan[at[1]:at[2]], cut(at[2], plan[2], 4)


@pytest.mark.parametrize("dtype,d,bs", [(_hip.SPV_BF16, 128, 16), (_hip.SPV_F32, 64, 16), (_hip.SPV_F16, 96, 7)])
@pytest.mark.parametrize("ids,lens", [
    ([7, 7, 7], [100, 100, 100]),
    ([7, -1, 3, 7, 3, 5], [100, 50, 17, 100, 17, 0]),
    ([2, 2, 2], [64, 65, 64]),               # one prefix, two lengths: two groups
    ([-1, -1], [0, 9]),                      # nobody has one
    ([0] * 200 + [1] * 57, [5000] * 200 + [33] * 57),
])
def test_plan_covers_every_row_and_key_once(lib, ids, lens, dtype, d, bs):
    """Items tile (rows of a group) x (keys of its prefix) without gap or overlap, for every kv head."""
    C, Hq, Hkv = 3, 4, 2
    G = C * Hq // Hkv
    plan = _plan(lib, ids, lens, C, Hq, Hkv, bs, d, dtype)
    assert plan[1] == len(plan)
    segs, members, entries = _sections(plan)
    tile = plan[13]
    assert tile == 256 or (dtype == _hip.SPV_F32 and tile in (64, 128))
    want = {}
    for b, (s, n) in enumerate(zip(ids, lens)):
        if s >= 0 and n > 0:
            want.setdefault((s, n), []).append(b)
    seen = 0
    for (sid, n), batch in want.items():
        rows = len(batch) * G
        first, nt, nr = entries[batch[0]][:3]
        assert [entries[b] for b in batch] == [[first, nt, nr, rank] for rank in range(len(batch))]
        assert first == seen and nt == -(-rows // tile)
        for h in range(Hkv):
            for t in range(nt):
                part = [segs[first + (h * nr + s) * nt + t] for s in range(nr)]
                for x in part:
                    assert x[:3] == [sid, n, h] and members[x[3]:x[3] + len(batch)] == batch
                    assert x[4] == tile * t and x[5] == min(tile, rows - tile * t)
                    assert x[6] < x[7] and x[6] % 64 == 0
                assert part[0][6] == 0 and part[-1][7] == n
                assert all(x[7] == y[6] for x, y in zip(part, part[1:]))
        seen += Hkv * nt * nr
    assert seen == len(segs)
    assert all(entries[b][0] == -1 for b, (s, n) in enumerate(zip(ids, lens)) if s < 0 or n == 0)


def test_plan_refusals(lib):
    ARG = _hip.SPV_ERR_ARG
    assert _plan(lib, [-2], [1]) == ARG
    assert _plan(lib, [1], [-1]) == ARG
    assert _plan(lib, [1], [1], Hq=5, Hkv=2) == ARG
    assert _plan(lib, [1], [1], C=0) == ARG
    assert _plan(lib, [1], [1], bs=0) == ARG
    assert _plan(lib, [1], [1], d=0) == ARG and _plan(lib, [1], [1], d=257) == ARG
    assert _plan(lib, [1], [1], dtype=17) == ARG
    assert lib.spv_shared_attn_plan(None, None, 1, 1, 2, 2, 64, 16, _hip.SPV_BF16, None, 0) == ARG
    assert lib.spv_shared_attn_workspace_bytes(None, 64, 16) == 0
    plan = (I32 * 4096)(*_plan(lib, [1, 1], [40, 40]))
    assert lib.spv_shared_attn_workspace_bytes(plan, 64, 2) == 0       # max_ctx below the chunk
    assert lib.spv_shared_attn_workspace_bytes(plan, 64, 48) > 0
    plan[0] = 0
    assert lib.spv_shared_attn_workspace_bytes(plan, 64, 48) == 0      # not a plan


def test_shared_attention_refusals_need_no_gpu(lib):
    ARG, WS = _hip.SPV_ERR_ARG, _hip.SPV_ERR_WORKSPACE
    plan = (I32 * 4096)(*_plan(lib, [1, 1], [40, 40]))
    f = ctypes.c_void_p(4096)  # never dereferenced: every call below is refused

    def go(q_dtype=1, kv_dtype=1, scales=None, maxb=8, B=2, C=3, Hq=4, Hkv=2, d=64, bs=16, layer=0, cap=8, max_ctx=48,
           ws=0, plan_host=plan, out=f):
        return lib.spv_shared_attn(out, f, q_dtype, f, f, kv_dtype, scales, f, maxb, f, f, f, f, B, C, Hq, Hkv, d, bs,
                                   layer, cap, max_ctx, 0.125, plan_host, f, f, ws, None)

    assert go() == WS
    for bad in (dict(q_dtype=3), dict(kv_dtype=9), dict(kv_dtype=3), dict(B=3), dict(C=2), dict(Hq=8), dict(Hkv=4),
                dict(bs=8), dict(d=0), dict(d=257), dict(layer=-1), dict(cap=0), dict(max_ctx=2), dict(maxb=2),
                dict(out=None), dict(plan_host=None)):
        assert go(ws=1 << 40, **bad) == ARG, bad
    assert go(ws=1 << 40, max_ctx=48, maxb=2) == ARG    # the prefix needs three blocks


def test_rotary_refusals_need_no_gpu(lib):
    ARG = _hip.SPV_ERR_ARG
    f = ctypes.c_void_p(4096)
    st = (ctypes.c_int64 * 12)()

    def rot(q=f, k=f, qo=f, ko=f, dt=1, kdt=1, strides=st, pos=f, inv=f, ax=f, axes=1, B=1, C=1, Hq=2, Hkv=1, d=64, R=64,
            inter=0):
        return lib.spv_rotary(qo, q, ko, k, dt, kdt, strides, pos, inv, ax, axes, 1.0, B, C, Hq, Hkv, d, R, inter, None)

    for bad in (dict(q=None, k=None), dict(qo=None), dict(ko=None), dict(dt=3), dict(kdt=2), dict(strides=None),
                dict(pos=None), dict(inv=None), dict(axes=0), dict(axes=3, ax=None), dict(C=0), dict(B=-1), dict(Hq=0),
                dict(d=0), dict(R=65), dict(R=66), dict(R=-2), dict(inter=2), dict(B=1 << 12, C=(1 << 11) + 1)):
        assert rot(**bad) == ARG, bad

    def app(q=f, k=f, qo=f, dt=1, pos=f, axes=1, C=1, Hkv=1, R=64, layer=0, cap=4, bs=16, alloc=0, follow=0, plan=None,
            maxb=4, stack=f, ctr=f):
        return lib.spv_kv_rotary_append(qo, q, k, f, dt, st, f, f, f, maxb, f, f, stack, f, ctr, f, f, pos, f, f, axes,
                                        1.0, 1, C, 2, Hkv, 64, R, 0, layer, cap, bs, alloc, follow, plan, None)

    for bad in (dict(k=None), dict(qo=None), dict(dt=3), dict(pos=None, axes=3), dict(C=0), dict(Hkv=0), dict(R=3),
                dict(layer=-1), dict(cap=0), dict(bs=0), dict(maxb=0), dict(follow=1), dict(follow=1, plan=f, alloc=1),
                dict(alloc=1, stack=None), dict(ctr=None), dict(cap=1 << 27)):
        assert app(**bad) == ARG, bad


def test_rotary_needs_a_gpu():
    with pytest.raises(_hip.HipLibraryError):
        Rotary(64, torch.device("cpu"))


@pytest.mark.parametrize("kw", [dict(rotary_dim=63), dict(rotary_dim=66), dict(rotary_dim=-2), dict(base=0.0),
                                dict(inv_freq=[1.0]), dict(sections=(8, 8)), dict(axis_of=[0] * 31),
                                dict(axis_of=[-1] * 32), dict(sections=(16, 16), axis_of=[0] * 32)])
def test_rotary_arguments(kw):
    with pytest.raises(ValueError):
        Rotary(64, torch.device("cpu"), **kw)


def test_embed_refuses_what_it_cannot_take():
    r = object.__new__(Rotary)
    r.head_dim, r.device, r.axes, r.rotary_dim, r._passed = 64, torch.device("cpu"), 1, 64, {}
    q, k, pos = torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 2, 64), torch.zeros(2, 3, dtype=torch.int32)
    for args in ((q[0], k, r, pos), (q.double(), k.double(), r, pos), (q, k[:1], r, pos), (q, k.half(), r, pos),
                 (q[..., :32], None, r, pos), (q, k, r, pos.float()), (q, k, r, pos[:1]), (q, k, r, pos[None, :1])):
        with pytest.raises(ValueError):
            rotary_embed(*args)
    with pytest.raises(ValueError):
        rotary_embed(q, None, r, pos, key_out=k)
    with pytest.raises(ValueError):
        rotary_embed(q, k, r, pos, query_out=q[:, :, :2])
    with pytest.raises(ValueError):
        rotary_embed(q, k, r, pos, key_dtype=torch.float16)
    both = torch.zeros(2, 3, 5, 64)
    with pytest.raises(ValueError):  # an output that overlaps its input elsewhere
        rotary_embed(both[:, :, :4], None, r, pos, query_out=both[:, :, 1:])
    with pytest.raises(ValueError):  # in place on rows that share memory
        e = torch.zeros(1, 3, 4, 64).expand(2, 3, 4, 64)
        rotary_embed(e, None, r, pos, query_out=e)
    with pytest.raises(ValueError):  # the key read while the query is written over it
        rotary_embed(q, q[:, :, :2], r, pos, query_out=q)


def test_overlap_rules():
    x = torch.zeros(3, 5, 8, 16)
    q, k, v = x.split([4, 2, 2], dim=2)
    assert _apart(q, k) and _apart(k, q) and _apart(q, v) and _apart(v, k)
    assert not _apart(q, x[:, :, 3:5]) and not _apart(q, q) and not _apart(x[:, 1:], x[:, :-1])
    assert _apart(x[0:1], x[1:2]) and not _apart(x[0:2], x[1:3])
    assert _apart(x[:1, :1, :4], x[:1, :1, 4:])
    assert not _apart(x.transpose(0, 1)[:3], x[:, :3])
    assert _one_place(q) and _one_place(x.transpose(0, 1)) and not _one_place(x[:1].expand(3, 5, 8, 16))
    assert not _one_place(torch.as_strided(x, (2, 2, 2, 16), (64, 16, 8, 1)))
