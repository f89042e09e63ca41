"""Rotary embedding and the rotating cache append against float64.

Tolerance of a rotated element y of the pair (a, b): half a step of the output
type, eps/2 |y| (in the subnormals half their spacing), plus the fp32 arithmetic
before it. The angle leaves the fp64 reduction with 2^-25 turns = 1.9e-7 rad,
sin and cos add 2 ulp = 2.4e-7, the factor 6e-8, the two products and their sum
1.8e-7 of (|a| + |b|): 1e-6 factor (|a| + |b|) covers their sum. At positions
near 2^31 the fp64 product has 2^-24 turns of its own on both sides.
"""

from __future__ import annotations

import random

import pytest
import torch

from engine.attention import VerifyPlan, append_verify_attention, verify_attention
from engine.kv import BlockExhaustedError, PagedKVCache, WritePlan
from engine.rotary import Rotary, rotary_append, rotary_embed

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SPACING = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


def _turned(x, pos, rot):
    """x (B, C, H, d) rotated in float64, and |a| + |b| per element."""
    x = x.detach().cpu().double()
    inv, axis = rot.inv_freq.cpu(), rot.axis_of.cpu().long()
    pos = pos.cpu().double()
    if pos.dim() == 2:
        pos = pos.expand(rot.axes, -1, -1)
    R = rot.rotary_dim
    ang = (pos[axis] * inv[:, None, None]).permute(1, 2, 0)[:, :, None, :]
    lo = torch.arange(0, R, 2) if rot.interleaved else torch.arange(R // 2)
    hi = lo + 1 if rot.interleaved else lo + R // 2
    a, b = x[..., lo], x[..., hi]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., lo] = (a * ang.cos() - b * ang.sin()) * rot.factor
    y[..., hi] = (b * ang.cos() + a * ang.sin()) * rot.factor
    size[..., lo] = size[..., hi] = (a.abs() + b.abs()) * abs(rot.factor)
    return y, size


def _close(got, want, size, slack=1e-6):
    err = (got.detach().cpu().double() - want).abs()
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() + SPACING[got.dtype] / 2 + slack * size
    assert bool((err <= bound).all()), float((err - bound).max())


def _rows(g, B, C, hq, hkv, d, dtype, layout, dev):
    x = torch.randn(B, C, hq + 2 * hkv, d, generator=g).to(dtype).to(dev)
    if layout == "packed":
        return x.split([hq, hkv, hkv], dim=2)
    parts = [t.contiguous() for t in x.split([hq, hkv, hkv], dim=2)]
    if layout == "dense":
        return parts
    if layout == "heads_first":  # (B, H, C, d) seen as (B, C, H, d)
        return [t.transpose(1, 2).contiguous().transpose(1, 2) for t in parts]
    if layout == "odd":  # rows that begin at an odd element
        out = []
        for t in parts:
            buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device=dev)
            buf[1:] = t.reshape(-1)
            out.append(buf[1:].view(t.shape))
        return out
    return [t.transpose(2, 3).contiguous().transpose(2, 3) for t in parts]  # "columns": no contiguous row


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,C,hq,hkv,d,R,layout", [
    (1, 1, 14, 2, 64, 64, "packed"),       # one token
    (3, 7, 12, 2, 128, 128, "packed"),
    (2, 65, 4, 4, 64, 32, "dense"),        # part of the row rotated
    (1, 133, 3, 1, 128, 64, "heads_first"),
    (2, 16, 2, 2, 80, 48, "dense"),        # pieces that are no power of two
    (2, 5, 3, 1, 10, 6, "dense"),          # rows of no whole 16-byte pieces
    (2, 9, 2, 1, 64, 64, "odd"),
    (2, 3, 2, 1, 32, 32, "columns"),
    (1, 4, 1, 1, 2, 2, "dense"),
    (1, 3, 2, 1, 7, 0, "dense"),           # nothing rotated
    (1, 5, 2, 1, 256, 256, "packed"),
])
def test_embed(cuda, dtype, interleaved, B, C, hq, hkv, d, R, layout):
    g = torch.Generator().manual_seed(B * 1000 + C * 10 + d)
    rot = Rotary(d, cuda, rotary_dim=R, interleaved=interleaved, factor=1.0 if d != 80 else 0.75)
    q, k, _ = _rows(g, B, C, hq, hkv, d, dtype, layout, cuda)
    pos = torch.randint(0, 5000, (B, C), generator=g).to(torch.int32).to(cuda)
    qo, ko = rotary_embed(q, k, rot, pos)
    for x, y in ((q, qo), (k, ko)):
        want, size = _turned(x, pos, rot)
        _close(y, want, size)
        assert torch.equal(y[..., R:], x[..., R:])
    q_only, none = rotary_embed(q, None, rot, pos)
    assert none is None and torch.equal(q_only, qo)
    if layout == "packed":  # in place, in the projection's own output
        qi, ki = rotary_embed(q, k, rot, pos, query_out=q, key_out=k)
        assert qi is q and ki is k and torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("how", ["sections", "axis_of"])
def test_embed_axes(cuda, dtype, how):
    g = torch.Generator().manual_seed(5)
    B, C, d = 2, 37, 128
    kw = dict(sections=(16, 24, 24)) if how == "sections" else dict(axis_of=[i % 3 for i in range(64)])
    rot = Rotary(d, cuda, base=1e6, **kw)
    assert rot.axes == 3
    q, k, _ = _rows(g, B, C, 6, 2, d, dtype, "packed", cuda)
    pos = torch.randint(0, 900, (3, B, C), generator=g).to(cuda)  # int64 is taken too
    qo, ko = rotary_embed(q, k, rot, pos)
    for x, y in ((q, qo), (k, ko)):
        _close(y, *_turned(x, pos, rot))
    # a text: one position on every axis is the one-axis rotation
    text = torch.arange(C, dtype=torch.int32, device=cuda).expand(B, C)
    one = Rotary(d, cuda, base=1e6)
    assert torch.equal(rotary_embed(q, None, rot, text)[0], rotary_embed(q, None, one, text)[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_embed_far_and_negative_positions(cuda, interleaved):
    g = torch.Generator().manual_seed(8)
    rot = Rotary(64, cuda, interleaved=interleaved)
    pos = torch.tensor([[0, -1, 1, 131071, 1000000, 16777217, -99999, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int64)
    q = torch.randn(1, pos.shape[1], 3, 64, generator=g).to(cuda)
    got, _ = rotary_embed(q, None, rot, pos.to(cuda))
    want, size = _turned(q, pos, rot)
    _close(got[:, :7], want[:, :7], size[:, :7])
    _close(got[:, 7:], want[:, 7:], size[:, 7:], slack=3e-6)  # + 2^-24 turns twice on both sides: 1.5e-6


def test_embed_empty(cuda):
    rot = Rotary(64, cuda)
    for B, C in ((0, 4), (3, 0)):
        q, k = torch.zeros(B, C, 4, 64, device=cuda), torch.zeros(B, C, 2, 64, device=cuda)
        qo, ko = rotary_embed(q, k, rot, torch.zeros(B, C, dtype=torch.int32, device=cuda))
        assert qo.shape == q.shape and ko.shape == k.shape


def test_embed_non_finite_stay_in_their_pair(cuda):
    rot = Rotary(64, cuda)
    q = torch.ones(1, 2, 2, 64, device=cuda)
    q[0, 1, 0, 3] = float("inf")
    q[0, 1, 0, 40] = float("nan")
    out, _ = rotary_embed(q, None, rot, torch.tensor([[3, 4]], device=cuda))
    bad = ~torch.isfinite(out[0, 1, 0])
    assert bad.nonzero().flatten().tolist() == [3, 8, 35, 40]
    assert bool(torch.isfinite(out[0, 0]).all()) and bool(torch.isfinite(out[0, 1, 1]).all())


# ------------------------------------------------------------------ append

def _caches(cuda, layers, hkv, d, cap, bs, dtype, nseq, g, maxb=None):
    """Two equal caches whose pools hold a pattern everywhere and whose free lists are shuffled."""
    out = []
    perm = torch.randperm(cap, generator=g).to(torch.int32)
    k = torch.randn(layers, cap, hkv, bs, d, generator=g)
    v = torch.randn(layers, cap, hkv, d, bs, generator=g)
    for _ in range(2):
        kv = PagedKVCache(layers, hkv, d, cap, bs, cuda, dtype, max_seqs=nseq, max_blocks_per_seq=maxb)
        if not kv.fp8:
            kv.k_pool.copy_(k.to(dtype))
            kv.v_pool.copy_(v.to(dtype))
        kv.allocator.load_free_list(perm)
        kv.add_sequence(nseq - 1)
        out.append(kv)
    return out


def _same_state(a, b):
    assert a.block_tables == b.block_tables
    assert a.seq_lengths == b.seq_lengths
    assert a.allocator.free_list() == b.allocator.free_list()
    assert torch.equal(a.v_pool.view(torch.uint8), b.v_pool.view(torch.uint8))


def _ids(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,C,hq,hkv,d,R,bs,layout,interleaved,own_pos", [
    (5, 1, 14, 2, 64, 64, 16, "packed", False, False),     # a draft step
    (6, 6, 12, 2, 128, 128, 16, "packed", False, True),    # a verify chunk behind a prefix
    (3, 16, 4, 2, 64, 64, 16, "dense", True, True),
    (2, 17, 4, 1, 128, 64, 16, "packed", False, False),
    (1, 333, 4, 2, 64, 64, 16, "packed", True, False),     # a prompt
    (2, 70, 2, 3, 128, 128, 16, "heads_first", False, True),
    (3, 11, 2, 2, 64, 64, 4, "dense", False, False),       # small blocks
    (2, 40, 2, 2, 64, 64, 24, "packed", False, False),     # blocks of no power of two
    (2, 5, 2, 1, 10, 6, 16, "dense", False, True),         # rows of no whole 16-byte pieces
    (2, 9, 2, 2, 64, 64, 16, "odd", False, False),
    (2, 9, 2, 2, 80, 32, 16, "columns", True, False),
])
def test_append(cuda, dtype, B, C, hq, hkv, d, R, bs, layout, interleaved, own_pos):
    """Tables, lengths, free list, values and every key outside the chunk as after
    write_block_device; the chunk's keys and the queries rotated."""
    g = torch.Generator().manual_seed(C * 7 + d + bs)
    r = random.Random(C + d)
    layers, nseq = 3, B + 2
    starts = [r.choice([0, 1, bs - 1, bs, r.randint(0, 90)]) for _ in range(B)]
    sids = r.sample(range(nseq), B)
    cap = sum(-(-(s + C) // bs) for s in starts) + 4
    a, b = _caches(cuda, layers, hkv, d, cap, bs, dtype, nseq, g, maxb=max(-(-(s + C) // bs) for s in starts) + 1)
    for kv in (a, b):
        for s, n in zip(sids, starts):
            if n:
                kv._ensure_blocks_up_to(s, (n - 1) // bs)
    rot = Rotary(d, cuda, rotary_dim=R, interleaved=interleaved)
    sid_t, st_t = _ids(sids, cuda), _ids(starts, cuda)
    pos = (st_t[:, None] + torch.arange(C, device=cuda, dtype=torch.int32)) + (1000 if own_pos else 0)
    plan = WritePlan()
    for layer in range(layers):
        q, k, v = _rows(g, B, C, hq, hkv, d, dtype, layout, cuda)
        before = a.k_pool.clone()
        qo = rotary_append(q, k, v, a, layer, sid_t, st_t, rot, pos if own_pos else None, alloc=layer == 0, plan=plan)
        b.write_block_device(layer, sid_t, st_t, k, v, alloc=layer == 0)
        _same_state(a, b)
        _close(qo, *_turned(q, pos, rot))
        want, size = _turned(k, pos, rot)
        tables = a.block_tables
        at = [(bb, j, tables[s][(n + j) // bs], (n + j) % bs) for bb, (s, n) in enumerate(zip(sids, starts))
              for j in range(C)]
        bb, jj, blk, off = (torch.tensor(x) for x in zip(*at))
        got = a.k_pool[layer].cpu()[blk, :, off]
        _close(got, want[bb, jj], size[bb, jj])
        rest = a.k_pool.clone()
        rest[layer, blk.to(cuda), :, off.to(cuda)] = before[layer, blk.to(cuda), :, off.to(cuda)]
        assert torch.equal(rest, before)
        b.k_pool.copy_(a.k_pool)


def test_append_follows_the_rules_of_an_exhausted_pool(cuda):
    """A pool that runs out mid-batch: the entry that finds it empty and those after
    it write only what the plain append writes, in the first layer and by its plan."""
    g = torch.Generator().manual_seed(3)
    B, C, hkv, d, bs = 4, 40, 2, 64, 16
    a, b = _caches(cuda, 2, hkv, d, 7, bs, BF16, B, g)
    rot = Rotary(d, cuda)
    sid_t, st_t = _ids([2, 0, 3, 1], cuda), _ids([0, 0, 0, 0], cuda)
    k, v = (torch.randn(B, C, hkv, d, generator=g).to(BF16).to(cuda) for _ in range(2))
    pos = torch.arange(C, dtype=torch.int32, device=cuda).expand(B, C)
    _, kr = rotary_embed(k, k, rot, pos)
    pa, pb = WritePlan(), WritePlan()
    for layer in range(2):
        rotary_append(None, k, v, a, layer, sid_t, st_t, rot, alloc=layer == 0, plan=pa)
        b.write_block_device(layer, sid_t, st_t, kr, v, alloc=layer == 0, plan=pb)
        if layer == 0:
            assert torch.equal(pa.rows[:B * C], pb.rows[:B * C])
    for kv in (a, b):
        with pytest.raises(BlockExhaustedError):
            kv.seq_lengths
    _same_state(a, b)
    assert torch.equal(a.k_pool, b.k_pool)


def test_append_plan_serves_the_other_planned_calls(cuda):
    """The rows a rotating append recorded drive write_block_device and the
    append-and-attend launch of later layers, and the other way round."""
    g = torch.Generator().manual_seed(4)
    B, C, hq, hkv, d, bs = 3, 6, 4, 2, 64, 16
    a, b = _caches(cuda, 3, hkv, d, 40, bs, BF16, B, g)
    rot = Rotary(d, cuda)
    sid_t, st_t = _ids([0, 1, 2], cuda), _ids([0, 0, 0], cuda)
    pos = torch.arange(C, dtype=torch.int32, device=cuda).expand(B, C)
    data = [_rows(g, B, C, hq, hkv, d, BF16, "dense", cuda) for _ in range(3)]
    plan = WritePlan()
    rotary_append(data[0][0], data[0][1], data[0][2], a, 0, sid_t, st_t, rot, plan=plan)
    a.write_block_device(1, sid_t, st_t, data[1][1], data[1][2], alloc=False, plan=plan)
    vp = VerifyPlan(a, sid_t, st_t, C, hq, C)
    got = append_verify_attention(data[2][0], data[2][1], data[2][2], a, 2, sid_t, st_t, C, vp, plan)
    kr = rotary_embed(data[0][0], data[0][1], rot, pos)[1]
    for layer, k in enumerate((kr, data[1][1], data[2][1])):
        b.write_block_device(layer, sid_t, st_t, k, data[layer][2], alloc=layer == 0)
    _same_state(a, b)
    assert torch.equal(a.k_pool, b.k_pool)
    assert torch.equal(got, verify_attention(data[2][0], b, 2, sid_t, st_t, C))
    other = WritePlan()
    b.write_block_device(0, sid_t, st_t, data[0][1], data[0][2], alloc=True, plan=other)
    rotary_append(None, data[1][1], data[1][2], b, 1, sid_t, st_t, rot, pos, alloc=False, plan=other)
    rotary_append(None, data[1][1], data[1][2], a, 1, sid_t, st_t, rot, pos, alloc=False)
    assert torch.equal(a.k_pool[1], b.k_pool[1])
    a.truncate(0, 2)
    with pytest.raises(ValueError):  # the plan's rows may belong to another sequence by now
        rotary_append(None, data[1][1], data[1][2], a, 1, sid_t, st_t, rot, alloc=False, plan=plan)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_append_fp8(cuda, dtype):
    """Codes and scales of an fp8 pool as after quantising the unrounded rotated keys."""
    g = torch.Generator().manual_seed(6)
    B, C, hq, hkv, d, bs = 3, 21, 4, 2, 64, 16
    a, b = _caches(cuda, 2, hkv, d, 30, bs, torch.float8_e4m3fn, B, g)
    rot = Rotary(d, cuda)
    sid_t = _ids([1, 0, 2], cuda)
    for start in (0, C - 4):
        st_t = _ids([start] * B, cuda)
        pos = st_t[:, None] + torch.arange(C, dtype=torch.int32, device=cuda)
        for layer in range(2):
            q, k, v = _rows(g, B, C, hq, hkv, d, dtype, "packed", cuda)
            qo = rotary_append(q, k, v, a, layer, sid_t, st_t, rot, alloc=layer == 0)
            qw, k32 = rotary_embed(q, k, rot, pos, key_dtype=F32)
            b.write_block_device(layer, sid_t, st_t, k32, v.float(), alloc=layer == 0)
            assert torch.equal(qo, qw)
            _close(k32, *_turned(k, pos, rot))
    _same_state(a, b)
    assert torch.equal(a.k_pool.view(torch.uint8), b.k_pool.view(torch.uint8))
    assert torch.equal(a.scales, b.scales)


def test_append_lists_and_refusals(cuda):
    g = torch.Generator().manual_seed(9)
    B, C, hkv, d = 2, 4, 2, 64
    a, b = _caches(cuda, 2, hkv, d, 20, 16, BF16, 3, g)
    rot = Rotary(d, cuda)
    q, k, v = _rows(g, B, C, 4, hkv, d, BF16, "dense", cuda)
    rotary_append(q, k, v, a, 0, [2, 0], [0, 0], rot)
    rotary_append(q, k, v, b, 0, _ids([2, 0], cuda), _ids([0, 0], cuda), rot)
    _same_state(a, b)
    assert torch.equal(a.k_pool, b.k_pool)
    for err, args, kw in (
            (ValueError, (q, k, v, a, 0, [1, 1], [0, 0], rot), {}),
            (ValueError, (q, k, v, a, 0, [1, 0], [0, -1], rot), {}),
            (IndexError, (q, k, v, a, 0, [1, 7], [0, 0], rot), {}),
            (IndexError, (q, k, v, a, 2, [1, 0], [0, 0], rot), {}),
            (ValueError, (q, k, v, a, 0, [1], [0], rot), {}),
            (ValueError, (q.float(), k, v, a, 0, [1, 0], [0, 0], rot), {}),
            (ValueError, (q, k.half(), v.half(), a, 0, [1, 0], [0, 0], rot), {}),
            (ValueError, (q, k[:, :2], v, a, 0, [1, 0], [0, 0], rot), {}),
            (ValueError, (q[:1], k, v, a, 0, [1, 0], [0, 0], rot), {}),
            (ValueError, (q, k, v, a, 0, [1, 0], [0, 0], Rotary(32, cuda)), {}),
            (ValueError, (q, k, v, a, 0, [1, 0], [0, 0], Rotary(d, cuda, sections=(16, 16))), {}),
            (ValueError, (None, k, v, a, 0, [1, 0], [0, 0], rot), dict(query_out=q)),
            (ValueError, (q, k, v, a, 0, [1, 0], [0, 0], rot), dict(positions=torch.zeros(B, C, device=cuda))),
            (ValueError, (q, k, v.cpu(), a, 0, [1, 0], [0, 0], rot), {})):
        with pytest.raises(err):
            rotary_append(*args, **kw)
    _same_state(a, b)
    assert torch.equal(a.k_pool, b.k_pool)
    wide, _ = _caches(cuda, 1, hkv, d, 40, 16, BF16, 1, g, maxb=2)
    kk = torch.randn(1, 100, hkv, d, generator=g).to(BF16).to(cuda)
    rotary_append(None, kk, kk, wide, 0, [0], [0], rot)  # lists: the tables widen
    assert wide.seq_lengths == [100]


def test_append_captured(cuda):
    """A captured round (allocating first layer, a later one by its plan) replayed at
    new positions equals the eager calls."""
    g = torch.Generator().manual_seed(12)
    B, C, hq, hkv, d = 3, 5, 4, 2, 64
    a, b = _caches(cuda, 2, hkv, d, 60, 16, BF16, B, g)
    rot = Rotary(d, cuda)
    sid_t, st_t = _ids([0, 1, 2], cuda), _ids([0, 0, 0], cuda)
    data = [_rows(g, B, C, hq, hkv, d, BF16, "packed", cuda) for _ in range(2)]
    plan, outs = WritePlan(), [torch.empty(B, C, hq, d, dtype=BF16, device=cuda) for _ in range(2)]

    def rounds(kv, plan, outs):
        for layer in range(2):
            rotary_append(*data[layer], kv, layer, sid_t, st_t, rot, alloc=layer == 0, plan=plan, query_out=outs[layer])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rounds(a, plan, outs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rounds(a, plan, outs)
    eager, eplan = [torch.empty_like(o) for o in outs], WritePlan()
    rounds(b, eplan, eager)
    for step in range(4):
        st_t.add_(C)
        graph.replay()
        torch.cuda.synchronize()
        a._stale = a.allocator._stale = True  # the host mirrors know of no replay
        rounds(b, eplan, eager)
        for x, y in zip(outs, eager):
            assert torch.equal(x, y)
        _same_state(a, b)
        assert torch.equal(a.k_pool, b.k_pool)
