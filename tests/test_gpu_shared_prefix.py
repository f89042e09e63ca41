"""Shared-prefix attention against float64 over the joined context.

Pools are filled with NaN before the sequences are written, so a read of any
position that a row may not see shows. Bars are those of the library's verify
attention: fp32 1e-5; bf16 per-entry relative L2 2e-3 and every element within
one bf16 ulp plus 2e-3 of the entry's largest; fp16 1e-3 and 2^-10.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from engine.attention import (SharedPrefix, VerifyPlan, gather_ctx, prefill_attention, shared_prefix_attention,
                              verify_attention)
from engine.kv import PagedKVCache, WritePlan
from engine.rotary import Rotary, rotary_append, rotary_embed

pytestmark = pytest.mark.gpu

F32, BF16, F16, FP8 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _check(out, want, dtype):
    out, want = out.detach().cpu().double(), want.double()
    assert bool(torch.isfinite(out).all())
    for b in range(out.shape[0]):
        err, top = (out[b] - want[b]).abs(), float(want[b].abs().max())
        if dtype == F32:
            assert bool((err <= 1e-5 + 1e-5 * want[b].abs()).all()), (b, float(err.max()))
            continue
        rel, step = (2e-3, 2.0 ** -7) if dtype == BF16 else (1e-3, 2.0 ** -10)
        assert float(err.norm() / want[b].norm()) <= rel, (b, float(err.norm() / want[b].norm()))
        assert bool((err <= step * want[b].abs() + rel * top).all()), (b, float(err.max()), top)


def _pool(cuda, lens, hkv, d, bs, dtype, g, layers=1, scale=1.0):
    """A cache of NaN with sequences of these lengths written, and their keys and values as stored (float64)."""
    cap = sum(-(-n // bs) for n in lens) + 6
    kv = PagedKVCache(layers, hkv, d, cap, bs, cuda, dtype, max_seqs=len(lens), max_blocks_per_seq=1)
    if kv.fp8:
        kv.k_pool.view(torch.uint8).fill_(0x7f)
        kv.v_pool.view(torch.uint8).fill_(0x7f)
    else:
        kv.k_pool.fill_(float("nan"))
        kv.v_pool.fill_(float("nan"))
    kv.allocator.load_free_list(torch.randperm(cap, generator=g).to(torch.int32))
    kv.add_sequence(len(lens) - 1)
    in_dt = BF16 if kv.fp8 else dtype
    for s, n in enumerate(lens):
        if n:
            for layer in range(layers):
                k, v = (torch.randn(1, n, hkv, d, generator=g).mul(scale).to(in_dt).to(cuda) for _ in range(2))
                kv.write_block(layer, [s], [0], k, v)
    ctx = [[gather_ctx(kv, layer, s, n).cpu().double() for s, n in enumerate(lens)] for layer in range(layers)]
    return kv, ctx


def _want(q, ctx, seq_ids, starts, ids, plens, scale=None):
    """softmax(scale q k) v in float64 over each entry's prefix and own keys, one row at a time."""
    q = q.detach().cpu().double()
    B, C, hq, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.empty_like(q)
    for b in range(B):
        k, v = (x.transpose(0, 1) for x in ctx[seq_ids[b]])  # (kv heads, positions, d)
        if ids[b] >= 0 and plens[b]:
            k, v = (torch.cat([x[:plens[b]].transpose(0, 1), y], 1) for x, y in zip(ctx[ids[b]], (k, v)))
        for j in range(C):
            n = (plens[b] if ids[b] >= 0 else 0) + starts[b] + j + 1
            rows = q[b, j].view(k.shape[0], -1, d)
            w = torch.softmax(torch.matmul(rows, k[:, :n].transpose(1, 2)) * scale, -1)
            out[b, j] = torch.matmul(w, v[:, :n]).reshape(hq, d)
    return out


def _q(g, B, C, hq, d, kv, dev):
    return torch.randn(B, C, hq, d, generator=g).to(BF16 if kv.fp8 else kv.dtype).to(dev)


SHAPES = [
    # B, C, hq, hkv, d, bs, prefix lengths, entries' prefixes, own starts
    (1, 1, 4, 2, 64, 16, [1], [0], [0]),                                  # one key of each
    (4, 1, 14, 2, 64, 16, [600], [0, 0, 0, 0], [3, 90, 0, 15]),
    (3, 6, 12, 2, 128, 16, [257], [0, 0, 0], [31, 64, 100]),
    (6, 5, 4, 2, 128, 16, [130, 15, 700], [0, 1, -1, 2, 1, 0], [0, 5, 77, 300, 16, 1]),
    (5, 9, 4, 4, 64, 16, [64], [0, 0, -1, 0, 0], [7, 8, 9, 10, 11]),      # one head a group
    (2, 3, 16, 1, 128, 16, [33], [0, 0], [12, 0]),                        # all heads a group
    (9, 7, 16, 2, 128, 16, [1025], [0] * 9, [5, 0, 40, 3, 2, 600, 1, 17, 16]),
    (40, 2, 8, 2, 64, 16, [80, 81], [0, 1] * 20, list(range(40))),
    (2, 4, 4, 2, 64, 16, [48], [-1, -1], [70, 20]),                       # nobody has a prefix
    (3, 2, 6, 2, 80, 16, [100], [0, 0, 0], [9, 30, 1]),                   # other head dims and blocks
    (3, 2, 4, 2, 64, 4, [50], [0, 0, -1], [9, 30, 1]),
    (2, 3, 2, 1, 256, 24, [90], [0, 0], [25, 0]),
    (2, 3, 2, 1, 9, 16, [20], [0, 0], [25, 0]),
    (2, 40, 8, 2, 64, 16, [90], [0, 0], [25, 0]),                         # long chunks
    (80, 7, 16, 2, 128, 16, [150, 33], [0, 1] * 40, list(range(80))),      # many rows
    (150, 4, 14, 2, 64, 16, [70], [0, 0, -1] * 50, list(range(150))),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16, FP8])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_joined_context(cuda, dtype, shape):
    B, C, hq, hkv, d, bs, plens, which, starts = shape
    g = torch.Generator().manual_seed(B * 100 + C * 10 + d)
    kv, (ctx,) = _pool(cuda, [s + C for s in starts] + plens, hkv, d, bs, dtype, g)
    ids = [B + w if w >= 0 else -1 for w in which]
    lens = [plens[w] if w >= 0 else 0 for w in which]
    prefix = SharedPrefix(kv, ids, lens, C, hq)
    q = _q(g, B, C, hq, d, kv, cuda)
    out = shared_prefix_attention(q, kv, 0, list(range(B)), starts, max(starts) + C, prefix)
    _check(out, _want(q, ctx, list(range(B)), starts, ids, lens), q.dtype)
    kv.seq_lengths  # no forbidden read was flagged
    again = shared_prefix_attention(q, kv, 0, list(range(B)), starts, max(starts) + C + 333, prefix)
    _check(again, _want(q, ctx, list(range(B)), starts, ids, lens), q.dtype)  # a looser bound, other ranges
    assert torch.equal(out, shared_prefix_attention(q, kv, 0, list(range(B)), starts, max(starts) + C, prefix))


@pytest.mark.parametrize("q_dtype,kv_dtype", [(F32, BF16), (F32, FP8), (BF16, F16), (F16, BF16), (BF16, F32), (F16, FP8)])
def test_mixed_types(cuda, q_dtype, kv_dtype):
    g = torch.Generator().manual_seed(2)
    B, C, hq, hkv, d = 3, 4, 8, 2, 64
    starts, plens = [5, 0, 60], [150]
    kv, (ctx,) = _pool(cuda, [s + C for s in starts] + plens, hkv, d, 16, kv_dtype, g)
    prefix = SharedPrefix(kv, [B] * B, plens * B, C, hq)
    q = torch.randn(B, C, hq, d, generator=g).to(q_dtype).to(cuda)
    out = shared_prefix_attention(q, kv, 0, [0, 1, 2], starts, 64, prefix)
    _check(out, _want(q, ctx, [0, 1, 2], starts, [B] * B, plens * B), q_dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16, FP8])
@pytest.mark.parametrize("d,plen", [(64, 4097), (128, 3001)])
def test_long_prefix_many_ranges(cuda, dtype, d, plen):
    g = torch.Generator().manual_seed(plen)
    B, C, hq, hkv = 7, 6, 14, 2
    starts = [0, 500, 33, 16, 1000, 2, 64]
    kv, (ctx,) = _pool(cuda, [s + C for s in starts] + [plen], hkv, d, 16, dtype, g)
    ids, lens = [B] * B, [plen] * B
    ids[3], lens[5] = -1, plen - 17        # one without, one with a shorter part of the same prefix
    lens[3] = 0
    prefix = SharedPrefix(kv, ids, lens, C, hq)
    q = _q(g, B, C, hq, d, kv, cuda)
    out = shared_prefix_attention(q, kv, 0, list(range(B)), starts, max(starts) + C, prefix)
    _check(out, _want(q, ctx, list(range(B)), starts, ids, lens), q.dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale", [None, 0.0, -0.2, 3.0])
def test_scales(cuda, dtype, scale):
    """Any scale; at 3.0 the scores spread over hundreds (one key decides most rows)."""
    g = torch.Generator().manual_seed(31)
    B, C, hq, hkv, d = 3, 3, 6, 2, 64
    starts, plens = [5, 40, 0], [200]
    kv, (ctx,) = _pool(cuda, [s + C for s in starts] + plens, hkv, d, 16, dtype, g)
    prefix = SharedPrefix(kv, [B] * B, plens * B, C, hq)
    q = _q(g, B, C, hq, d, kv, cuda)
    out = shared_prefix_attention(q, kv, 0, [0, 1, 2], starts, 43, prefix, scale=scale)
    want = _want(q, ctx, [0, 1, 2], starts, [B] * B, plens * B, d ** -0.5 if scale is None else scale)
    if scale == 3.0 and dtype == F32:
        # scores up to 3 * 64 * |q k|: the fp32 dot product is off by 2^-24 of some 300 (1.8e-5 each
        # of 64 steps, in random signs about 1.5e-4), which enters the result as a relative error
        err = (out.cpu().double() - want).abs()
        assert bool((err <= 1e-3 * want.abs().max()).all())
    else:
        _check(out, want, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("where", ["late", "early", "own"])
def test_magnitudes_of_values(cuda, dtype, where):
    """Values of very different sizes: a part of the keys holds values 2^20 (bf16, fp32) or
    2^9 (fp16) times the others'."""
    g = torch.Generator().manual_seed(17)
    B, C, hq, hkv, d = 4, 3, 8, 2, 128
    starts, plen = [20, 3, 64, 0], 700
    kv, _ = _pool(cuda, [s + C for s in starts] + [plen], hkv, d, 16, dtype, g)
    big = 2.0 ** 9 if dtype == F16 else 2.0 ** 20
    sid, lo, hi = (B, 600, 700) if where == "late" else (B, 0, 30) if where == "early" else (0, 0, starts[0] + C)
    k, v = gather_ctx(kv, 0, sid, hi)
    kv.write_block(0, [sid], [lo], k[None, lo:].clone(), (v[None, lo:] * big).to(dtype))
    ctx = [gather_ctx(kv, 0, s, n).cpu().double() for s, n in enumerate([s + C for s in starts] + [plen])]
    prefix = SharedPrefix(kv, [B] * B, [plen] * B, C, hq)
    q = _q(g, B, C, hq, d, kv, cuda)
    out = shared_prefix_attention(q, kv, 0, list(range(B)), starts, 67, prefix)
    want = _want(q, ctx, list(range(B)), starts, [B] * B, [plen] * B)
    if dtype == F32:  # relative to the entry's largest output
        for b in range(B):
            assert float((out[b].cpu().double() - want[b]).abs().max()) <= 1e-5 * float(want[b].abs().max())
    else:
        _check(out, want, dtype)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B", [1, 9])
def test_fp8_pages_of_very_different_scales(cuda, d, B):
    """Pages of zeros (keys, values, both) and of values 2^-40 and 2^-110 times the others' among
    a prefix's pages; what they add to the sums is the keys' share alone."""
    g = torch.Generator().manual_seed(37)
    C, hq, hkv, plen = 5, 16, 2, 300
    kv, _ = _pool(cuda, [C + 8] * B + [plen], hkv, d, 16, FP8, g)
    k, v = (torch.randn(1, plen, hkv, d, generator=g) for _ in range(2))
    k[:, 16:32] = 0
    v[:, 48:64] = 0
    k[:, 80:96] = v[:, 80:96] = 0
    v[:, 112:128] *= 2.0 ** -40
    v[:, 208:224] *= 2.0 ** -110
    kv.truncate(B, 0)
    kv.write_block(0, [B], [0], k.to(BF16).to(cuda), v.to(BF16).to(cuda))
    ctx = [gather_ctx(kv, 0, s, n).cpu().double() for s, n in enumerate([C + 8] * B + [plen])]
    prefix = SharedPrefix(kv, [B] * B, [plen] * B, C, hq)
    q = _q(g, B, C, hq, d, kv, cuda)
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [8] * B, C + 8, prefix)
    _check(out, _want(q, ctx, list(range(B)), [8] * B, [B] * B, [plen] * B), q.dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_what_later_positions_hold_reaches_no_earlier_row(cuda, dtype, d, bad):
    g = torch.Generator().manual_seed(23)
    B, C, hq, hkv = 3, 6, 4, 2
    starts, plen = [10, 13, 0], 100
    kv, (ctx,) = _pool(cuda, [s + C for s in starts] + [plen], hkv, d, 16, dtype, g)
    prefix = SharedPrefix(kv, [B] * B, [plen] * B, C, hq)
    q = _q(g, B, C, hq, d, kv, cuda)
    x = torch.full((B, 2, hkv, d), bad, dtype=dtype, device=cuda)
    kv.write_block(0, [0, 1, 2], [s + 4 for s in starts], x, x)
    out = shared_prefix_attention(q, kv, 0, [0, 1, 2], starts, 19, prefix)
    want = _want(q[:, :4], ctx, [0, 1, 2], starts, [B] * B, [plen] * B)
    _check(out[:, :4], want, dtype)
    assert not bool(torch.isfinite(out[:, 4:]).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_non_finite_keys_and_values_that_are_seen(cuda, dtype):
    """A NaN among a prefix's keys reaches every row of its entries, a NaN among one entry's
    values that entry alone, and an infinite value only its dimension."""
    g = torch.Generator().manual_seed(29)
    B, C, hq, hkv, d = 3, 2, 4, 2, 64
    kv, _ = _pool(cuda, [20 + C] * B + [90, 50], hkv, d, 16, dtype, g)
    prefix = SharedPrefix(kv, [B, B + 1, B + 1], [90, 50, 50], C, hq)
    q = _q(g, B, C, hq, d, kv, cuda)
    k, v = (x[None, 30:31].clone() for x in gather_ctx(kv, 0, B, 31))
    k[0, 0, 0, 3] = float("nan")
    kv.write_block(0, [B], [30], k, v)
    k, v = (x[None, 7:8].clone() for x in gather_ctx(kv, 0, 2, 8))
    v[0, 0, 1, 5] = float("inf")
    kv.write_block(0, [2], [7], k, v)
    out = shared_prefix_attention(q, kv, 0, [0, 1, 2], [20] * B, 22, prefix).float().cpu()
    assert bool(torch.isnan(out[0, :, :2]).all()) and bool(torch.isfinite(out[0, :, 2:]).all())
    assert bool(torch.isfinite(out[1]).all())
    bad = ~torch.isfinite(out[2])
    assert bool(bad[:, 2:, 5].all()) and int(bad.sum()) == C * 2


def test_forbidden_reads_are_reported(cuda):
    g = torch.Generator().manual_seed(1)
    C, hq, hkv, d = 2, 4, 2, 64
    for case in ("short prefix", "unwritten", "max_ctx"):
        kv, _ = _pool(cuda, [12, 30, 100], hkv, d, 16, BF16, g)
        prefix = SharedPrefix(kv, [2, 2], [100, 100], C, hq)
        starts, max_ctx = [10, 28], 30
        if case == "short prefix":
            kv.truncate(2, 80)
        elif case == "unwritten":
            starts = [10, 29]
            max_ctx = 31
        else:
            max_ctx = 29
        q = _q(g, 2, C, hq, d, kv, cuda)
        shared_prefix_attention(q, kv, 0, [0, 1], starts, max_ctx, prefix)
        with pytest.raises(IndexError):
            kv.seq_lengths
        kv.seq_lengths


def test_refusals(cuda):
    g = torch.Generator().manual_seed(1)
    kv, _ = _pool(cuda, [12, 30, 100], 2, 64, 16, BF16, g, layers=2)
    for err, args in ((IndexError, ([2, 7], [10, 10], 2, 4)), (IndexError, ([2, 2], [101, 5], 2, 4)),
                      (ValueError, ([2], [1, 1], 2, 4)), (ValueError, ([2, -2], [1, 1], 2, 4)),
                      (ValueError, ([2, 2], [1, -1], 2, 4)), (ValueError, ([2, 2], [1, 1], 0, 4)),
                      (ValueError, ([2, 2], [1, 1], 2, 5))):
        with pytest.raises(err):
            SharedPrefix(kv, *args)
    p = SharedPrefix(kv, [2, -1], [100, 0], 2, 4)
    q = _q(g, 2, 2, 4, 64, kv, cuda)
    go = lambda q=q, kv=kv, layer=0, sids=(0, 1), st=(10, 28), mc=30, **kw: shared_prefix_attention(  # noqa: E731
        q, kv, layer, sids, st, mc, p, **kw)
    other, _ = _pool(cuda, [12, 30, 100], 2, 64, 16, BF16, g)
    for err, kw in ((ValueError, dict(q=q[:1])), (ValueError, dict(q=q[:, :1])), (ValueError, dict(q=q[:, :, :2])),
                    (ValueError, dict(q=q[..., :32])), (ValueError, dict(kv=other)), (IndexError, dict(layer=2)),
                    (ValueError, dict(sids=(0,))), (IndexError, dict(sids=(0, 9))), (ValueError, dict(st=(10,))),
                    (ValueError, dict(mc=1)), (ValueError, dict(out=q)), (ValueError, dict(out=q.float())),
                    (ValueError, dict(q=q.cpu()))):
        with pytest.raises(err):
            go(**kw)
    assert torch.isfinite(go()).all()
    empty = SharedPrefix(kv, [], [], 2, 4)
    assert shared_prefix_attention(q[:0], kv, 0, [], [], 30, empty).shape == (0, 2, 4, 64)


def test_strided_queries_and_own_output(cuda):
    g = torch.Generator().manual_seed(41)
    kv, (ctx,) = _pool(cuda, [12, 30, 100], 2, 64, 16, BF16, g)
    p = SharedPrefix(kv, [2, 2], [100, 100], 2, 4)
    wide = torch.randn(2, 2, 9, 64, generator=g).to(BF16).to(cuda)
    q, out = wide[:, :, 3:7], torch.empty(2, 2, 4, 64, dtype=BF16, device=cuda)
    got = shared_prefix_attention(q, kv, 0, [1, 0], [28, 10], 30, p, out=out)
    assert got is out
    _check(out, _want(q, ctx, [1, 0], [28, 10], [2, 2], [100, 100]), BF16)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_on_any_address(cuda, dtype, d):
    """Queries and outputs one element behind a 16-byte address."""
    g = torch.Generator().manual_seed(43)
    kv, (ctx,) = _pool(cuda, [12, 30, 100], 2, d, 16, dtype, g)
    p = SharedPrefix(kv, [2, 2], [100, 100], 2, 4)
    q = _q(g, 2, 2, 4, d, kv, cuda)
    buf_q, buf_out = (torch.empty(q.numel() + 1, dtype=dtype, device=cuda) for _ in range(2))
    odd = buf_q[1:].view(q.shape)
    odd.copy_(q)
    want = _want(q, ctx, [0, 1], [10, 28], [2, 2], [100, 100])
    _check(shared_prefix_attention(odd, kv, 0, [0, 1], [10, 28], 30, p), want, dtype)
    out = buf_out[1:].view(q.shape)
    _check(shared_prefix_attention(q, kv, 0, [0, 1], [10, 28], 30, p, out=out), want, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16, FP8])
def test_one_sequence_in_several_entries(cuda, dtype):
    """Entries that read the same own sequence, as of different positions, and one whose
    prefix is its own sequence."""
    g = torch.Generator().manual_seed(47)
    C, hq, hkv, d = 3, 8, 2, 64
    kv, (ctx,) = _pool(cuda, [90, 150], hkv, d, 16, dtype, g)
    sids, starts, ids, lens = [0, 0, 0, 1, 1], [5, 87, 40, 0, 147], [1, 1, -1, 1, 0], [150, 70, 0, 33, 90]
    p = SharedPrefix(kv, ids, lens, C, hq)
    q = _q(g, len(sids), C, hq, d, kv, cuda)
    out = shared_prefix_attention(q, kv, 0, sids, starts, 150, p)
    _check(out, _want(q, ctx, sids, starts, ids, lens), q.dtype)


@pytest.mark.parametrize("dtype,q_dtype", [(BF16, BF16), (F32, F32), (BF16, F16)])
def test_blocks_past_32_bit_offsets(cuda, dtype, q_dtype):
    """The last blocks of pools of more than 2^31 elements, written and attended: bit for bit what
    a small pool gives (its blocks 0, 1, ... in the same order)."""
    g = torch.Generator().manual_seed(53)
    B, C, hq, hkv, d, P, cap = 3, 4, 8, 2, 128, 200, 540_000
    rot = Rotary(d, cuda)
    data = [[torch.randn(b, n, h, d, generator=g).to(dtype).to(cuda) for h in (hkv, hkv)]
            for b, n in ((1, P), (B, C))]
    q = torch.randn(B, C, hq, d, generator=g).to(q_dtype).to(cuda)
    outs = []
    for blocks in (40, cap):
        kv = PagedKVCache(1, hkv, d, blocks, 16, cuda, dtype, max_seqs=B + 1)
        kv.allocator.load_free_list(torch.arange(blocks, dtype=torch.int32))  # the last ones first
        kv.add_sequence(B)
        rotary_append(None, *data[0], kv, 0, [B], [0], rot)
        rotary_append(None, *data[1], kv, 0, list(range(B)), [0] * B, rot)
        prefix = SharedPrefix(kv, [B] * B, [P] * B, C, hq)
        outs.append(shared_prefix_attention(q, kv, 0, list(range(B)), [0] * B, C, prefix))
        used = [b for s in range(B + 1) for b in kv.block_tables[s]]
        assert min(used) >= blocks - 20
        outs.append(gather_ctx(kv, 0, B, P))
        del kv, prefix
    assert cap * hkv * 16 * d > 2 ** 31
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    assert bool(torch.isfinite(outs[0]).all())


def test_captured_graphs_and_streams(cuda):
    """Two graphs of one plan, captured at the same time and replayed on two streams with
    new start positions, equal eager calls."""
    g = torch.Generator().manual_seed(51)
    B, C, hq, hkv, d = 4, 3, 8, 2, 128
    kv, _ = _pool(cuda, [200] * B + [333], hkv, d, 16, BF16, g, layers=2)
    p = SharedPrefix(kv, [B, B, -1, B], [333, 333, 0, 300], C, hq)
    sid, st = (torch.arange(B, dtype=torch.int32, device=cuda) for _ in range(2))
    qs = [_q(g, B, C, hq, d, kv, cuda) for _ in range(2)]
    shared_prefix_attention(qs[0], kv, 0, sid, st, 200, p)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for layer in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(shared_prefix_attention(qs[layer], kv, layer, sid, st, 200, p))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(4):
        st.copy_(torch.tensor([7 * step, 150, 30 + step, 100 - step], dtype=torch.int32))
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            assert torch.equal(outs[layer], shared_prefix_attention(qs[layer], kv, layer, sid, st, 200, p))


@pytest.mark.parametrize("dtype", [BF16, F16, F32, FP8])
def test_rounds_behind_a_shared_prompt(cuda, dtype):
    """A shared prompt is embedded, prefilled and written once; verify rounds then rotate and
    append each sequence's chunk behind it and attend over both; after a rewind the next
    round does the same. Every attention equals the one of a cache where each sequence
    holds the prompt itself, and float64."""
    g = torch.Generator().manual_seed(61)
    B, C, hq, hkv, d, layers, P = 4, 5, 8, 2, 64, 2, 150
    in_dt = BF16 if dtype == FP8 else dtype
    kv = PagedKVCache(layers, hkv, d, 200, 16, cuda, dtype, max_seqs=B + 1)
    full = PagedKVCache(layers, hkv, d, 400, 16, cuda, dtype, max_seqs=B)
    kv.add_sequence(B)
    full.add_sequence(B - 1)
    rot = Rotary(d, cuda, base=1e6)
    rnd = lambda *s: torch.randn(*s, generator=g).to(in_dt).to(cuda)  # noqa: E731
    pos = torch.arange(P, dtype=torch.int32, device=cuda)[None]
    for layer in range(layers):
        q, k, v = rnd(1, P, hq, d), rnd(1, P, hkv, d), rnd(1, P, hkv, d)
        qr = rotary_append(q, k, v, kv, layer, [B], [0], rot, alloc=layer == 0)
        q2, kr = rotary_embed(q, k, rot, pos)
        assert torch.equal(qr, q2)
        assert bool(torch.isfinite(prefill_attention(qr, kr, v, [P])).all())
        for s in range(B):
            rotary_append(None, k, v, full, layer, [s], [0], rot)
    prefix = SharedPrefix(kv, [B] * B, [P] * B, C, hq)
    sid = torch.arange(B, dtype=torch.int32, device=cuda)
    own = [0] * B
    for rnd_no in range(3):
        st = torch.tensor(own, dtype=torch.int32, device=cuda)
        at = st[:, None] + torch.arange(C, dtype=torch.int32, device=cuda) + P
        plan, max_ctx = WritePlan(), max(own) + C
        fplan = None
        for layer in range(layers):
            q, k, v = rnd(B, C, hq, d), rnd(B, C, hkv, d), rnd(B, C, hkv, d)
            qr = rotary_append(q, k, v, kv, layer, sid, st, rot, at, alloc=layer == 0, plan=plan)
            out = shared_prefix_attention(qr, kv, layer, sid, st, max_ctx, prefix)
            qf = rotary_append(q, k, v, full, layer, sid, st + P, rot, alloc=layer == 0)
            assert torch.equal(qr, qf)
            if fplan is None:
                fplan = VerifyPlan(full, sid, st + P, C, hq, max_ctx + P)
            whole = verify_attention(qf, full, layer, sid, st + P, max_ctx + P, plan=fplan)
            ctx = [gather_ctx(kv, layer, s, n).cpu().double() for s, n in enumerate([x + C for x in own] + [P])]
            _check(out, _want(qr, ctx, list(range(B)), own, [B] * B, [P] * B), in_dt)
            if dtype != FP8:  # fp8 blocks that hold the prompt's end and the chunk have other scales
                _check(whole, out.cpu(), F32 if dtype == F32 else in_dt)
        own = [n + 1 + (rnd_no + s) % C for s, n in enumerate(own)]
        kv.rewind(list(range(B)), own)
        full.rewind(list(range(B)), [n + P for n in own])
