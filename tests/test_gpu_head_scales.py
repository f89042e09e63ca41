"""The 8-bit cache with a scale for each block and head, on the GPU.

Writes are compared with the oracle code by code (``HeadScaledPagedKVCache``),
read-backs with its dequantised values, attention with float64 over them.

Attention's tolerance, per element of row r: half a step of the output type of
|o|, plus eps_p sum_i p_i |v_i|. A weight p_i is off by its score, 2 (d + 4) 2^-24
times the largest sum_e |q_e k_e| scale of the row (d products and sums, the
scales' products, the maximum taken off; 2 for the row's sum, which is off as
much), by exp2 and the running rescales (2^-20), and by its own rounding before
the product with v: for fp16 and fp32 queries to 16 bits or more (2^-17 with the
sum's), for bf16 queries to fp16, whose step is 2^-10 of the power of two below the
weight: at most 2^-11 of the weight, an eighth of what bf16 outputs are rounded by.
"""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

from engine.attention import (SharedPrefix, VerifyPlan, append_verify_attention, gather_ctx, paged_attention_decode,
                              paged_attention_extend, verify_attention)
from engine.kv import BlockExhaustedError, PagedKVCache, WritePlan
from engine.rotary import HeadNorm, Rotary, rotary_append, rotary_embed
from oracle.kv_fp8 import HeadScaledPagedKVCache, e4m3_decode, e4m3_encode
from oracle.kv_pool import BlockExhaustedError as RefExhausted

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _pair(cuda, layers, H, d, cap, bs, n_seq, **kw):
    gpu = PagedKVCache(layers, H, d, cap, bs, cuda, FP8, head_scales=True, **kw)
    cpu = HeadScaledPagedKVCache(layers, H, d, cap, bs)
    for s in range(n_seq):
        gpu.add_sequence(s)
        cpu.add_sequence(s)
    return gpu, cpu


def _canonical(codes):
    """Codes with every NaN as 0x7f."""
    return torch.where((codes & 0x7F) == 0x7F, torch.full_like(codes, 0x7F), codes)


def _same(gpu, cpu):
    assert gpu.block_tables == cpu.block_tables
    assert gpu.seq_lengths == cpu.seq_lengths
    assert gpu.allocator.free_list() == cpu.allocator.free_list
    k = gpu.k_pool.view(torch.uint8).permute(0, 1, 3, 2, 4).cpu()
    v = gpu.v_pool.view(torch.uint8).permute(0, 1, 4, 2, 3).cpu()
    assert np.array_equal(gpu.scales.cpu().numpy().view(np.uint32), cpu.scales.view(np.uint32))
    assert torch.equal(_canonical(k), _canonical(cpu.k)) and torch.equal(_canonical(v), _canonical(cpu.v))


def _random(g, shape, dtype, spread=True):
    x = torch.randn(shape, generator=g)
    if spread:  # heads of very different sizes
        x = x * torch.pow(10.0, torch.randint(-4, 4, (shape[2],), generator=g).float())[:, None]
    return x.to(dtype)


# ---------------------------------------------------------------------------
# writing
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,H,d,bs", [
    (F32, 2, 16, 4), (BF16, 3, 64, 16), (F16, 1, 128, 16), (F32, 2, 128, 32), (BF16, 2, 64, 64), (F32, 4, 10, 7),
    (BF16, 1, 1, 1), (F16, 2, 80, 48), (F32, 2, 256, 16),
])
def test_trace_matches_oracle(cuda, dtype, H, d, bs):
    rng, g = random.Random(d * bs), torch.Generator().manual_seed(d + bs)
    gpu, cpu = _pair(cuda, 2, H, d, 20, bs, 4)
    for _ in range(40):
        op = rng.random()
        if op < 0.6:
            sids = rng.sample(range(4), rng.randint(1, 3))
            chunk = rng.randint(1, 2 * bs + 3)
            starts = [max(0, cpu.seq_lengths[s] - rng.randint(0, 3)) for s in sids]
            layer = rng.randrange(2)
            kn, vn = (_random(g, (len(sids), chunk, H, d), F32) * 10.0 ** rng.uniform(-2, 0) for _ in range(2))
            kn, vn = kn.to(dtype), vn.to(dtype)
            raised = []
            for kv, k, v, e in ((gpu, kn.to(cuda), vn.to(cuda), BlockExhaustedError), (cpu, kn, vn, RefExhausted)):
                try:
                    kv.write_block(layer, sids, starts, k, v)
                    raised.append(False)
                except e:
                    raised.append(True)
            assert raised[0] == raised[1]
        else:
            s = rng.randrange(4)
            n = rng.randint(0, cpu.seq_lengths[s])
            for kv in (gpu, cpu):
                kv.truncate(s, n) if op < 0.85 else kv.clear(s)
        _same(gpu, cpu)


def test_codes_are_the_nearest(cuda):
    """A head whose largest element is 448 has scale 1: its codes are the e4m3 encodings of the
    inputs (every code, the ties between neighbours, subnormals, the saturation's edge)."""
    vals = e4m3_decode(np.arange(0, 0x7F, dtype=np.uint8)).astype(np.float64)
    mids = ((vals[:-1] + vals[1:]) / 2).astype(np.float32)
    near = np.concatenate([np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(1e9))])
    rng = np.random.default_rng(0)
    H, d, bs = 2, 128, 32
    x = np.concatenate([[448.0], vals[:127], mids, near, [0.0, 2.0 ** -10, 2.0 ** -11, 1e-30, 1e-42, 447.99997],
                        rng.uniform(-448, 448, bs * d), rng.uniform(-0.03, 0.03, bs * d)]).astype(np.float32)
    x = np.concatenate([x[:1], -x[1:]])[:bs * d]
    gpu, _ = _pair(cuda, 1, H, d, 4, bs, 1)
    both = torch.from_numpy(np.stack([x, x * 2.0 ** 20]).reshape(H, bs, d)).permute(1, 0, 2)[None]
    gpu.write_block(0, [0], [0], both.to(cuda), both.flip(1).to(cuda))
    blk = gpu.block_tables[0][0]
    want = torch.from_numpy(e4m3_encode(x)).view(bs, d)
    assert torch.equal(want, torch.from_numpy(x).view(bs, d).to(FP8).view(torch.uint8))
    k, v = gpu.k_pool.view(torch.uint8)[0, blk].cpu(), gpu.v_pool.view(torch.uint8)[0, blk].cpu()
    assert gpu.scales[0, :, blk, 0].tolist() == [1.0, 2.0 ** 20]
    assert torch.equal(k[0], want) and torch.equal(k[1], want)
    assert torch.equal(v[0], want.flip(0).t()) and torch.equal(v[1], want.flip(0).t())


@pytest.mark.parametrize("dtype,C", [(F32, 5), (BF16, 21), (F16, 3)])
def test_not_finite(cuda, dtype, C):
    g = torch.Generator().manual_seed(C)
    gpu, cpu = _pair(cuda, 1, 2, 64, 8, 16, 1)
    for start, mag in ((0, 1.0), (C, 30.0), (2, 0.1)):
        x = (torch.randn(1, C, 2, 64, generator=g) * mag).to(dtype)
        x[0, 0, 1, 7], x[0, C - 1, 0, 0], x[0, 1, 1, 63] = float("nan"), float("inf"), float("-inf")
        gpu.write_block(0, [0], [start], x.to(cuda), -x.to(cuda))
        cpu.write_block(0, [0], [start], x, -x)
        _same(gpu, cpu)


def test_zeros_and_tiny_values(cuda):
    gpu, cpu = _pair(cuda, 1, 2, 16, 8, 4, 1)
    x = torch.zeros(1, 6, 2, 16)
    x[0, 3, 0, 2], x[0, 4, 1, 1], x[0, 5, 1, 2] = 1e-44, 1e-38, -3e38
    for start in (0, 1):
        gpu.write_block(0, [0], [start], x.to(cuda), x.to(cuda))
        cpu.write_block(0, [0], [start], x, x)
        _same(gpu, cpu)


@pytest.mark.parametrize("layout", ["packed", "heads_first", "columns", "expanded"])
def test_device_writes_of_views(cuda, layout):
    """The layers of a round, keys and values in any strides; the first layer allocates."""
    g = torch.Generator().manual_seed(2)
    H, d, bs, layers, B, C = 2, 64, 16, 3, 3, 9
    gpu, cpu = _pair(cuda, layers, H, d, 32, bs, B)
    sids, starts = [2, 0, 1], [0, 0, 0]
    sid, st = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (sids, starts))
    for _ in range(2):
        for layer in range(layers):
            x = torch.randn(B, C, 3 * H, d, generator=g).to(BF16)
            if layout == "expanded":  # one head's keys for all heads
                x = x[:, :, :1].expand(B, C, 3 * H, d)
            kn, vn = x[:, :, H:2 * H], x[:, :, 2 * H:]
            y = x.to(cuda) if layout != "expanded" else x[:, :, :1].to(cuda).expand(B, C, 3 * H, d)
            if layout == "heads_first":
                y = y.transpose(1, 2).contiguous().transpose(1, 2)
            elif layout == "columns":
                y = y.transpose(2, 3).contiguous().transpose(2, 3)
            gpu.write_block_device(layer, sid, st, y[:, :, H:2 * H], y[:, :, 2 * H:], alloc=layer == 0,
                                   plan=WritePlan())
            cpu.write_block(layer, sids, starts, kn, vn)
        starts = [C] * B
        st = torch.full_like(st, C)
    _same(gpu, cpu)


@pytest.mark.parametrize("dtype,H,d,bs", [(F32, 2, 128, 16), (BF16, 3, 64, 64), (F32, 1, 80, 48), (F32, 2, 64, 32),
                                           (F32, 1, 128, 128), (F16, 1, 256, 64)])
def test_pieces_of_pages(cuda, dtype, H, d, bs):
    """Chunks that begin and end inside a page's 16-byte pieces, under scales that grow from 1e-25 to 1e25 (past
    what a rounded reciprocal may stand in for, both ways), rows at odd addresses beside aligned ones."""
    g = torch.Generator().manual_seed(d + bs)
    gpu, cpu = _pair(cuda, 1, H, d, 16, bs, 1)
    odd, _ = _pair(cuda, 1, H, d, 16, bs, 1)
    at, C = 0, bs // 2 + 5
    for mag in (1e-25, 1e-19, 1e-18, 1e-6, 1.0, 0.3, 77.7, 1e17, 1e18, 1e25):
        for start in (at, max(0, at - C + 3)):
            kn, vn = ((torch.randn(1, C, H, d, generator=g) * mag).to(dtype) for _ in range(2))
            kn[0, 1, 0, :4] = torch.tensor([0.0, -0.0, 448.0, -1e-30])
            gpu.write_block(0, [0], [start], kn.to(cuda), vn.to(cuda))
            cpu.write_block(0, [0], [start], kn, vn)
            wide = torch.zeros(2, 1, C, H, d + 1, dtype=dtype, device=cuda)
            wide[0, ..., 1:], wide[1, ..., 1:] = kn.to(cuda), vn.to(cuda)
            odd.write_block(0, [0], [start], wide[0, ..., 1:], wide[1, ..., 1:])
        at += 7
        _same(gpu, cpu)
        _same(odd, cpu)


def test_exhaustion_and_table_width(cuda):
    gpu, cpu = _pair(cuda, 2, 2, 16, 5, 4, 3)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 9, 2, 16, generator=g)
    with pytest.raises(BlockExhaustedError):
        gpu.write_block(0, [0, 1, 2], [0, 0, 0], x.to(cuda), x.to(cuda))
    with pytest.raises(RefExhausted):
        cpu.write_block(0, [0, 1, 2], [0, 0, 0], x, x)
    _same(gpu, cpu)
    ids = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    gpu2, _ = _pair(cuda, 2, 2, 16, 5, 4, 3)
    gpu2.write_block_device(0, ids, torch.zeros_like(ids), x.to(cuda), x.to(cuda))
    with pytest.raises(BlockExhaustedError):
        gpu2.seq_lengths
    assert torch.equal(gpu2.k_pool.view(torch.uint8), gpu.k_pool.view(torch.uint8))
    assert torch.equal(gpu2.scales, gpu.scales) and gpu2.seq_lengths == gpu.seq_lengths


def test_rows_outside_the_chunk_keep_their_bytes(cuda):
    """A chunk that does not raise the scale leaves every other byte of both pools as it was."""
    g = torch.Generator().manual_seed(5)
    gpu, _ = _pair(cuda, 2, 2, 64, 6, 16, 2)
    big = torch.randn(2, 40, 2, 64, generator=g) * 10
    gpu.write_block(1, [0, 1], [0, 0], big.to(cuda), big.to(cuda))
    before = [t.clone() for t in (gpu.k_pool.view(torch.uint8), gpu.v_pool.view(torch.uint8), gpu.scales)]
    gpu.write_block(1, [1], [21], big[:1, :3].to(cuda) * 0.01, big[:1, :3].to(cuda) * 0.01)
    after = [gpu.k_pool.view(torch.uint8), gpu.v_pool.view(torch.uint8), gpu.scales]
    assert torch.equal(before[2], after[2])
    blk = gpu.block_tables[1][1]
    k, v = after[0].clone(), after[1].clone()
    k[1, blk, :, 5:8], v[1, blk, :, :, 5:8] = before[0][1, blk, :, 5:8], before[1][1, blk, :, :, 5:8]
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    assert not torch.equal(after[0], before[0])


# ---------------------------------------------------------------------------
# normed and rotated on the way
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("hq,H,d,R,bs,C,inter,layout", [
    (4, 2, 64, 64, 16, 1, False, "packed"),
    (6, 2, 128, 128, 16, 6, False, "packed"),
    (3, 1, 128, 64, 32, 37, True, "packed"),
    (4, 2, 64, 32, 16, 100, False, "dense"),
    (2, 2, 10, 6, 7, 9, True, "dense"),       # no whole pieces
    (2, 1, 256, 256, 64, 130, False, "dense"),  # blocks staged in parts
    (4, 2, 128, 128, 64, 130, True, "packed"),  # blocks of more than 64 KiB staged at once
    (4, 2, 64, 64, 64, 5, False, "packed"),     # few rows of a large block
    (2, 2, 64, 64, 16, 5, False, "columns"),
])
def test_rotating_append(cuda, dtype, normed, hq, H, d, R, bs, C, inter, layout):
    """The queries are ``rotary_embed``'s; the codes are those of the fp32 keys that ``rotary_embed``
    leaves, where their last bits agree: both are within 2e-6 (|a| + |b|) <= 3e-6 of the pair's
    length (tests/test_gpu_head_norm.py), so a scale may be 6e-6 off, and a key that near a border
    between two codes (a share of 2 * 6e-6 / 2^-4 of them, 2e-4) takes the one or the other."""
    g = torch.Generator().manual_seed(d + C)
    rot = Rotary(d, cuda, rotary_dim=R, interleaved=inter)
    norm = HeadNorm(d, cuda, 1 + 0.3 * torch.randn(d, generator=g), 1 + 0.3 * torch.randn(d, generator=g)) \
        if normed else None
    a, cpu = _pair(cuda, 1, H, d, 64, bs, 3)
    b, _ = _pair(cuda, 1, H, d, 64, bs, 3)
    lens = [2, 0, bs + 3]
    for s, n in enumerate(lens):
        if n:
            x = torch.randn(1, n, H, d, generator=g) * 0.5
            for kv in (a, b):
                kv.write_block(0, [s], [0], x.to(cuda), x.to(cuda))
    sid, start = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([2, 0, 1], [bs + 3, 2, 0]))
    x = torch.randn(3, C, hq + 2 * H, d, generator=g).to(dtype).to(cuda)
    if layout == "columns":
        x = x.transpose(2, 3).contiguous().transpose(2, 3)
    q, k, v = x.split([hq, H, H], dim=2)
    if layout == "dense":
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pos = start[:, None] + torch.arange(C, dtype=torch.int32, device=cuda)
    qe, _ = rotary_embed(q, None, rot, pos, norm=norm)
    _, ke = rotary_embed(q, k, rot, pos, key_dtype=F32, norm=norm)
    qo = rotary_append(q, k, v, a, 0, sid, start, rot, norm=norm)
    assert torch.equal(qo, qe)
    b.write_block_device(0, sid, start, ke, v.float())
    assert a.block_tables == b.block_tables and a.seq_lengths == b.seq_lengths
    assert torch.equal(a.v_pool.view(torch.uint8), b.v_pool.view(torch.uint8))
    assert torch.equal(a.scales[..., 1], b.scales[..., 1])
    sa, sb = a.scales[..., 0], b.scales[..., 0]
    assert bool(((sa - sb).abs() <= 6e-6 * sb).all())
    ka, kb = a.k_pool.float(), b.k_pool.float()
    differ = ka != kb
    assert float(differ.float().mean()) <= 1e-3
    step = torch.maximum(kb.abs() * 0.125, torch.tensor(2.0 ** -9, device=cuda))
    assert bool(((ka - kb).abs() <= step)[differ].all())


def test_rotating_append_given_positions_and_no_query(cuda):
    g = torch.Generator().manual_seed(6)
    rot = Rotary(64, cuda, sections=(8, 12, 12))
    a, _ = _pair(cuda, 1, 2, 64, 8, 16, 1)
    b, _ = _pair(cuda, 1, 2, 64, 8, 16, 1)
    k, v = (torch.randn(1, 7, 2, 64, generator=g).to(BF16).to(cuda) for _ in range(2))
    pos = torch.randint(0, 1000, (3, 1, 7), generator=g).to(cuda)
    ids = torch.zeros(1, dtype=torch.int32, device=cuda)
    assert rotary_append(None, k, v, a, 0, ids, ids, rot, pos) is None
    rotary_append(k, k, v, b, 0, [0], [0], rot, pos)
    assert torch.equal(a.k_pool.view(torch.uint8), b.k_pool.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    with pytest.raises(ValueError):
        rotary_append(None, k, v, a, 0, ids, ids, rot)  # several axes need positions


# ---------------------------------------------------------------------------
# reading back
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("H,d,bs,n", [(2, 64, 16, 333), (2, 128, 16, 16), (1, 128, 32, 47), (2, 64, 64, 200),
                                      (3, 10, 7, 20), (2, 64, 16, 1), (1, 1, 1, 5), (2, 48, 8, 30), (4, 256, 16, 70)])
def test_gather(cuda, H, d, bs, n):
    g = torch.Generator().manual_seed(n)
    gpu, cpu = _pair(cuda, 2, H, d, -(-n // bs) + 3, bs, 2)
    x = _random(g, (1, n + 1, H, d), F32)
    y = torch.randn(1, n + 1, H, d, generator=g)
    for kv, a, b in ((gpu, x.to(cuda), y.to(cuda)), (cpu, x, y)):
        kv.write_block(1, [1], [0], a, b)
    deq = cpu.dequantized()
    table = cpu.block_tables[1]
    want = torch.stack([t[1, table].reshape(-1, H, d)[:n] for t in (deq.k, deq.v)])
    assert torch.equal(gather_ctx(gpu, 1, 1, n).cpu(), want)
    for dtype in (F32, BF16, F16):
        got = gather_ctx(gpu, 1, 1, n, dtype=dtype)
        assert got.dtype == dtype and got.shape == (2, n, H, d)
        assert torch.equal(got.cpu(), want.to(dtype))
    assert gather_ctx(gpu, 1, 1, 0, dtype=BF16).shape == (2, 0, H, d)
    with pytest.raises(IndexError):
        gather_ctx(gpu, 1, 1, (-(-n // bs) + 1) * bs + 1)
    with pytest.raises(IndexError):
        gather_ctx(gpu, 2, 1, n)
    with pytest.raises(ValueError):
        gather_ctx(gpu, 1, 1, n, dtype=torch.float64)


def test_gather_of_other_pools_as_a_type(cuda):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 20, 2, 64, generator=g).to(cuda)
    one = PagedKVCache(1, 2, 64, 4, 16, cuda, FP8)
    half = PagedKVCache(1, 2, 64, 4, 16, cuda, F16)
    for kv in (one, half):
        kv.add_sequence(0)
        kv.write_block(0, [0], [0], x, x)
    assert torch.equal(gather_ctx(one, 0, 0, 20, dtype=BF16), gather_ctx(one, 0, 0, 20).to(BF16))
    assert torch.equal(gather_ctx(half, 0, 0, 20, dtype=F16), gather_ctx(half, 0, 0, 20))
    with pytest.raises(ValueError):
        gather_ctx(half, 0, 0, 20, dtype=BF16)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _filled(cuda, lens, H, d, bs, seed, mags=None, layers=1, layer=0):
    """A cache of random contexts, loaded page by page with scales of each block and head."""
    g = torch.Generator().manual_seed(seed)
    nb = [-(-n // bs) for n in lens]
    cap = sum(nb) + 3
    perm = torch.randperm(cap, generator=g).tolist()
    tables, at = [], 0
    for n in nb:
        tables.append(perm[at:at + n])
        at += n
    kv = PagedKVCache(layers, H, d, cap, bs, cuda, FP8, max_seqs=len(lens), max_blocks_per_seq=max(nb + [1]),
                      head_scales=True)
    kv.load_state(tables, lens, perm[at:])
    k, v = torch.randn(cap, H, bs, d, generator=g), torch.randn(cap, H, d, bs, generator=g)
    if mags is not None:
        v = v * torch.tensor([[mags(b, h) for h in range(H)] for b in range(cap)])[..., None, None]
    for pool, x, kind in ((kv.k_pool, k, 0), (kv.v_pool, v, 1)):
        s = x.abs().amax(dim=(2, 3)) / 448.0
        codes = torch.where(s[..., None, None] > 0, x / s[..., None, None], torch.zeros_like(x)).clamp(-448, 448)
        pool[layer].view(torch.uint8).copy_(codes.to(FP8).view(torch.uint8))
        kv.scales[layer, :, :, kind] = s.t().to(cuda)
    return kv, g


def _context64(kv, layer, sid, n):
    """Keys and values (H, n, d) of a sequence in float64, on the CPU."""
    bs, H, d = kv.block_size, kv.num_kv_heads, kv.head_dim
    blocks = torch.tensor(kv.block_tables[sid][:-(-n // bs)], dtype=torch.long)
    deq = lambda t: torch.from_numpy(e4m3_decode(t.view(torch.uint8).cpu().numpy())).double()  # noqa: E731
    k, v, s = deq(kv.k_pool[layer])[blocks], deq(kv.v_pool[layer])[blocks], kv.scales[layer].cpu().double()[:, blocks]
    s = s.permute(1, 0, 2)[..., None, None]
    k, v = k * s[:, :, 0], v * s[:, :, 1]
    return k.transpose(0, 1).reshape(H, -1, d)[:, :n], v.permute(1, 0, 3, 2).reshape(H, -1, d)[:, :n]


def _check(out, q, kv, layer, sids, starts, scale=None, rows=None):
    """Every row against float64, within the tolerance above."""
    B, C, hq, d = q.shape
    H = kv.num_kv_heads
    scale = d ** -0.5 if scale is None else scale
    q_dtype = q.dtype
    out, q = out.detach().cpu().double(), q.detach().cpu()
    half = torch.finfo(q.dtype).eps / 2
    tiny = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[q.dtype]
    q = q.double()
    for b, (sid, s0) in enumerate(zip(sids, starts)):
        k, v = _context64(kv, layer, sid, s0 + C)
        for j in (range(C) if rows is None else rows):
            n = s0 + j + 1
            qq = q[b, j].view(H, hq // H, d)
            z = torch.matmul(qq, k[:, :n].transpose(1, 2)) * scale
            size = (torch.matmul(qq.abs(), k[:, :n].abs().transpose(1, 2)) * abs(scale)).amax(-1, keepdim=True)
            p = torch.softmax(z, -1)
            o, a = torch.matmul(p, v[:, :n]), torch.matmul(p, v[:, :n].abs())
            eps_p = 2 * (d + 4) * 2.0 ** -24 * size + 2.0 ** -20 + (2.0 ** -11 if q_dtype is BF16 else 2.0 ** -17)
            bound = half * o.abs() + tiny / 2 + (1 + half) * eps_p * a
            err = (out[b, j].view(H, hq // H, d) - o).abs()
            assert bool((err <= bound).all()), (b, j, float((err / bound).max()))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hq,H,d,bs,C,starts", [
    (14, 2, 64, 16, 1, [0, 15, 16, 17, 63, 64, 65, 599]),       # decode, from the first token
    (12, 2, 128, 16, 6, [0, 1, 250, 1000, 58, 59]),              # verify chunks that end inside and at pages
    (16, 2, 128, 32, 7, [31, 32, 400, 777]),
    (14, 2, 64, 64, 9, [2000, 37, 300, 0]),
    (4, 4, 64, 16, 3, [100, 5]),                                 # no sharing of heads
    (40, 1, 128, 16, 2, [333, 64]),                              # one kv head of many
    (6, 2, 128, 48, 4, [100, 47]),                               # blocks of three units
    (4, 2, 10, 7, 5, [0, 20, 33]),                               # off the matrix path: rows, blocks
    (4, 2, 96, 16, 5, [70]),
    (2, 1, 256, 16, 2, [100]),
    (4, 2, 64, 8, 3, [50, 9]),
    (3, 3, 1, 1, 2, [4]),
])
def test_attention(cuda, dtype, hq, H, d, bs, C, starts):
    kv, g = _filled(cuda, [s + C for s in starts], H, d, bs, d + C)
    q = torch.randn(len(starts), C, hq, d, generator=g).to(dtype).to(cuda)
    sids = list(range(len(starts)))
    out = verify_attention(q, kv, 0, sids, starts, max(starts) + C)
    assert out.dtype == dtype and out.shape == q.shape
    _check(out, q, kv, 0, sids, starts)
    # the same bits again, with a looser bound, device tensors, another order, an output of the caller's
    sid, st = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (sids, starts))
    own = torch.full_like(q, 7.0)
    assert verify_attention(q, kv, 0, sid, st, max(starts) + C, out=own) is own
    assert torch.equal(own, out)
    assert kv.seq_lengths == [s + C for s in starts]  # nothing was flagged


@pytest.mark.parametrize("dtype,hq,H,d,C,starts", [
    (BF16, 14, 2, 64, 9, [9000, 20000, 5]),
    (BF16, 12, 2, 128, 1, [16383, 1, 4097]),
    (F16, 12, 2, 128, 6, [7001] * 3),
    (F32, 12, 2, 128, 5, [5000, 100]),
])
def test_long_contexts(cuda, dtype, hq, H, d, C, starts):
    kv, g = _filled(cuda, [s + C for s in starts], H, d, 16, C)
    q = torch.randn(len(starts), C, hq, d, generator=g).to(dtype).to(cuda)
    out = verify_attention(q, kv, 0, list(range(len(starts))), starts, max(starts) + C)
    _check(out, q, kv, 0, list(range(len(starts))), starts, rows=sorted({0, C // 2, C - 1}))


@pytest.mark.parametrize("dtype,B,hq,H,d,C", [(BF16, 140, 12, 2, 128, 6), (F16, 300, 14, 2, 64, 1),
                                              (F32, 70, 4, 2, 64, 2)])
def test_many_short_sequences(cuda, dtype, B, hq, H, d, C):
    starts = [(i * 37) % 211 for i in range(B)]
    kv, g = _filled(cuda, [s + C for s in starts], H, d, 16, B)
    q = torch.randn(B, C, hq, d, generator=g).to(dtype).to(cuda)
    out = verify_attention(q, kv, 0, list(range(B)), starts, 211 + C)
    pick = list(range(0, B, 7))
    _check(out[pick], q[pick], kv, 0, pick, [starts[i] for i in pick])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,hq", [(64, 14), (128, 6)])
def test_prompt_sized_chunks(cuda, dtype, d, hq):
    """Chunks of more rows than one tile, from the first position and behind a context."""
    C, starts = 133, [0, 300]
    kv, g = _filled(cuda, [s + C for s in starts], 2, d, 16, d)
    q = torch.randn(2, C, hq, d, generator=g).to(dtype).to(cuda)
    out = verify_attention(q, kv, 0, [0, 1], starts, 433)
    _check(out, q, kv, 0, [0, 1], starts, rows=[0, 1, 15, 16, 63, 64, 100, 132])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_value_scales_of_every_size(cuda, dtype, d):
    """Blocks and heads whose values lie from 0 and 1e-20 to 1e20 (1e-4 to 1e3 for fp16 outputs) side by side."""
    sizes = [1.0, 0.0, 1e-4, 1e3, 1e-2, 30.0] if dtype == F16 else [1.0, 0.0, 1e-7, 1e6, 1e-20, 1e20]
    starts, C = [900, 50, 333], 4
    kv, g = _filled(cuda, [s + C for s in starts], 2, d, 16, 7, mags=lambda b, h: sizes[(b * 7 + h) % len(sizes)])
    q = torch.randn(3, C, 12, d, generator=g).to(dtype).to(cuda)
    _check(verify_attention(q, kv, 0, [0, 1, 2], starts, 904), q, kv, 0, [0, 1, 2], starts)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_peaked_rows_and_scales(cuda, dtype):
    """Rows whose weight jumps from key to key, a large and a negative softmax scale, and scores near 0."""
    starts, C = [700, 64, 3], 5
    kv, g = _filled(cuda, [s + C for s in starts], 2, 64, 16, 8)
    q = torch.randn(3, C, 8, 64, generator=g).to(dtype).to(cuda)
    for scale in (2.0, -0.3, 1e-6, 0.0):
        out = verify_attention(q, kv, 0, [0, 1, 2], starts, 705, scale=scale)
        _check(out, q, kv, 0, [0, 1, 2], starts, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32), (10, 7)])
def test_what_masked_places_hold(cuda, dtype, d, bs):
    """NaN codes behind the last position, in pages that the table holds beyond it, and at a later
    chunk position reach no row that does not attend them; a row that attends one is NaN."""
    starts, C = [45, 100, 0], 6
    lens = [s + C for s in starts]
    kv, g = _filled(cuda, [n + 2 * bs for n in lens], 2, d, bs, 9)
    q = torch.randn(3, C, 6, d, generator=g).to(dtype).to(cuda)
    clean = verify_attention(q, kv, 0, [0, 1, 2], starts, max(lens))
    _check(clean, q, kv, 0, [0, 1, 2], starts)
    k8, v8 = kv.k_pool.view(torch.uint8), kv.v_pool.view(torch.uint8)
    for s, n in enumerate(lens):
        for pos in range(n, n + bs + 3):
            blk, off = kv.block_tables[s][pos // bs], pos % bs
            k8[0, blk, :, off], v8[0, blk, :, :, off] = 0x7F, 0xFF
    assert torch.equal(verify_attention(q, kv, 0, [0, 1, 2], starts, max(lens)), clean)
    # the values of chunk token 3 of entry 1, in one dimension of one head
    pos = starts[1] + 3
    v8[0, kv.block_tables[1][pos // bs], 1, 2, pos % bs] = 0x7F
    got = verify_attention(q, kv, 0, [0, 1, 2], starts, max(lens))
    assert torch.equal(got[[0, 2]], clean[[0, 2]]) and torch.equal(got[1, :3], clean[1, :3])
    bad = torch.zeros(3, 6, d, dtype=torch.bool, device=cuda)
    bad[:, 3:, 2] = True
    assert bool(got[1, 3:][bad].isnan().all()) and torch.equal(got[1, 3:][~bad], clean[1, 3:][~bad])
    # the keys of chunk token 4
    pos = starts[1] + 4
    k8[0, kv.block_tables[1][pos // bs], 0, pos % bs, 0] = 0x7F
    got2 = verify_attention(q, kv, 0, [0, 1, 2], starts, max(lens))
    assert torch.equal(got2[1, :4].nan_to_num(7.0), got[1, :4].nan_to_num(7.0))
    assert bool(got2[1, 4:, :3].isnan().all()) and torch.equal(got2[1, 4:, 3:].nan_to_num(7.0), got[1, 4:, 3:].nan_to_num(7.0))


def test_infinite_and_nan_queries_stay_in_their_rows(cuda):
    starts, C = [100, 20], 3
    kv, g = _filled(cuda, [s + C for s in starts], 2, 64, 16, 10)
    q = torch.randn(2, C, 4, 64, generator=g).to(BF16).to(cuda)
    clean = verify_attention(q, kv, 0, [0, 1], starts, 103)
    bad = q.clone()
    bad[0, 1, 2, 5], bad[1, 0, 0, 0] = float("nan"), float("inf")
    got = verify_attention(bad, kv, 0, [0, 1], starts, 103)
    keep = torch.ones(2, C, 4, dtype=torch.bool, device=cuda)
    keep[0, 1, 2] = keep[1, 0, 0] = False
    assert torch.equal(got[keep], clean[keep]) and bool(got[0, 1, 2].isnan().all()) and bool(got[1, 0, 0].isnan().any())


def test_forbidden_reads_are_flagged(cuda):
    kv, g = _filled(cuda, [50, 20], 2, 64, 16, 11)
    q = torch.randn(2, 3, 4, 64, generator=g).to(BF16).to(cuda)
    verify_attention(q, kv, 0, [0, 1], [47, 18], 50)  # 18 + 3 > 20
    with pytest.raises(IndexError):
        kv.seq_lengths
    assert kv.seq_lengths == [50, 20]
    st = torch.tensor([47, -1], dtype=torch.int32, device=cuda)
    ids = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    verify_attention(q, kv, 0, ids, st, 50)
    with pytest.raises(IndexError):
        kv.seq_lengths
    kv.tables_dev[0, 1] = 10 ** 6  # a block id outside the pool reads block 0
    out = verify_attention(q, kv, 0, ids, torch.tensor([47, 17], dtype=torch.int32, device=cuda), 50)
    with pytest.raises(IndexError):
        kv.seq_lengths
    _check(out[1:], q[1:], kv, 0, [1], [17])


def test_offsets_past_32_bits(cuda):
    """The last layer of a pool of more than 2^32 bytes of keys."""
    layers, H, d, bs = 9, 2, 128, 64
    cap = (1 << 32) // (8 * H * d * bs) + 1
    kv = PagedKVCache(layers, H, d, cap, bs, cuda, FP8, head_scales=True)
    assert kv.k_pool.numel() > 1 << 32
    g = torch.Generator().manual_seed(12)
    kv.add_sequence(0)
    x, y = (torch.randn(1, 200, H, d, generator=g).to(BF16).to(cuda) for _ in range(2))
    kv.write_block(layers - 1, [0], [0], x, y)
    deq = gather_ctx(kv, layers - 1, 0, 200)
    err = (deq - torch.stack([x[0], y[0]]).float()).abs()
    assert bool((err <= 2.0 ** -4 * deq.abs() * (1 + 2.0 ** -3) + 1e-4).all())
    q = torch.randn(1, 2, 4, d, generator=g).to(BF16).to(cuda)
    out = verify_attention(q, kv, layers - 1, [0], [198], 200).double()
    p = torch.softmax(torch.einsum("jhe,nhe->jhn", q[0].cpu().double(), deq[0].cpu().double().repeat_interleave(2, 1))
                      .masked_fill(torch.arange(200) > torch.tensor([198, 199])[:, None, None], -math.inf) * d ** -0.5, -1)
    want = torch.einsum("jhn,nhe->jhe", p, deq[1].cpu().double().repeat_interleave(2, 1))
    assert float((out[0].cpu() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 1e-4


# ---------------------------------------------------------------------------
# together, as a serving loop uses them
# ---------------------------------------------------------------------------

def test_a_round_of_layers(cuda):
    """Prompts, then two rounds: norm, rotate, quantise and write, attend, rewind -- layer by layer, by
    lists and by device tensors, with and without a plan; every output against float64 of what is stored."""
    g = torch.Generator().manual_seed(13)
    layers, hq, H, d, bs, C, B = 2, 6, 2, 64, 16, 4, 3
    kv = PagedKVCache(layers, H, d, 64, bs, cuda, FP8, head_scales=True)
    rot = Rotary(d, cuda, base=1e6)
    norm = HeadNorm(d, cuda, 1 + 0.2 * torch.randn(d, generator=g), 1 + 0.2 * torch.randn(d, generator=g))
    for s in range(B):
        kv.add_sequence(s)
        n = 11 + 30 * s
        for layer in range(layers):
            x = torch.randn(1, n, hq + 2 * H, d, generator=g).to(BF16).to(cuda)
            rotary_append(*x.split([hq, H, H], dim=2), kv, layer, [s], [0], rot, alloc=layer == 0, norm=norm)
    sids = [2, 0, 1]
    for _ in range(2):
        starts = [kv.seq_lengths[s] for s in sids]
        sid, st = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (sids, starts))
        plan = None
        for layer in range(layers):
            x = torch.randn(B, C, hq + 2 * H, d, generator=g).to(BF16).to(cuda)
            q = rotary_append(*x.split([hq, H, H], dim=2), kv, layer, sid, st, rot, alloc=layer == 0, norm=norm)
            plan = plan or VerifyPlan(kv, sid, st, C, hq, max(starts) + C)
            out = verify_attention(q, kv, layer, sid, st, max(starts) + C, plan=plan)
            _check(out, q, kv, layer, sids, starts)
            assert torch.equal(out, paged_attention_extend(q, kv, layer, sids, starts, hq))
            last = paged_attention_decode(q[:, -1].contiguous(), kv, layer, sids, [s + C for s in starts], hq)
            _check(last[:, None], q[:, -1:], kv, layer, sids, [s + C - 1 for s in starts])
        kv.rewind_device(sid, st + 2, torch.zeros_like(st))
        assert kv.seq_lengths[2] == starts[0] + 2


def test_verify_step_and_appending_attention(cuda):
    """The framework's round over this cache: ``VerifyStep`` and the later layers' append and attention."""
    from engine.spec_scheduler import VerifyStep

    g = torch.Generator().manual_seed(14)
    layers, hq, H, d, gamma, B = 3, 4, 2, 64, 3, 2
    C = gamma + 1
    kv, other = (PagedKVCache(layers, H, d, 32, 16, cuda, FP8, head_scales=True) for _ in range(2))
    for cache in (kv, other):
        gg = torch.Generator().manual_seed(15)
        for s, n in enumerate((20, 33)):
            cache.add_sequence(s)
            for layer in range(layers):
                x = torch.randn(1, n, H, d, generator=gg).to(cuda)
                cache.write_block(layer, [s], [0], x, x * 2)
    q, k, v = ([torch.randn(B, C, n, d, generator=g).to(BF16).to(cuda) for _ in range(layers)] for n in (hq, H, H))
    outs = VerifyStep(kv, gamma, 1.0).attend_layers([0, 1], [20, 33], q, k, v)
    sid, st = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, 1], [20, 33]))
    for layer in range(layers):
        other.write_block_device(layer, sid, st, k[layer], v[layer], alloc=layer == 0)
        want = verify_attention(q[layer], other, layer, sid, st, 37)
        assert torch.equal(outs[layer], want)
        _check(want, q[layer], other, layer, [0, 1], [20, 33])
    plan, wplan = VerifyPlan(kv, sid, st, C, hq, 37), WritePlan()
    got = append_verify_attention(q[1], k[1], v[1], kv, 1, sid, st, 37, plan, wplan)
    assert torch.equal(got, outs[1])
    with pytest.raises(ValueError):
        SharedPrefix(kv, [0, 0], [16, 16], C, hq)
    with pytest.raises(ValueError):
        kv.rewind_append_device(sid, None, None, st, k[0], v[0])


@pytest.mark.parametrize("hq,H,d", [(14, 2, 64), (12, 2, 128)])
def test_draft_loop(cuda, hq, H, d):
    """Draft steps of several layers, eager and as one captured graph (many attention calls in one pool of
    memory): the same bits in every replay, and float64's attention of what is stored."""
    from engine.spec_scheduler import DraftLoop

    g = torch.Generator().manual_seed(d)
    layers, gamma, B, V, ctx = 3, 3, 4, 97, [700, 15, 33, 1]
    kv = PagedKVCache(layers, H, d, 128, 16, cuda, FP8, head_scales=True)
    for s, n in enumerate(ctx):
        kv.add_sequence(s)
        for layer in range(layers):
            kv.write_block(layer, [s], [0], *(torch.randn(1, n, H, d, generator=g).to(BF16).to(cuda) for _ in "kv"))
    q, k, v = ([[torch.randn(B, 1, n, d, generator=g).to(BF16).to(cuda) for _ in range(layers)] for _ in range(gamma)]
               for n in (hq, H, H))
    logits = [torch.randn(B, V, generator=g).to(cuda) for _ in range(gamma)]
    noise = [torch.empty(B, V).exponential_(generator=g).to(cuda) for _ in range(gamma)]
    sid, at = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (range(B), ctx))
    loop = DraftLoop(kv, gamma, 1.0)
    run = lambda: loop.run(sid, at, max(ctx), q, k, v, logits, noise)  # noqa: E731
    run()
    want_p, want = run()  # the same rows again, into scales that no longer grow
    for layer in range(layers):
        _check(want[-1][layer], q[-1][layer], kv, layer, list(range(B)), [n + gamma - 1 for n in ctx])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got_p, got = run()
    before = kv.k_pool.view(torch.uint8).clone()
    for _ in range(3):
        for row in got:
            for o in row:
                o.zero_()
        verify_attention(q[0][0], kv, 0, sid, at, max(ctx) + 1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got_p, want_p) and torch.equal(kv.k_pool.view(torch.uint8), before)
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


def test_alignment_clears_the_scales(cuda):
    """Blocks that a draft alignment hands out start with zero scales in every layer and head."""
    kv = PagedKVCache(2, 3, 16, 8, 4, cuda, FP8, head_scales=True)
    kv.add_sequence(0)
    x = torch.ones(1, 4, 3, 16, device=cuda)
    for layer in range(2):
        kv.write_block(layer, [0], [0], x, x)
    kv.scales.fill_(5.0)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    tokens = torch.zeros(1, 4, dtype=torch.int32, device=cuda)
    cn, cp, ct = i32(0), i32(0), torch.zeros(1, 4, dtype=torch.int32, device=cuda)
    kv.align_device(i32(0), i32(3), i32(3), i32(0), tokens, cn, cp, ct, max_len=8)
    first, second = kv.block_tables[0]
    assert bool((kv.scales[:, :, second] == 0).all()) and bool((kv.scales[:, :, first] == 5).all())


def test_captured_graphs_and_streams(cuda):
    """Two graphs captured one after another and replayed on two streams side by side, with eager calls
    between, give the eager results: each graph has a workspace of its own."""
    starts, C = [3000, 900, 40], 5
    kv, g = _filled(cuda, [s + C for s in starts], 2, 128, 16, 16)
    ids = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    st = torch.tensor(starts, dtype=torch.int32, device=cuda)
    qs = [torch.randn(3, C, 12, 128, generator=g).to(BF16).to(cuda) for _ in range(2)]
    call = lambda q: verify_attention(q, kv, 0, ids, st, 3005)  # noqa: E731
    want = [call(q) for q in qs]
    for q, w in zip(qs, want):
        _check(w, q, kv, 0, [0, 1, 2], starts, rows=[0, C - 1])
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(q))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [call(q) for q in qs]
        torch.cuda.synchronize()
        for w, o, e in zip(want, outs, eager):
            assert torch.equal(o, w) and torch.equal(e, w)
    with torch.cuda.stream(streams[0]):
        a = call(qs[0])
    with torch.cuda.stream(streams[1]):
        b = call(qs[1])
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_captured_writes(cuda):
    """A captured allocating write, replayed on new contents, is the eager one's."""
    g = torch.Generator().manual_seed(17)
    a, _ = _pair(cuda, 2, 2, 64, 16, 16, 2)
    b, _ = _pair(cuda, 2, 2, 64, 16, 16, 2)
    ids = torch.tensor([1, 0], dtype=torch.int32, device=cuda)
    st = torch.zeros(2, dtype=torch.int32, device=cuda)
    k, v = (torch.randn(2, 5, 2, 64, generator=g).to(BF16).to(cuda) for _ in range(2))
    a.write_block_device(0, ids, st, k, v)
    b.write_block_device(0, ids, st, k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.write_block_device(0, ids, st, k, v)
        a.write_block_device(1, ids, st, k, v, alloc=False)
    for i in range(4):
        st += 5
        k.mul_(1.7)
        v.mul_(-0.6)
        graph.replay()
        for layer in range(2):
            b.write_block_device(layer, ids, st, k, v, alloc=layer == 0)
        torch.cuda.synchronize()
        assert torch.equal(a.k_pool.view(torch.uint8), b.k_pool.view(torch.uint8))
        assert torch.equal(a.v_pool.view(torch.uint8), b.v_pool.view(torch.uint8))
        assert torch.equal(a.scales, b.scales) and torch.equal(a.tables_dev, b.tables_dev)
