"""Attention over the cache with head scales, on the GPU: value scales that fall and rise along a
context, weights far below a row's largest, and every way its work is shared out.

The tolerance is that of ``test_gpu_head_scales``: an element is off by half a step of its type, and
by eps_p sum_i p_i |v_i| for the weights, whatever part of a row's output they make up.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from engine.attention import verify_attention
from engine.kv import PagedKVCache
from oracle.kv_fp8 import e4m3_decode

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LN2 = math.log(2.0)


def _cache(cuda, lens, H, d, seed, bs=16):
    """Contexts of random finite codes in shuffled blocks, K scales that give scores of about 1, V scales near 2^-5."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    nb = [-(-n // bs) for n in lens]
    cap = sum(nb) + 3
    perm = torch.randperm(cap, generator=torch.Generator().manual_seed(seed)).tolist()
    tables, at = [], 0
    for n in nb:
        tables.append(perm[at:at + n])
        at += n
    kv = PagedKVCache(1, H, d, cap, bs, cuda, FP8, max_seqs=len(lens), max_blocks_per_seq=max(nb), head_scales=True)
    kv.load_state(tables, lens, perm[at:])
    for pool in (kv.k_pool, kv.v_pool):
        codes = torch.randint(0, 256, tuple(pool.shape), generator=g, device=cuda, dtype=torch.uint8)
        pool.view(torch.uint8).copy_(torch.where((codes & 0x7F) == 0x7F, codes - 1, codes))
    kv.scales.copy_(torch.rand(tuple(kv.scales.shape), generator=g, device=cuda) * 0.02 + 0.02)
    return kv, g, tables


def _check(out, q, kv, tables, picked, starts, scale=None, rows=None):
    """The picked entries' rows against float64 over the stored codes, within the tolerance above."""
    B, C, hq, d = q.shape
    H, bs = kv.num_kv_heads, kv.block_size
    scale = d ** -0.5 if scale is None else scale
    half = torch.finfo(q.dtype).eps / 2
    tiny = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[q.dtype]
    values = torch.from_numpy(np.asarray(e4m3_decode(np.arange(256, dtype=np.uint8)), dtype=np.float64)).to(kv.device)
    for b in picked:
        n = starts[b] + C
        at = torch.tensor(tables[b][:-(-n // bs)], device=kv.device)
        s = kv.scales[0][:, at].double()[..., None, None]  # (H, blocks, K | V, 1, 1)
        k = values[kv.k_pool[0].view(torch.uint8)[at].long()].transpose(0, 1) * s[:, :, 0]
        v = values[kv.v_pool[0].view(torch.uint8)[at].long()].permute(1, 0, 3, 2) * s[:, :, 1]
        k, v = (x.reshape(H, -1, d)[:, :n].contiguous() for x in (k, v))
        kt = k.transpose(1, 2).contiguous()
        j = torch.tensor(range(C) if rows is None else rows, device=kv.device)
        qq = q[b, j].double().view(len(j), H, hq // H, d).transpose(0, 1).reshape(H, -1, d)
        seen = (starts[b] + j + 1).repeat_interleave(hq // H)[None, :, None]
        masked = torch.arange(n, device=kv.device) >= seen
        z = torch.matmul(qq, kt) * scale
        size = (torch.matmul(qq.abs(), kt.abs()) * abs(scale)).masked_fill(masked, 0.0).amax(-1, keepdim=True)
        p = torch.softmax(z.masked_fill(masked, -math.inf), -1)
        o, a = torch.matmul(p, v), torch.matmul(p, v.abs())
        eps_p = 2 * (d + 4) * 2.0 ** -24 * size + 2.0 ** -20 + (2.0 ** -11 if q.dtype is BF16 else 2.0 ** -17)
        bound = half * o.abs() + tiny / 2 + (1 + half) * eps_p * a
        got = out[b, j].double().view(len(j), H, hq // H, d).transpose(0, 1).reshape(H, -1, d)
        worst = float(((got - o).abs() / bound).max())
        assert worst <= 1.0, (b, worst)


def _set_blocks(kv, tables, n_blocks, k_level, v_exp):
    """Logical block i of every sequence: keys +-1 in dimension 0 alone, times a scale that makes q = e_0's score
    ``k_level(i)``; the values' scale 2^v_exp(i), codes as they are."""
    k8 = kv.k_pool.view(torch.uint8)
    k8.zero_()
    level = torch.tensor([float(k_level(i)) for i in range(n_blocks)])
    exp = torch.tensor([float(v_exp(i)) for i in range(n_blocks)])
    sign = torch.where(level < 0, 0xB8, 0x38).to(torch.uint8).to(kv.device)  # -1, 1
    level, size = level.abs().to(kv.device), torch.exp2(exp.double()).float().to(kv.device)
    for row in torch.tensor([t[:n_blocks] for t in tables]).to(kv.device):
        k8[0, row, :, :, 0] = sign[:, None, None]
        kv.scales[0, :, row, 0] = level
        kv.scales[0, :, row, 1] = size


def _unit_queries(B, C, hq, d, g, cuda):
    """Queries of 1 in dimension 0 (the keys have no other), anything elsewhere."""
    q = torch.randn(B, C, hq, d, generator=g, device=cuda)
    q[..., 0] = 1.0
    return q


@pytest.mark.parametrize("dtype", [BF16, F32, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("first", ["small", "large"])
@pytest.mark.parametrize("ratio,weight", [(40, 30.5), (60, 45.3), (30, 27.4), (16, 20.6), (12, 24.5)])
def test_small_weights_on_large_values(cuda, dtype, d, first, ratio, weight):
    """Half of a row's keys have weights 2^-weight of the others' and values 2^ratio of theirs: what such keys add
    keeps its bits, whether they make up most of the output or a part that its rounding hides."""
    if dtype == F16:  # outputs within the type
        ratio, weight = min(ratio, 14), min(weight, 20.6)
    B, C, hq, n = 140, 2, 8, 1344
    kv, g, tables = _cache(cuda, [n] * B, 2, d, 21)
    large = lambda i: (32 <= i < 64) == (first == "small")  # noqa: E731  eight steps of four blocks in turn
    _set_blocks(kv, tables, n // 16, lambda i: -weight * LN2 if large(i) else 0.0, lambda i: -8 + ratio * large(i))
    q = _unit_queries(B, C, hq, d, g, cuda).to(dtype)
    starts = [n - C - 5 * (b % 3) for b in range(B)]
    out = verify_attention(q, kv, 0, list(range(B)), starts, n, scale=1.0)
    pick = list(range(0, B, 23))
    _check(out, q, kv, tables, pick, starts, scale=1.0)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("balanced", [False, True])
@pytest.mark.parametrize("exps", [
    [0, -1, -2, -3, -4], [0, 1, 2, 3, 4], [0, -15, 0, -15, -14], [0, -16, 0, -16, -1], [0, 7, 7, -8, 0],
    [0, 8, 0, 8, -7], [-15, 0, 7, 8, 15], [15, 8, 7, 0, -15], [0, -9, -12, -13, 3], [0, 12, 13, 1, -4],
    [0, 6, -5, 5, 1], [0, 0, 7, 0, 0], [0, -6, 0, -6, 0], [5, -1, 5, 11, 0],
], ids=str)
def test_value_scales_of_near_powers(cuda, dtype, d, balanced, exps):
    """Block scales of powers of two that differ from one turn of a wave (8 steps) to the next, and by one between the
    blocks of a step; codes of the smallest subnormal, of 448 and of every size. ``balanced``: weights 2^-exps, so
    that every block counts in the output."""
    B, C, hq, n = 70, 3, 8, 2560
    if dtype == F16:
        exps = [min(e, 4) for e in exps]
    kv, g, tables = _cache(cuda, [n] * B, 2, d, 22)
    v_exp = lambda i: exps[i // 32 % len(exps)] - (i % 4 == 2) - 3  # noqa: E731
    _set_blocks(kv, tables, n // 16, lambda i: -v_exp(i) * LN2 if balanced else math.sin(i), v_exp)
    v8 = kv.v_pool.view(torch.uint8)
    v8[0, :, :, 0], v8[0, :, :, 1], v8[0, :, :, 2] = 0x01, 0x7E, 0x87
    q = _unit_queries(B, C, hq, d, g, cuda).to(dtype)
    starts = [n - C - 11 * (b % 5) for b in range(B)]
    out = verify_attention(q, kv, 0, list(range(B)), starts, n, scale=1.0)
    pick = [0, 13, 26, 44, 69]
    _check(out, q, kv, tables, pick, starts, scale=1.0, rows=[0, C - 1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_long_sequences_among_many_short_ones(cuda, dtype, d):
    """Equal shares of all steps, where two sequences take eight shares and more each."""
    B, C, hq = 200, 2, 8
    starts = [(i * 7) % 19 for i in range(B)]
    starts[3], starts[150] = 20011, 23456
    kv, g, tables = _cache(cuda, [s + C for s in starts], 2, d, 23)
    q = torch.randn(B, C, hq, d, generator=g, device=cuda).to(dtype)
    call = lambda: verify_attention(q, kv, 0, list(range(B)), starts, max(starts) + C)  # noqa: E731
    out = call()
    pick = [0, 2, 3, 4, 5, 75, 148, 149, 150, 151, 152, 199]
    _check(out, q, kv, tables, pick, starts)
    assert torch.equal(call(), out)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d,C,hq", [(64, 24, 8), (128, 17, 12), (64, 33, 14)])
def test_row_groups_in_equal_shares(cuda, dtype, d, C, hq):
    """Three row groups and more of each kv head, and more segments than half the workgroups."""
    B = 44
    starts = [(i * 331) % 3001 for i in range(B)]
    kv, g, tables = _cache(cuda, [s + C for s in starts], 2, d, 24)
    q = torch.randn(B, C, hq, d, generator=g, device=cuda).to(dtype)
    call = lambda: verify_attention(q, kv, 0, list(range(B)), starts, max(starts) + C)  # noqa: E731
    out = call()
    pick = [0, 1, 8, 9, 10, 30, 43]
    _check(out, q, kv, tables, pick, starts, rows=sorted({0, 7, 8, 15, 16, C - 1}))
    assert torch.equal(call(), out)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_thousands_of_sequences(cuda, dtype):
    """More than 64 entries for each lane that looks a share's segment up."""
    B, hq = 4200, 4
    starts = [(i * 5) % 16 for i in range(B)]
    starts[4150] = 3000
    kv, g, tables = _cache(cuda, [s + 1 for s in starts], 2, 64, 25)
    q = torch.randn(B, 1, hq, 64, generator=g, device=cuda).to(dtype)
    call = lambda: verify_attention(q, kv, 0, list(range(B)), starts, max(starts) + 1)  # noqa: E731
    out = call()
    pick = sorted({0, 1, 63, 64, 65, 66, 67, 131, 132, 2111, 4149, 4150, 4151, 4199, *range(100, 4200, 177)})
    _check(out, q, kv, tables, pick, starts)
    assert torch.equal(call(), out)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [2016, 2017, 2048])
def test_the_widest_heads(cuda, dtype, d):
    starts, C = [40, 3], 3
    kv, g, tables = _cache(cuda, [s + C for s in starts], 1, d, 26)
    q = torch.randn(2, C, 2, d, generator=g, device=cuda).to(dtype)
    out = verify_attention(q, kv, 0, [0, 1], starts, 43)
    _check(out, q, kv, tables, [0, 1], starts)
