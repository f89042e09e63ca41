"""Shared-prefix attention where a prefix is walked in tiles of more than 64 rows, row by row
against float64.

A row's error is held to half a step of the output type, eps / 2 of the element, and to what
the weights' rounding adds: at most 2^-11 of sum w |v| (fp16 weights, 2^-12 each, and the sum
that divides them), 2^-10 with the fp32 exponents and sums beside it (scores of a few tens in
log2 units at 2^-24, products of bf16 or fp16 values exact).
"""

from __future__ import annotations

import pytest
import torch

from engine.attention import SharedPrefix, gather_ctx, shared_prefix_attention
from engine.kv import PagedKVCache

pytestmark = pytest.mark.gpu

F32, BF16, F16, FP8 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn


def cache(cuda, contexts, dtype):
    """A cache whose sequence s holds contexts[s], a pair (1, n, kv heads, d) of keys and values."""
    hkv, d = contexts[0][0].shape[2:]
    lens = [int(k.shape[1]) for k, _ in contexts]
    kv = PagedKVCache(1, hkv, d, sum(-(-n // 16) for n in lens) + 3, 16, cuda, dtype, max_seqs=len(lens))
    kv.add_sequence(len(lens) - 1)
    for s, (k, v) in enumerate(contexts):
        put = [x.to(BF16 if kv.fp8 else dtype).to(cuda) for x in (k, v)]
        kv.write_block(0, [s], [0], *put)
    return kv


def exact(q, kv, starts, ids, lens):
    """The attention of entry b over its prefix and its own sequence b in float64, and sum w |v|."""
    B, C, hq, d = q.shape
    q, out = q.double(), []
    contexts = {}
    for b in range(B):
        n = starts[b] + C
        parts = [gather_ctx(kv, 0, b, n).double()]
        if ids[b] >= 0 and lens[b]:
            at = (ids[b], lens[b])
            if at not in contexts:
                contexts[at] = gather_ctx(kv, 0, *at).double()
            parts.insert(0, contexts[at])
        k, v = torch.cat(parts, 1).permute(0, 2, 1, 3).contiguous()  # (kv heads, positions, d)
        hkv, total = k.shape[:2]
        each = []
        for j in range(C):  # only what the row sees, so that an infinity behind it meets no weight of 0
            at, rows = total - C + j + 1, q[b, j].view(hkv, hq // hkv, d)
            w = torch.softmax(torch.matmul(rows, k[:, :at].transpose(1, 2).contiguous()) * d ** -0.5, -1)
            each.append([torch.matmul(w, x[:, :at].contiguous()).view(hq, d) for x in (v, v.abs())])
        out.append([torch.stack(x) for x in zip(*each)])
    return [torch.stack(x) for x in zip(*out)]


def near(out, want, size, dtype):
    err = (out - want).abs()
    bound = torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -10 if dtype != F32 else 2.0 ** -17) * size
    worst = float((err / bound.clamp(min=1e-300)).max())
    assert worst <= 1, worst


def close(out, want, size):
    """Every finite element, by the bound above; infinities and NaN where they belong."""
    dtype, out = out.dtype, out.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out[~fine].nan_to_num(), want[~fine].nan_to_num())
    near(out[fine], want[fine], size[fine], dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("B", [2, 20])
@pytest.mark.parametrize("where", ["prefix", "own", "chunk"])
def test_infinite_values_that_are_seen(cuda, dtype, d, B, where):
    """An infinite value reaches its dimension of the rows that see it, with its sign, and no other;
    infinities of both signs give NaN there. Tiles of few rows, of more than 64, and own keys."""
    g = torch.Generator().manual_seed(73)
    C, hq, hkv, P = 4, 8, 2, 150
    parts = [[torch.randn(1, n, hkv, d, generator=g) for _ in range(2)] for n in [30 + C] * B + [P]]
    inf = float("inf")
    v, at = (parts[B][1], 70) if where == "prefix" else (parts[1][1], 3 if where == "own" else 30 + 2)
    v[0, at, 0, 7], v[0, at, 1, 20] = inf, -inf
    v[0, at - 2, 1, 33], v[0, at, 1, 33] = inf, -inf
    kv = cache(cuda, parts, dtype)
    q = torch.randn(B, C, hq, d, generator=g).to(dtype).to(cuda)
    ids, lens = [B] * B, [P] * B
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [30] * B, 30 + C, SharedPrefix(kv, ids, lens, C, hq))
    want, size = exact(q, kv, [30] * B, ids, lens)
    assert bool(torch.isposinf(want).any()) and bool(torch.isneginf(want).any()) and bool(torch.isnan(want).any())
    close(out, want, size)
