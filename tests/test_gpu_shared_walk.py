"""Shared-prefix attention where a prefix is walked in tiles of more than 64 rows, row by row
against float64.

A row's error is held to half a step of the output type, eps / 2 of the element, and to what
the weights' rounding adds: at most 2^-11 of sum w |v| (fp16 weights, 2^-12 each, and the sum
that divides them), 2^-10 with the fp32 exponents and sums beside it (scores of a few tens in
log2 units at 2^-24, products of bf16 or fp16 values exact). In fp32 a score of 8 log2 units,
the sum of some hundred products of 2^-24 each, is off by about 2^-19 at most: 2^-17 of sum w |v|.
Plans are cut by hand where a test needs long segments.
"""

from __future__ import annotations

import pytest
import torch

from engine.attention import SharedPrefix, gather_ctx, shared_prefix_attention
from engine.kv import PagedKVCache
from shared_plans import recut

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


def exact(q, kv, starts, ids, lens, own=None):
    """The attention of entry b over its prefix and its own sequence (b, or own[b]) in float64, and
    sum w |v|."""
    B, C, hq, d = q.shape
    q, out = q.double(), []
    contexts = {}

    def context(sid, n):
        if (sid, n) not in contexts:
            contexts[sid, n] = gather_ctx(kv, 0, sid, n).double()
        return contexts[sid, n]

    for b in range(B):
        parts = [context(b if own is None else own[b], starts[b] + C)]
        if ids[b] >= 0 and lens[b]:
            parts.insert(0, context(ids[b], lens[b]))
        k, v = torch.cat(parts, 1).permute(0, 2, 1, 3).contiguous()  # (kv heads, positions, d)
        hkv, total = k.shape[:2]
        each = []
        for j in range(C):  # only what the row sees, so that an infinity behind it meets no weight of 0
            at, rows = total - C + j + 1, q[b, j].view(hkv, hq // hkv, d)
            w = torch.softmax(torch.matmul(rows, k[:, :at].transpose(1, 2).contiguous()) * d ** -0.5, -1)
            each.append([torch.matmul(w, x[:, :at].contiguous()).view(hq, d) for x in (v, v.abs())])
        out.append([torch.stack(x) for x in zip(*each)])
    return [torch.stack(x) for x in zip(*out)]


def near(out, want, size, dtype, fp32, half):
    err = (out - want).abs()
    bound = torch.finfo(dtype).eps / 2 * want.abs() + (half if dtype != F32 else fp32) * size
    worst = float((err / bound.clamp(min=1e-300)).max())
    assert worst <= 1, worst


def close(out, want, size, fp32=2.0 ** -17, half=2.0 ** -10):
    """Every finite element, by the bound above; infinities and NaN where they belong."""
    dtype, out = out.dtype, out.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out[~fine].nan_to_num(), want[~fine].nan_to_num())
    near(out[fine], want[fine], size[fine], dtype, fp32, half)


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


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,C,hq", [(4, 1, 14), (2, 7, 8), (30, 3, 16)])
def test_fp16_weights_keep_their_bits(cuda, d, B, C, hq):
    """Few rows behind a prefix, and own keys alone: the output's rounding and what fp32 arithmetic
    adds, no more (P in one fp16 would add up to 2^-12 of every weight)."""
    g = torch.Generator().manual_seed(97)
    hkv, P = 2, 600
    parts = [[torch.randn(1, n, hkv, d, generator=g) for _ in range(2)] for n in [200 + C] * B + [P]]
    kv = cache(cuda, parts, F16)
    q = torch.randn(B, C, hq, d, generator=g).half().to(cuda)
    few = B * C * hq // hkv <= 64
    ids, lens = [B if few else -1] * B, [P if few else 0] * B
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [200] * B, 200 + C, SharedPrefix(kv, ids, lens, C, hq))
    close(out, *exact(q, kv, [200] * B, ids, lens), half=2.0 ** -17)


@pytest.mark.parametrize("dtype", [BF16, F16, F32, FP8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("first", [1.0, 0.0, 2.0 ** -14])
@pytest.mark.parametrize("later", [1.0, 2.0 ** 5, 2.0 ** 10, 2.0 ** 40])
def test_values_of_other_sizes_behind_the_first_tile(cuda, dtype, d, first, later):
    """The first 64 keys' values scaled by ``first``, a page's behind them by ``later``, in one segment
    of eight units: whether or not a tile's staging holds both."""
    if dtype == F16 and later > 2.0 ** 10:
        pytest.skip("past the type")
    g = torch.Generator().manual_seed(79)
    B, C, hq, hkv, P = 8, 5, 8, 2, 500
    parts = [[torch.randn(1, n, hkv, d, generator=g) for _ in range(2)] for n in [9 + C] * B + [P]]
    parts[B][1][:, :64] *= first
    parts[B][1][:, 208:224] *= later
    kv = cache(cuda, parts, dtype)
    q = torch.randn(B, C, hq, d, generator=g).to(BF16 if dtype == FP8 else dtype).to(cuda)
    ids, lens = [B] * B, [P] * B
    prefix = SharedPrefix(kv, ids, lens, C, hq)
    segs = recut(prefix, ids, lens, lambda units: units)
    assert len(segs) == hkv and all(s[5] == B * C * hq // hkv > 64 and s[7] - s[6] == P for s in segs)
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [9] * B, 9 + C, prefix)
    close(out, *exact(q, kv, [9] * B, ids, lens))


@pytest.mark.parametrize("dtype", [BF16, F16, F32, FP8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("slope", [-60.0, 60.0])
def test_scores_that_rise_or_fall_along_a_segment(cuda, dtype, d, slope):
    """The reference maximum grows in every tile of a segment, or in none behind the first. (fp32
    scores of up to 90 log2 units are off by 2^-15.)"""
    g = torch.Generator().manual_seed(83)
    B, C, hq, hkv, P = 8, 5, 8, 2, 700
    u = torch.randn(d, generator=g)
    u = u / u.norm() * d ** 0.25
    parts = [[torch.randn(1, n, hkv, d, generator=g) for _ in range(2)] for n in [9 + C] * B + [P]]
    parts[B][0].add_((slope * torch.arange(P) / P)[None, :, None, None] * u)
    kv = cache(cuda, parts, dtype)
    q = (0.5 * torch.randn(B, C, hq, d, generator=g) + u).to(BF16 if dtype == FP8 else dtype).to(cuda)
    ids, lens = [B] * B, [P] * B
    prefix = SharedPrefix(kv, ids, lens, C, hq)
    recut(prefix, ids, lens, lambda units: units)
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [9] * B, 9 + C, prefix)
    close(out, *exact(q, kv, [9] * B, ids, lens), fp32=2.0 ** -14)


@pytest.mark.parametrize("dtype", [BF16, F16, FP8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("P", [65, 129, 1024, 1088, 1090, 2049, 2100, 2500, 4200])
def test_long_segments(cuda, dtype, d, P):
    """Segments of 2 to 66 units of 64 keys, their last one whole or not, by tiles of more than 64
    rows: page numbers and scales change hands every 16 units, values go round three slots."""
    g = torch.Generator().manual_seed(P)
    B, C, hq, hkv = 9, 4, 8, 1
    parts = [[torch.randn(1, n, hkv, d, generator=g) for _ in range(2)] for n in [3 + C] * B + [P]]
    if dtype == FP8:  # each page with scales of its own
        for x in parts[B]:
            x.mul_((2.0 ** torch.randint(-3, 1, (-(-P // 16),), generator=g)).repeat_interleave(16)[:P].view(1, P, 1, 1))
    kv = cache(cuda, parts, dtype)
    q = torch.randn(B, C, hq, d, generator=g).to(BF16 if dtype == FP8 else dtype).to(cuda)
    ids, lens = [B] * B, [P] * B
    want = exact(q, kv, [3] * B, ids, lens)
    for units in (lambda n: n, lambda n: (n + 1) // 2):
        prefix = SharedPrefix(kv, ids, lens, C, hq)
        segs = recut(prefix, ids, lens, units)
        assert max(s[7] - s[6] for s in segs) == min(P, units(-(-P // 64)) * 64) and max(s[5] for s in segs) == 256
        out = shared_prefix_attention(q, kv, 0, list(range(B)), [3] * B, 3 + C, prefix)
        close(out, *want)


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("P", [70, 1500, 2100])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, FP8])
def test_tiles_of_every_size(cuda, dtype, tile, d, P):
    """fp32 walks page by page in tiles of up to 256 rows (few waves then share them); the 16-bit
    types may be given any of them by a plan, too."""
    g = torch.Generator().manual_seed(P + tile)
    B, C, hq, hkv = 10, 5, 12, 2  # 300 rows
    parts = [[torch.randn(1, n, hkv, d, generator=g) for _ in range(2)] for n in [3 + C] * B + [P]]
    kv = cache(cuda, parts, dtype)
    q = torch.randn(B, C, hq, d, generator=g).to(BF16 if dtype == FP8 else dtype).to(cuda)
    ids, lens = [B] * B, [P] * B
    prefix = SharedPrefix(kv, ids, lens, C, hq)
    segs = recut(prefix, ids, lens, lambda n: n, tile)
    assert max(s[5] for s in segs) == tile
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [3] * B, 3 + C, prefix)
    close(out, *exact(q, kv, [3] * B, ids, lens))


@pytest.mark.parametrize("dtype", [F32, BF16, F16, FP8])
@pytest.mark.parametrize("C,n", [(2, 9000), (10, 4500)])
def test_long_own_contexts_in_one_range(cuda, dtype, C, n):
    """Own contexts of more pages than a wave's lanes hold the numbers of (64 pages for each of
    8 waves up to 32 rows, of 4 up to 64): more entries than CUs leave one range each."""
    g = torch.Generator().manual_seed(n)
    B, hq, hkv, d, P = 150, 8, 2, 64, 40
    parts = [[torch.randn(1, m, hkv, d, generator=g) for _ in range(2)] for m in (n, P)]
    kv = cache(cuda, parts, dtype)
    q = torch.randn(B, C, hq, d, generator=g).to(BF16 if dtype == FP8 else dtype).to(cuda)
    starts = [n - C - 7 * b for b in range(B)]
    out = shared_prefix_attention(q, kv, 0, [0] * B, starts, n, SharedPrefix(kv, [1] * B, [P] * B, C, hq))
    some = [0, 1, 40, B - 1]
    pick = lambda x: [x[i] for i in some]  # noqa: E731
    close(out[some], *exact(q[some], kv, pick(starts), [1] * 4, [P] * 4, own=[0] * 4))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("margin", [0.0, 8.0, 25.0])
@pytest.mark.parametrize("power", [-3, -8, -11, -13, -16, -18, -22, -40])
def test_fp8_rows_on_pages_of_small_v_scale(cuda, d, margin, power):
    """Five pages of values 2^power times the others'; the queries' scores on their keys lie ``margin``
    (natural units) above the rest, so that from 8 on those pages hold most of a row's weight."""
    g = torch.Generator().manual_seed(71)
    B, C, hq, hkv, P = 8, 5, 8, 2, 400
    assert B * C * (hq // hkv) > 64
    u = torch.randn(d, generator=g)
    u = u / u.norm() * d ** 0.5
    k, v = (torch.randn(1, P, hkv, d, generator=g) for _ in range(2))
    k[:, 80:160] += 2 * u
    v[:, 80:160] *= 2.0 ** power
    own = [[torch.randn(1, 9 + C, hkv, d, generator=g) for _ in range(2)] for _ in range(B)]
    kv = cache(cuda, [*own, (k, v)], FP8)
    q = (torch.randn(B, C, hq, d, generator=g) + margin / 2 * d ** -0.5 * u).to(BF16).to(cuda)
    ids, lens = [B] * B, [P] * B
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [9] * B, 9 + C, SharedPrefix(kv, ids, lens, C, hq))
    close(out, *exact(q, kv, [9] * B, ids, lens))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("margin", [0.0, 8.0, 14.0, 19.0, 25.0])
@pytest.mark.parametrize("dtype,power", [(BF16, -8), (BF16, -12), (BF16, -16), (BF16, -20), (BF16, -24), (BF16, -27),
                                         (BF16, -31), (BF16, -60), (F16, -8), (F16, -12), (F32, -8), (F32, -60)])
def test_rows_on_pages_of_small_values(cuda, dtype, d, margin, power):
    """As over fp8: pages whose values are 2^power times the others', with most of a row's weight from
    a margin of 8 on, in one segment with the others."""
    g = torch.Generator().manual_seed(89)
    B, C, hq, hkv, P = 8, 5, 8, 2, 400
    u = torch.randn(d, generator=g)
    u = u / u.norm() * d ** 0.5
    k, v = (torch.randn(1, P, hkv, d, generator=g) for _ in range(2))
    k[:, 80:160] += 2 * u
    v[:, 80:160] *= 2.0 ** power
    own = [[torch.randn(1, 9 + C, hkv, d, generator=g) for _ in range(2)] for _ in range(B)]
    kv = cache(cuda, [*own, (k, v)], dtype)
    q = (torch.randn(B, C, hq, d, generator=g) + margin / 2 * d ** -0.5 * u).to(dtype).to(cuda)
    ids, lens = [B] * B, [P] * B
    prefix = SharedPrefix(kv, ids, lens, C, hq)
    segs = recut(prefix, ids, lens, lambda n: n)
    assert all(s[5] > 64 and s[7] - s[6] == P for s in segs)
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [9] * B, 9 + C, prefix)
    # fp32: scores of up to 60 log2 units
    close(out, *exact(q, kv, [9] * B, ids, lens), fp32=2.0 ** -15)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B", [1, 20])
def test_an_infinite_value_of_little_weight(cuda, dtype, d, B):
    """A weight of e^-50, nothing in fp16, still takes an infinite value to its dimension."""
    g = torch.Generator().manual_seed(101)
    C, hq, hkv, P = 4, 8, 2, 300
    u = torch.randn(d, generator=g)
    u = u / u.norm() * d ** 0.25
    parts = [[torch.randn(1, n, hkv, d, generator=g) for _ in range(2)] for n in [9 + C] * B + [P]]
    parts[B][0][:, 100:120] += 25 * u
    parts[B][0][:, 200:220] -= 25 * u
    parts[B][1][0, 210, 0, 7], parts[B][1][0, 211, 1, 9] = float("inf"), -float("inf")
    kv = cache(cuda, parts, dtype)
    q = (0.5 * torch.randn(B, C, hq, d, generator=g) + u).to(dtype).to(cuda)
    ids, lens = [B] * B, [P] * B
    prefix = SharedPrefix(kv, ids, lens, C, hq)
    recut(prefix, ids, lens, lambda units: units)
    out = shared_prefix_attention(q, kv, 0, list(range(B)), [9] * B, 9 + C, prefix)
    want, size = exact(q, kv, [9] * B, ids, lens)
    assert int(torch.isinf(want).sum()) == B * C * hq
    close(out, want, size, fp32=2.0 ** -15)


def test_rows_of_nan_queries(cuda):
    """A NaN in an entry's queries is that row's alone, and sends nothing to a slower walk's result."""
    g = torch.Generator().manual_seed(103)
    B, C, hq, hkv, d, P = 20, 4, 8, 2, 64, 300
    for dtype in (BF16, F16, F32, FP8):
        parts = [[torch.randn(1, n, hkv, d, generator=g) for _ in range(2)] for n in [9 + C] * B + [P]]
        kv = cache(cuda, parts, dtype)
        q = torch.randn(B, C, hq, d, generator=g).to(BF16 if dtype == FP8 else dtype).to(cuda)
        prefix = SharedPrefix(kv, [B] * B, [P] * B, C, hq)
        want = shared_prefix_attention(q, kv, 0, list(range(B)), [9] * B, 9 + C, prefix)
        q[3, 1, 2, 5] = float("nan")
        out = shared_prefix_attention(q, kv, 0, list(range(B)), [9] * B, 9 + C, prefix)
        assert bool(torch.isnan(out[3, 1, 2]).all())
        out[3, 1, 2] = want[3, 1, 2]
        assert torch.equal(out, want)
