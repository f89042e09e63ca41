"""Head norms with the rotation, dense and on the way into the cache, against float64.

Tolerance of an element y of the pair (a, b) of the normed row: half a step of the
output type (in the subnormals half their spacing), the rotation's 1e-6 factor
(|a| + |b|) (tests/test_gpu_rotary.py), and the norm's fp32 arithmetic, relative to
the normed value: a sum of squares of at most 20 additions one after another (16
elements of a thread and 6 steps between threads, or d / 64 and 6), halved by the
square root, the division by d, eps, the root, its reciprocal and two products: at
most 16 steps of 2^-24, 1e-6. Together 2e-6 of |a| + |b|.
"""

from __future__ import annotations

import pytest
import torch

from engine.attention import verify_attention
from engine.kv import PagedKVCache, WritePlan
from engine.rotary import HeadNorm, Rotary, rotary_append, rotary_embed
from test_gpu_rotary import BF16, F16, F32, _rows, _turned

pytestmark = pytest.mark.gpu

SPACING = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


def _normed(x, w, eps):
    x = x.detach().cpu().double()
    y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    return y if w is None else y * w.detach().cpu().double()


def _want(x, w, eps, pos, rot):
    y, size = _turned(_normed(x, w, eps), pos, rot)
    size[..., rot.rotary_dim:] = y[..., rot.rotary_dim:].abs()
    return y, size


def _close(got, want, size):
    err = (got.detach().cpu().double() - want).abs()
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() + SPACING[got.dtype] / 2 + 2e-6 * size
    assert bool((err <= bound).all()), float((err - bound).max())


def _norm(g, d, dev, eps=1e-6, dtype=F32):
    wq, wk = (1.0 + 0.5 * torch.randn(2, d, generator=g)).to(dtype).to(dev)
    return HeadNorm(d, dev, wq, wk, eps), wq, wk


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
    (1, 3, 2, 1, 7, 0, "dense"),           # normed alone
    (2, 3, 2, 1, 64, 0, "packed"),
    (1, 5, 2, 1, 256, 256, "packed"),
    (1, 3, 2, 1, 1024, 1024, "dense"),     # a wave per row and more
    (1, 2, 1, 1, 2056, 8, "dense"),        # more pieces than a wave's threads
])
def test_embed(cuda, dtype, interleaved, B, C, hq, hkv, d, R, layout):
    g = torch.Generator().manual_seed(B * 1000 + C * 10 + d)
    rot = Rotary(d, cuda, rotary_dim=R, interleaved=interleaved)
    norm, wq, wk = _norm(g, d, cuda, eps=1e-5)
    q, k, _ = _rows(g, B, C, hq, hkv, d, dtype, layout, cuda)
    pos = torch.randint(0, 5000, (B, C), generator=g).to(torch.int32).to(cuda)
    qo, ko = rotary_embed(q, k, rot, pos, norm=norm)
    assert qo.dtype == ko.dtype == dtype
    for x, w, y in ((q, wq, qo), (k, wk, ko)):
        _close(y, *_want(x, w, 1e-5, pos, rot))
    q_only, none = rotary_embed(q, None, rot, pos, norm=norm)
    assert none is None and torch.equal(q_only, qo)
    if layout == "packed":  # in place, in the projection's own output
        qi, ki = rotary_embed(q, k, rot, pos, query_out=q, key_out=k, norm=norm)
        assert qi is q and ki is k and torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights_eps_and_unrounded_keys(cuda, dtype):
    g = torch.Generator().manual_seed(3)
    rot = Rotary(64, cuda, sections=(8, 12, 12))
    q, k, _ = _rows(g, 2, 19, 4, 2, 64, dtype, "packed", cuda)
    pos = torch.randint(0, 900, (3, 2, 19), generator=g).to(cuda)
    _, wq, wk = _norm(g, 64, cuda)
    for a, b, eps in ((None, None, 1e-6), (wq, None, 0.0), (None, wk, 0.5), (wq.half(), wk.to(BF16), 1e-6)):
        norm = HeadNorm(64, cuda, a, b, eps=eps)
        qo, ko = rotary_embed(q, k, rot, pos, key_dtype=F32, norm=norm)
        _close(qo, *_want(q, a, eps, pos, rot))
        assert ko.dtype == F32
        _close(ko, *_want(k, b, eps, pos, rot))
    norm = HeadNorm(64, cuda, wq, wk)
    kept = norm.query_weight.clone()
    wq.zero_()  # the caller's tensor is not the norm's
    assert torch.equal(norm.query_weight, kept)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 24])
def test_small_large_and_bad_rows(cuda, dtype, d):
    """Rows of zeros stay zeros, rows of any size come to the same size, and what is not
    finite stays within its row."""
    g = torch.Generator().manual_seed(4)
    rot = Rotary(d, cuda)
    norm, wq, wk = _norm(g, d, cuda)
    x = torch.randn(1, 6, 3, d, generator=g)
    x[0, 0] = 0.0
    x[0, 1] *= 1e-3
    x[0, 2] *= 1e15
    bad = x.clone()
    bad[0, 3, 1, 5], bad[0, 4, 2, 0] = float("nan"), float("inf")
    x, bad = x.to(dtype).to(cuda), bad.to(dtype).to(cuda)
    pos = torch.arange(6, dtype=torch.int32, device=cuda)[None]
    qo, ko = rotary_embed(x, x, rot, pos, norm=norm)
    _close(qo, *_want(x, wq, 1e-6, pos, rot))
    _close(ko, *_want(x, wk, 1e-6, pos, rot))
    assert not qo[0, 0].any()
    qb, kb = rotary_embed(bad, bad, rot, pos, norm=norm)
    for y, yb in ((qo, qb), (ko, kb)):
        assert yb[0, 3, 1].isnan().all() and yb[0, 4, 2].isnan().any()
        keep = torch.ones(6, 3, dtype=torch.bool)
        keep[3, 1] = keep[4, 2] = False
        assert torch.equal(y[0][keep], yb[0][keep])


def _filled(cuda, lens, Hkv, d, bs, dtype, layers, seed, **kw):
    kv = PagedKVCache(layers, Hkv, d, sum(-(-n // bs) for n in lens) + 4 * len(lens) + 3, bs, cuda, dtype, **kw)
    g = torch.Generator().manual_seed(seed)
    fp8 = dtype.itemsize == 1
    for s, n in enumerate(lens):
        kv.add_sequence(s)
        for layer in range(layers):
            if n:
                k, v = (torch.randn(1, n, Hkv, d, generator=g).to(F32 if fp8 else dtype).to(cuda) for _ in range(2))
                kv.write_block(layer, [s], [0], k, v)
    return kv


@pytest.mark.parametrize("dtype,d,R", [(F32, 64, 64), (BF16, 128, 64), (F16, 64, 64), (BF16, 10, 6)])
@pytest.mark.parametrize("C", [1, 6, 37])
def test_append(cuda, dtype, d, R, C):
    """The normed append leaves the pools of ``write_block_device`` of the normed and rotated
    keys, the first layer and those that follow its plan."""
    g = torch.Generator().manual_seed(d + C)
    lens, hq, hkv, bs, layers = [5, 0, 31], 4, 2, 16, 3
    rot = Rotary(d, cuda, rotary_dim=R)
    norm, _, _ = _norm(g, d, cuda)
    a, b = (_filled(cuda, lens, hkv, d, bs, dtype, layers, 1) for _ in range(2))
    sid, start = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([2, 0, 1], [31, 5, 0]))
    pos = start[:, None] + torch.arange(C, dtype=torch.int32, device=cuda)
    plan, other = WritePlan(), WritePlan()
    for layer in range(layers):
        q, k, v = _rows(g, 3, C, hq, hkv, d, dtype, "packed", cuda)
        qo = rotary_append(q, k, v, a, layer, sid, start, rot, alloc=layer == 0, plan=plan, norm=norm)
        qe, ke = rotary_embed(q, k, rot, pos, norm=norm)
        b.write_block_device(layer, sid, start, ke, v.contiguous(), alloc=layer == 0, plan=other)
        assert torch.equal(qo, qe)
    assert a.block_tables == b.block_tables and a.seq_lengths == b.seq_lengths
    assert torch.equal(a.k_pool, b.k_pool) and torch.equal(a.v_pool, b.v_pool)


def test_append_into_an_fp8_pool_of_one_scale(cuda):
    g = torch.Generator().manual_seed(9)
    rot = Rotary(64, cuda)
    norm, _, _ = _norm(g, 64, cuda)
    a, b = (_filled(cuda, [20], 2, 64, 16, torch.float8_e4m3fn, 1, 2) for _ in range(2))
    sid, start = (torch.tensor([x], dtype=torch.int32, device=cuda) for x in (0, 20))
    q, k, v = _rows(g, 1, 5, 4, 2, 64, BF16, "packed", cuda)
    qo = rotary_append(q, k, v, a, 0, sid, start, rot, norm=norm)
    pos = start[:, None] + torch.arange(5, dtype=torch.int32, device=cuda)
    qe, ke = rotary_embed(q, k, rot, pos, norm=norm, key_dtype=F32)
    b.write_block_device(0, sid, start, ke, v.float())
    assert torch.equal(qo, qe) and torch.equal(a.scales, b.scales)
    assert torch.equal(a.k_pool.view(torch.uint8), b.k_pool.view(torch.uint8))


def test_captured_and_on_another_stream(cuda):
    g = torch.Generator().manual_seed(11)
    rot = Rotary(64, cuda)
    norm, _, _ = _norm(g, 64, cuda)
    kv = _filled(cuda, [40, 7], 2, 64, 16, BF16, 1, 5)
    sid, start = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, 1], [40, 7]))
    q, k, v = (t.contiguous() for t in _rows(g, 2, 3, 4, 2, 64, BF16, "packed", cuda))
    kv.write_block_device(0, sid, start, k, v)

    def step():
        qo = rotary_append(q, k, v, kv, 0, sid, start, rot, alloc=False, norm=norm)
        return verify_attention(qo, kv, 0, sid, start, 43)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=g).to(BF16))
        k.copy_(torch.randn(k.shape, generator=g).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())
