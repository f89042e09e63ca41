"""CPU checks of head norms and of the cache with head scales: refusals before anything
touches a GPU, what a call passes on, and the lifetimes of a norm's weights."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from engine import _hip
from engine import attention as attention_module
from engine import kv as kv_module
from engine import rotary as rotary_module
from engine.attention import SharedPrefix, VerifyPlan, gather_ctx, verify_attention
from engine.kv import PagedKVCache
from engine.rotary import HeadNorm, Rotary, rotary_append, rotary_embed
from engine.scheduler import bytes_per_block

FP8 = torch.float8_e4m3fn
ARG, UNSUP = _hip.SPV_ERR_ARG, _hip.SPV_ERR_UNSUPPORTED
F = ctypes.c_void_p(4096)  # never dereferenced: every call below is refused


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_hip.LIB_PATH):
        pytest.fail("libspecverify.so is not built; run __graft_entry__.build()")
    return _hip.lib()


def test_append_refusals(lib):
    st = (ctypes.c_int64 * 6)()

    def go(kp=F, scales=F, dt=1, k=F, v=F, strides=st, tables=F, maxb=4, nb=F, lens=F, stack=F, flag=F, ctr=F, sid=F,
           start=F, B=1, C=1, layer=0, layers=2, cap=4, bs=16, H=2, d=64, alloc=0, limit=-1):
        return lib.spv_kv_append_fp8_heads(kp, F, scales, dt, k, v, strides, tables, maxb, nb, lens, stack, flag, ctr,
                                           sid, start, B, C, layer, layers, cap, bs, H, d, alloc, limit, None)

    for bad in (dict(kp=None), dict(scales=None), dict(dt=3), dict(k=None), dict(v=None), dict(strides=None),
                dict(tables=None), dict(maxb=0), dict(nb=None), dict(lens=None), dict(ctr=None), dict(sid=None),
                dict(start=None), dict(B=-1), dict(C=0), dict(layer=-1), dict(layer=2), dict(cap=0), dict(bs=0),
                dict(H=0), dict(H=65536), dict(d=0), dict(limit=-2), dict(limit=2), dict(alloc=1, stack=None),
                dict(alloc=1, flag=None)):
        assert go(**bad) == ARG, bad
    assert go(d=8177) == UNSUP
    assert go(B=0) == 0


def test_rotating_append_refusals(lib):
    st = (ctypes.c_int64 * 12)()

    def go(qo=F, q=F, k=F, v=F, dt=1, strides=st, normed=1, wq=F, eps=1e-6, kp=F, scales=F, maxb=4, stack=F, ctr=F,
           pos=F, inv=F, ax=F, axes=1, B=1, C=1, hq=4, H=2, d=64, R=64, inter=0, layer=0, layers=2, cap=4, bs=16,
           alloc=0):
        return lib.spv_kv_rotary_append_fp8_heads(qo, q, k, v, dt, strides, normed, wq, wq, eps, kp, F, scales, F, maxb,
                                                  F, F, stack, F, ctr, F, F, pos, inv, ax, axes, 1.0, B, C, hq, H, d, R,
                                                  inter, layer, layers, cap, bs, alloc, None)

    for bad in (dict(qo=None), dict(k=None), dict(v=None), dict(dt=3), dict(strides=None), dict(eps=-1.0),
                dict(eps=float("nan")), dict(kp=None), dict(scales=None), dict(maxb=0), dict(ctr=None), dict(inv=None),
                dict(pos=None, axes=3), dict(ax=None, axes=3), dict(axes=0), dict(C=0), dict(hq=0), dict(H=0),
                dict(R=65), dict(R=63), dict(R=-2), dict(R=66), dict(inter=2), dict(layer=2), dict(cap=0), dict(bs=0),
                dict(alloc=1, stack=None), dict(B=1 << 12, C=(1 << 11) + 1)):
        assert go(**bad) == ARG, bad
    assert go(d=5460, R=5460) == UNSUP
    assert go(B=0) == 0


def test_gather_and_attention_refusals(lib):
    def read(kp=F, scales=F, table=F, maxb=4, sid=0, n=10, layer=0, cap=4, bs=16, H=2, d=64, out=F, dt=1):
        return lib.spv_kv_gather_fp8_heads(kp, F, scales, table, maxb, sid, n, layer, cap, bs, H, d, out, dt, None)

    for bad in (dict(kp=None), dict(scales=None), dict(table=None), dict(maxb=0), dict(n=65), dict(sid=-1), dict(n=-1),
                dict(layer=-1), dict(cap=0), dict(bs=0), dict(H=0), dict(d=0), dict(out=None), dict(dt=3)):
        assert read(**bad) == ARG, bad
    assert read(n=0) == 0

    def attend(out=F, q=F, dt=1, scales=F, table=F, maxb=4, sid=F, start=F, B=1, C=2, hq=4, H=2, d=64, bs=16, layer=0,
               cap=4, ctx=64, ws=F, nbytes=1 << 40):
        return lib.spv_verify_attn_fp8_heads(out, q, dt, F, F, scales, table, maxb, sid, start, F, F, B, C, hq, H, d, bs,
                                             layer, cap, ctx, 0.125, ws, nbytes, None)

    for bad in (dict(out=None), dict(q=None), dict(dt=3), dict(scales=None), dict(table=None), dict(maxb=3),
                dict(sid=None), dict(start=None), dict(B=-1), dict(C=0), dict(hq=5), dict(hq=0), dict(H=0), dict(d=0),
                dict(bs=0), dict(layer=-1), dict(cap=0), dict(ctx=0)):
        assert attend(**bad) == ARG, bad
    assert attend(d=2049) == UNSUP
    assert attend(B=0) == 0


def test_norm_refusals(lib):
    st = (ctypes.c_int64 * 12)()

    def go(eps=1e-6, q=F, k=F, qo=F, ko=F, dt=1, kdt=1, R=64, d=64, pos=F, inv=F):
        return lib.spv_norm_rotary(qo, q, ko, k, dt, kdt, st, F, F, eps, pos, inv, F, 1, 1.0, 1, 1, 2, 1, d, R, 0, None)

    for bad in (dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(q=None, k=None), dict(qo=None),
                dict(ko=None), dict(dt=3), dict(kdt=2), dict(R=66), dict(pos=None), dict(inv=None)):
        assert go(**bad) == ARG, bad
    args = [F, F, F, F, 1, st, F, F, -1.0] + [F, F, F, 4, F, F, F, F, F, F, F, F, F, F, 1, 1.0, 1, 1, 2, 1, 64, 64, 0, 0,
                                              4, 16, 0, 0, None, None]
    assert lib.spv_kv_norm_rotary_append(*args) == ARG


@pytest.mark.parametrize("kw", [dict(head_dim=0), dict(eps=-1.0), dict(eps=float("nan")),
                                dict(query_weight=torch.ones(63)), dict(key_weight=torch.ones(2, 64)),
                                dict(key_weight=torch.ones(64, dtype=torch.int32))])
def test_norm_arguments(kw):
    with pytest.raises(ValueError):
        HeadNorm(**{"head_dim": 64, "device": torch.device("cpu"), **kw})


def test_a_norm_and_a_cache_need_a_gpu():
    with pytest.raises(_hip.HipLibraryError):
        HeadNorm(64, torch.device("cpu"))
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 8, 4, 16, "cpu", torch.float32, head_scales=True)
    with pytest.raises(_hip.HipLibraryError):
        PagedKVCache(1, 1, 8, 4, 16, "cpu", FP8, head_scales=True)


class Calls(list):
    now, capturing = 0, False

    def names(self):
        return [c[0] for c in self]


@pytest.fixture
def calls(monkeypatch):
    """Launches and streams recorded in place of being made; tensors on the CPU."""
    made = Calls()
    made.kept = []
    for module in (_hip, attention_module, kv_module, rotary_module):
        monkeypatch.setattr(module, "call", lambda name, *args: made.append((name, *args)))
    monkeypatch.setattr(_hip, "require_gpu", torch.device)
    monkeypatch.setattr(_hip, "stream_of", lambda device: made.now)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: made.now)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: made.capturing)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: made.kept.append((t.data_ptr(), stream)))
    return made


def _cache(H=2, d=8, layers=2):
    kv = PagedKVCache(layers, H, d, 6, 16, "cpu", FP8, head_scales=True)
    kv.add_sequence(0)
    kv.add_sequence(1)
    return kv


def test_a_cache_with_head_scales(calls):
    kv = _cache(H=3, layers=2)
    assert tuple(kv.scales.shape) == (2, 3, 6, 2)
    assert kv.kv_memory_bytes == 2 * 2 * 6 * 3 * 16 * 8 + 2 * 3 * 6 * 2 * 4
    per_block = bytes_per_block(2, 16, 3, 8, FP8, head_scales=True)
    assert per_block * 6 == kv.kv_memory_bytes and bytes_per_block(2, 16, 3, 8, FP8) == per_block - 8 * 2 * 2
    ids = torch.zeros(1, dtype=torch.int32)
    kv.align_device(ids, ids, ids, ids, torch.zeros(1, 4, dtype=torch.int32), ids, ids, torch.zeros(1, 4))
    name, *args = calls[-1]
    assert name == "spv_kv_draft_align" and args[7] == kv.scales.data_ptr() and args[8] == 2 * 3


def test_writes_refuse_what_they_cannot_take(calls):
    kv = _cache()
    ids = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 3, 2, 8)
    kv.write_block_device(0, ids, ids, x, x)
    assert calls[-1][0] == "spv_kv_append_fp8_heads"
    n = len(calls)
    for bad in (lambda: kv.write_block_device(0, ids, ids, x[:, :, :1], x),
                lambda: kv.write_block_device(0, ids, ids, x, x[:, :2]),
                lambda: kv.write_block_device(0, ids, ids, x.double(), x.double()),
                lambda: kv.write_block_device(0, ids, ids, x, x.half()),
                lambda: kv.write_block_device(0, ids.long(), ids, x, x),
                lambda: kv.write_block_device(0, ids, torch.zeros(2, dtype=torch.int32), x, x),
                lambda: kv.write_block(0, [0], [0], x.to(FP8), x.to(FP8))):
        with pytest.raises(ValueError):
            bad()
    for layer in (-1, 2):
        with pytest.raises(IndexError):
            kv.write_block_device(layer, ids, ids, x, x)
    kv.write_block_device(0, ids[:0], ids[:0], x[:0], x[:0])
    kv.write_block_device(0, ids, ids, x[:, :0], x[:, :0])
    assert len(calls) == n
    with pytest.raises(ValueError):
        SharedPrefix(kv, [0], [0], 1, 2)


def test_a_write_passes_views_on(calls):
    kv = _cache()
    ids = torch.zeros(1, dtype=torch.int32)
    packed = torch.zeros(1, 3, 6, 8)
    k, v = packed[:, :, 2:4], packed[:, :, 4:]
    kv.write_block_device(1, ids, ids, k, v, alloc=False)
    args = calls[-1][1:]
    assert args[4:6] == (k.data_ptr(), v.data_ptr()) and list(args[6]) == [144, 48, 8] * 2
    columns = torch.zeros(1, 3, 8, 2).transpose(2, 3)
    kv.write_block_device(1, ids, ids, columns, v, alloc=False)
    assert calls[-1][5] != columns.data_ptr() and list(calls[-1][7])[:3] == [48, 16, 8]


def test_attention_refuses_what_it_cannot_take(calls):
    kv = _cache()
    kv._lens, kv._nb = [20, 20], [2, 2]
    ids, st = torch.tensor([0, 1], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 3, 4, 8)
    n = len(calls)
    for bad in (dict(query_3d=q.double()), dict(query_3d=q[..., :4]), dict(query_3d=q[:, :, :3]), dict(max_ctx=2),
                dict(out=q), dict(out=q[:, :2]), dict(out=q.half()), dict(out=torch.zeros(2, 4, 3, 8).transpose(1, 2)),
                dict(seq_ids=[0]), dict(start_positions=st[:1])):
        with pytest.raises(ValueError):
            verify_attention(**{"query_3d": q, "kv": kv, "layer": 0, "seq_ids": ids, "start_positions": st,
                                "max_ctx": 20, **bad})
    for bad in (dict(layer=2), dict(layer=-1), dict(seq_ids=[0, 2])):
        with pytest.raises(IndexError):
            verify_attention(**{"query_3d": q, "kv": kv, "layer": 0, "seq_ids": ids, "start_positions": st,
                                "max_ctx": 20, **bad})
    plan = VerifyPlan(kv, ids, st, 3, 4, 20)
    assert plan.buf is None and len(calls) == n
    with pytest.raises(ValueError):
        verify_attention(q, kv, 0, ids, st, 21, plan=plan)
    assert verify_attention(q[:, :0], kv, 0, ids, st, 20).shape == (2, 0, 4, 8)
    for layer in (-1, 2):
        with pytest.raises(IndexError):
            gather_ctx(kv, layer, 0, 20)
    with pytest.raises(ValueError):
        gather_ctx(kv, 0, 0, 20, dtype=FP8)
    assert len(calls) == n


def test_a_norm_belongs_to_its_heads(calls):
    rot, kv = Rotary(8, "cpu"), _cache()
    q, pos = torch.zeros(1, 3, 2, 8), torch.zeros(1, 3, dtype=torch.int32)
    wrong = HeadNorm(16, "cpu")
    ids = torch.zeros(1, dtype=torch.int32)
    del calls[:]
    for bad in (lambda: rotary_embed(q, q, rot, pos, norm=wrong),
                lambda: rotary_append(q, q, q, kv, 0, ids, ids, rot, norm=wrong)):
        with pytest.raises(ValueError):
            bad()
    assert not calls


def test_a_norms_weights_are_copies_and_are_kept(calls):
    """What a dropped norm holds stays until the other streams given it are done; a captured graph's
    owner keeps it by itself."""
    w = torch.ones(16)[::2]
    rot, norm, kv = Rotary(8, "cpu"), HeadNorm(8, "cpu", w, w.half()), _cache()
    assert norm.query_weight.data_ptr() != w.data_ptr() and norm.key_weight.dtype == torch.float32
    q, pos = torch.zeros(1, 3, 2, 8), torch.zeros(1, 3, dtype=torch.int32)
    ids = torch.zeros(1, dtype=torch.int32)
    del calls[:]
    held = {norm.query_weight.data_ptr(), norm.key_weight.data_ptr()}
    for go in (lambda: rotary_embed(q, q, rot, pos, norm=norm),
               lambda: rotary_append(q, q, q, kv, 0, ids, ids, rot, norm=norm)):
        calls.now, calls.capturing, calls.kept = 0, False, []
        go()
        assert not calls.kept
        calls.now = 7
        go()
        assert held <= {p for p, s in calls.kept if s == 7}
        calls.capturing, calls.kept = True, []
        go()
        assert not calls.kept
    assert {c[0] for c in calls} == {"spv_norm_rotary", "spv_kv_rotary_append_fp8_heads"}


def test_which_entry_point(calls):
    """Pools in the keys' type take the normed append, fp8 pools of one scale the norm and then their write."""
    rot, norm = Rotary(8, "cpu"), HeadNorm(8, "cpu")
    ids = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 3, 2, 8)
    for dtype, want in ((torch.float32, ["spv_kv_norm_rotary_append"]),
                        (FP8, ["spv_norm_rotary", "spv_kv_append_fp8"])):
        kv = PagedKVCache(1, 2, 8, 4, 16, "cpu", dtype)
        del calls[:]
        rotary_append(x, x, x, kv, 0, ids, ids, rot, norm=norm)
        assert calls.names() == want
        rotary_append(x, x, x, kv, 0, ids, ids, rot)
        assert calls.names()[len(want):] == [n.replace("norm_", "") for n in want]


@pytest.mark.parametrize("pool,head_scales,dtypes", [
    (FP8, False, [None, torch.float32, torch.bfloat16, torch.float16]),
    (FP8, True, [None, torch.float32, torch.bfloat16, torch.float16]),
    (torch.float16, False, [None, torch.float16]),
])
def test_an_empty_read_has_the_type_asked_for(calls, pool, head_scales, dtypes):
    kv = PagedKVCache(1, 2, 8, 4, 16, "cpu", pool, head_scales=head_scales)
    kv.add_sequence(0)
    for dtype in dtypes:
        out = gather_ctx(kv, 0, 0, 0, dtype=dtype)
        assert out.shape == (2, 0, 2, 8)
        assert out.dtype == (dtype or (torch.float32 if pool == FP8 else pool))


_TOO_LARGE = [
    dict(bs=1 << 24, d=128),                   # a page past 2^30 codes
    dict(bs=1 << 30, d=2),
    dict(B=1 << 10, C=1 << 20, bs=1, H=1),     # too many blocks of chunks
    dict(B=1 << 6, C=1 << 15, bs=1, H=32),     # too many workgroups for a launch of 256 threads
    dict(B=1 << 4, C=1 << 19, bs=64, H=512, d=128),  # or of 1,024
]


@pytest.mark.parametrize("kw", _TOO_LARGE, ids=str)
@pytest.mark.parametrize("alloc", [0, 1])
@pytest.mark.parametrize("turned", [False, True])
def test_writes_too_large_for_a_launch_are_refused_before_they_allocate(lib, kw, alloc, turned):
    """An allocation that was launched would end in another error here, where there is no GPU."""
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    B, C, H, d, bs = (kw.get(n, v) for n, v in (("B", 1), ("C", 1), ("H", 2), ("d", 64), ("bs", 16)))
    st = (ctypes.c_int64 * 12)()
    if turned:
        if B * C > 1 << 23:
            B = (1 << 23) // C
            H = H * kw["B"] // B
        rc = lib.spv_kv_rotary_append_fp8_heads(F, F, F, F, 1, st, 1, F, F, 1e-6, F, F, F, F, 4, F, F, F, F, F, F, F, F, F,
                                                F, 1, 1.0, B, C, 4, H, d, d, 0, 0, 2, 4, bs, alloc, None)
    else:
        rc = lib.spv_kv_append_fp8_heads(F, F, F, 1, F, F, st, F, 4, F, F, F, F, F, F, F, B, C, 0, 2, 4, bs, H, d, alloc,
                                         -1, None)
    assert rc == ARG
