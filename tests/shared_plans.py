"""Plans of shared-prefix batches cut as a test wants them, in the layout of
spv_shared_attn_plan: a header, segments (sequence, length, kv head, first member, first
row, rows, first key, end of keys) ordered by group, kv head, range and tile, the groups'
members, and per entry its group's first segment, tiles, ranges and its rank there."""

from __future__ import annotations

import ctypes

import torch

UNIT = 64  # keys


def cut_plan(plan, ids, lens, units, tile):
    """``plan`` (a list of words) with ranges of ``units(units of a group's prefix)`` units of 64 keys
    and tiles of ``tile`` rows in place of the library's choice."""
    B, C, hq, hkv = plan[2:6]
    G = C * (hq // hkv)
    groups = {}
    for b, (s, n) in enumerate(zip(ids, lens)):
        if s >= 0 and n > 0:
            groups.setdefault((s, n), []).append(b)
    segs, members, entries = [], [], [[-1, 0, 0, 0] for _ in range(B)]
    for (s, n), who in groups.items():
        all_units, rows = -(-n // UNIT), len(who) * G
        per = units(all_units)
        tiles, ranges = -(-rows // tile), -(-all_units // per)
        first = len(segs)
        for h in range(hkv):
            for r in range(ranges):
                for t in range(tiles):
                    segs.append([s, n, h, len(members), t * tile, min(tile, rows - t * tile), r * per * UNIT,
                                 min((r + 1) * per * UNIT, n)])
        for rank, b in enumerate(who):
            entries[b] = [first, tiles, ranges, rank]
        members += who
    out = list(plan[:14])
    out[7], out[13] = len(segs), tile
    for word, part in ((9, sum(segs, [])), (10, members), (11, sum(entries, []))):
        out += [0] * (-len(out) % 16)
        out[word] = len(out)
        out += part
    out[1] = len(out)
    return out


def segments(plan):
    return [plan[plan[9] + 8 * i:plan[9] + 8 * i + 8] for i in range(plan[7])]


def recut(prefix, ids, lens, units, tile=256):
    """Gives a ``SharedPrefix`` made of ``ids`` and ``lens`` a plan cut so; returns its segments."""
    plan = cut_plan(list(prefix._host), ids, lens, units, tile)
    prefix._host = (ctypes.c_int32 * len(plan))(*plan)
    prefix._dev = torch.tensor(plan, dtype=torch.int32, device=prefix.kv.device)
    prefix._bytes = (0, 0)
    return segments(plan)
