"""The rule that cuts 4-bit attention tiles over their keys, on the host: uneven and equal tiles around the
number of workgroups that fills the device."""
import numpy as np
import pytest

from fdl import lib, ops
from fdl.schedule import SeqRows, make_plan

CUS = 256


def _parts(lengths, rows, heads=32, kv_heads=32):
    """(64-key blocks of each tile, parts, blocks per part) of tiles of `rows` rows over these key counts."""
    most = max(lengths)
    plan = make_plan([SeqRows(batch=j, k_end=n, rows=np.arange(rows)) for j, n in enumerate(lengths)],
                     np.zeros((len(lengths), -(-most // 32)), np.int32), 5)
    got, parts, per = ops._kv4_parts(plan, 0, len(lengths), rows, heads // kv_heads, kv_heads, CUS)
    assert got == rows and 1 <= parts <= lib.KV4_MAX_PARTS and per >= 1
    return [-(-n // 64) for n in lengths], parts, per


def _longest(blocks, parts, per):
    """The longest run of blocks that a workgroup takes: parts of `per`, the last one with the rest."""
    out = 0
    for n in blocks:
        p = min(parts, -(-n // per))
        out = max(out, n - (p - 1) * per, per if p > 1 else n)
    return out


@pytest.mark.parametrize("short", [5, 6, 7, 8, 15, 31])
@pytest.mark.parametrize("long,rows", [(65501, 64), (20000, 64), (32000, 128), (65501, 200)])
def test_one_long_tile_beside_short_ones(long, rows, short):
    """However many short tiles stand beside it, the longest run of blocks is a small part of the long one
    (a share of all blocks for every workgroup that the device holds, twice over)."""
    blocks, parts, per = _parts([long] + [768] * short, rows)
    wgs = 32 * -(-rows // 128) if rows > 64 else 32
    share = -(-sum(blocks) * wgs // (2 * CUS))
    assert _longest(blocks, parts, per) <= 2 * share + 12
    assert _longest(blocks, parts, per) * 3 < blocks[0]


def test_several_long_tiles():
    blocks, parts, per = _parts([32000, 768] * 4, 96)
    assert _longest(blocks, parts, per) * 3 < blocks[0]


@pytest.mark.parametrize("n,keys,rows", [(8, 768, 64), (8, 6000, 64), (16, 1024, 64), (8, 1024, 128), (64, 4000, 64)])
def test_equal_tiles_that_fill_the_device_stay_whole(n, keys, rows):
    assert _parts([keys] * n, rows)[1] == 1


def test_slightly_uneven_tiles_stay_whole():
    assert _parts([1536] * 2 + [768] * 6, 64)[1] == 1


def test_fewer_parts_than_asked_for_are_longer_ones(monkeypatch):
    monkeypatch.setattr(ops, "_kv4_most_parts", lambda *a: 3)
    blocks, parts, per = _parts([65501] + [768] * 7, 64)
    assert parts == 3 and _longest(blocks, parts, per) <= -(-blocks[0] // 3)
    blocks, parts, per = _parts([30000, 500], 1, 8, 8)
    assert parts == 3 and _longest(blocks, parts, per) <= -(-blocks[0] // 3) + 3
