"""Attention over the 4-bit cache cut over its keys on the GPU: uneven tiles that fill the device, and workspaces
whose unwritten records hold NaN."""
import math

import numpy as np
import pytest
import torch

import kv4_plain as plain
from fdl import lib, ops
from fdl.schedule import SeqRows, make_plan
from test_gpu_kv4 import _check_verify

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
SCALE = 1.0 / math.sqrt(128)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


@pytest.mark.parametrize("lengths,rows,heads,kv_heads", [
    ([9000] + [150] * 8, 64, 32, 32), ([150, 9000] + [64] * 3, 200, 32, 32), ([8000, 100] * 4, 40, 32, 16)])
def test_uneven_tiles_that_fill_the_device(lengths, rows, heads, kv_heads):
    """One or few long tiles beside short ones are cut; every row equals the definition and every call itself."""
    rng = np.random.default_rng(rows)
    need = [-(-n // 32) for n in lengths]
    perm = rng.permutation(sum(need))
    table = np.zeros((len(lengths), max(need)), np.int32)
    at = 0
    for j, n in enumerate(need):
        table[j, :n] = perm[at:at + n]
        at += n
    n_slots = 32 * len(perm)
    cache = plain.random_cache(rng, n_slots, kv_heads)
    q = torch.from_numpy(rng.standard_normal((rows * len(lengths), heads * 128))).to(BF16)
    plan = make_plan([SeqRows(batch=j, k_end=n, rows=np.arange(j * rows, (j + 1) * rows), n_imp=min(rows, 32))
                      for j, n in enumerate(lengths)], table, 5, device=DEV)
    group = heads // kv_heads
    (first, count, tile), = [x for x in ops._kv4_ranges(plan, group) if x[1]]
    tile, parts, _ = ops._kv4_parts(plan, first, count, tile, group, kv_heads, ops._cus(torch.device(DEV)))
    assert parts > 1
    floats = parts * count * tile * heads * lib.KV4_PART_FLOATS
    ws = torch.full((floats + 1024,), float("nan"), device=DEV)
    out = torch.full(q.shape, 5.0, dtype=BF16, device=DEV)
    imp = torch.zeros((heads, n_slots), device=DEV)
    ops.kv4_attention(q.to(DEV), _dev(cache), plan, out, heads, SCALE, lib.IMP_RAW_LOGIT, imp, workspace=ws)
    assert ws[floats:].isnan().all() and not ws[:floats].isnan().all()
    for j, n in enumerate(lengths):
        slots = (table[j, np.arange(n) >> 5].astype(np.int64) << 5) | (np.arange(n) & 31)
        k, v = (torch.from_numpy(x) for x in plain.get(cache, slots))
        r = slice(j * rows, (j + 1) * rows)
        for h in range(0, heads, 5):  # 64-bit arithmetic for some of the heads
            q64 = q[r].double().view(rows, heads, 128)[:, h:h + 1]
            kh, vh = (x[:, h // group:h // group + 1] for x in (k, v))
            o, tol, raw = plain.attend(q64, kh, vh, SCALE)
            plain.close(out[r].double().cpu().view(rows, heads, 128)[:, h:h + 1], o, tol, f"sequence {j}")
            plain.close(imp.double().cpu()[h:h + 1, slots], raw[:, :min(rows, 32)].sum(1),
                        plain.importance_bound(q64, kh, min(rows, 32)), f"importance {j}")
    again = torch.full_like(out, 5.0)
    ops.kv4_attention(q.to(DEV), _dev(cache), plan, again, heads, SCALE)
    assert torch.equal(out, again)


@pytest.mark.parametrize("heads,kv_heads,block_rows,blocks", [
    (4, 4, 64, [(1500, 64)]),                      # (keys, rows)
    (8, 2, 128, [(3001, 70), (40, 128)]),          # the second within the first part
    (4, 1, 256, [(2000, 256), (0, 200)]),
    (2, 2, 16, [(4400, 9), (2100, 16)])])          # slots in more than one stage
@pytest.mark.parametrize("per", [None, 1, 3])
def test_verify_parts_in_the_given_workspace(monkeypatch, heads, kv_heads, block_rows, blocks, per):
    """The workspace given is the one used, up to its documented size, and records that no part writes are not
    read: they hold NaN."""
    rng = np.random.default_rng(block_rows + heads)
    n_slots = 16 * 300
    n_rows = sum(r for _, r in blocks) + 2
    q = torch.from_numpy(rng.standard_normal((n_rows, heads * 128)) * 1.5).to(BF16)
    kb, vb = (torch.from_numpy(rng.standard_normal((n_rows, kv_heads * 128))).to(BF16) for _ in range(2))
    cache = plain.random_cache(rng, n_slots, kv_heads)
    keys = [rng.permutation(n_slots)[:n].astype(np.int64) for n, _ in blocks]
    vblocks, at, row = [], 0, 1
    for n, r in blocks:
        vblocks.append((at, at + n, row, row + r))
        at, row = at + n, row + r
    masks = [rng.random((r, r)) < 0.5 for _, r in blocks]
    dense = np.ones((len(blocks) * block_rows, block_rows), bool)
    for i, m in enumerate(masks):
        m[0] = False
        dense[i * block_rows:i * block_rows + len(m), :len(m)] = m
    parts, _ = ops._kv4_verify_parts(at, len(blocks), block_rows, heads // kv_heads, kv_heads,
                                     ops._cus(torch.device(DEV)))
    if per is not None:
        parts = min(at // (64 * per) + 4, 256)
        monkeypatch.setattr(ops, "_kv4_verify_parts", lambda *_: (parts, per))
    assert parts > 1
    floats = parts * len(blocks) * block_rows * heads * lib.KV4_PART_FLOATS
    ws = torch.full((floats + 1024,), float("nan"), device=DEV)
    out = torch.full(q.shape, 5.0, dtype=BF16, device=DEV)
    ops.kv4_verify_attention(q.to(DEV), kb.to(DEV), vb.to(DEV), _dev(cache), _dev(np.concatenate(keys)),
                             _dev(np.asarray(vblocks, np.int32)), _dev(dense), block_rows, out, heads, SCALE,
                             workspace=ws)
    assert ws[floats:].isnan().all() and not ws[:floats].isnan().all()
    _check_verify(q, kb, vb, cache, np.concatenate(keys), vblocks, masks, out, heads, kv_heads)
    assert (out[0] == 5.0).all() and (out[n_rows - 1:] == 5.0).all()
