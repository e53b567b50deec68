"""The 4-bit cache's attention holds its logits in 32 bits, also where one channel's product is far above the
others': against 64 bits, with bounds from the roundings alone."""
import math

import numpy as np
import pytest
import torch

import kv4_plain as plain
from fdl import ops
from fdl.schedule import SeqRows, make_plan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
SCALE = 1.0 / math.sqrt(128)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _cache(rng, n_slots, kv_heads):
    """Random codes at scale 1, channel 5 of every group of K the same value (4) in every slot."""
    cache = plain.random_cache(rng, n_slots, kv_heads)
    cache[..., 2048:] = 127
    k = cache[..., :1024].reshape(*cache.shape[:2], 16, 4, 16)
    k[..., 2] = (k[..., 2] & 0x0f) | 0x60
    return cache


def _queries(rng, rows, heads, top):
    """Channel 5 of every group is `top`: it adds the same to every key's logit."""
    q = 0.6 * rng.standard_normal((rows, heads, 4, 32))
    q[..., 5] = top
    return torch.from_numpy(q.reshape(rows, heads * 128)).to(BF16)


def _expected(q, k, v, seen=None):
    """out [rows, h, 128] and its bound. With weights p (1 + e) in the place of p, |e| <= d, the normalised sum
    moves by at most d / (1 - d) sum p |v - out|. d: the logit's 128 exact products summed in 32 bits (128
    roundings of 2^-24 of sum |q k|), its product with the scale, the maximum's and their difference (3
    of 2^-24 of the logit), exp2 (2^-22), and the rounding of p to bf16 (2^-8). The keys' sum in 32 bits adds
    n 2^-24 sum p |v|, the output's rounding 2^-8."""
    grp = q.shape[1] // k.shape[1]
    qh = q.transpose(0, 1)
    kh, vh = (x.transpose(0, 1).repeat_interleave(grp, 0) for x in (k, v))
    s = qh @ kh.transpose(1, 2) * SCALE
    mag = (qh.abs() @ kh.abs().transpose(1, 2)).amax(-1, keepdim=True) * SCALE
    if seen is not None:
        s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    o = p @ vh
    d = mag * 2.0 ** -17 + 3 * mag * 2.0 ** -24 + 2.0 ** -22
    d = torch.expm1(d) + 2.0 ** -8
    spread = torch.stack([(p[:, r, :, None] * (vh - o[:, r, None]).abs()).sum(1) for r in range(q.shape[0])], 1)
    tol = d / (1 - d) * spread + len(k) * 2.0 ** -24 * (p @ vh.abs())
    return o.transpose(0, 1), (tol + (o.abs() + tol) * 2.0 ** -8).transpose(0, 1)


@pytest.mark.parametrize("top", [64.0, 1024.0])
@pytest.mark.parametrize("rows,heads,kv_heads,keys", [
    (1, 4, 4, 40), (1, 8, 2, 2300), (20, 2, 2, 70), (40, 2, 2, 70), (70, 4, 2, 130), (300, 1, 1, 90)])
def test_attention_with_a_dominant_channel(top, rows, heads, kv_heads, keys):
    rng = np.random.default_rng(rows + heads)
    n_slots = -(-keys // 32) * 32
    cache = _cache(rng, n_slots, kv_heads)
    q = _queries(rng, rows, heads, top)
    table = rng.permutation(n_slots // 32).astype(np.int32)[None]
    slots = (table[0, np.arange(keys) >> 5].astype(np.int64) << 5) | (np.arange(keys) & 31)
    plan = make_plan([SeqRows(batch=0, k_end=keys, rows=np.arange(rows))], table, 5, device=DEV)
    out = torch.zeros(q.shape, dtype=BF16, device=DEV)
    ops.kv4_attention(q.to(DEV), _dev(cache), plan, out, heads, SCALE)
    k, v = (torch.from_numpy(x) for x in plain.get(cache, slots))
    o, tol = _expected(q.double().view(rows, heads, 128), k, v)
    plain.close(out.double().cpu().view(rows, heads, 128), o, tol)


@pytest.mark.parametrize("top", [64.0, 1024.0])
@pytest.mark.parametrize("rows,heads,kv_heads,keys", [(48, 2, 2, 70), (48, 4, 1, 70), (200, 2, 2, 150)])
def test_verify_with_a_dominant_channel(top, rows, heads, kv_heads, keys):
    rng = np.random.default_rng(rows + heads)
    n_slots = 256
    cache = _cache(rng, n_slots, kv_heads)
    q = _queries(rng, rows, heads, top)
    kb = rng.standard_normal((rows, kv_heads, 4, 32))
    kb[..., 5] = 4.0
    kb, vb = (torch.from_numpy(x.reshape(rows, -1)).to(BF16) for x in (kb, rng.standard_normal((rows, kv_heads * 128))))
    slots = rng.permutation(n_slots)[:keys].astype(np.int64)
    mask = rng.random((rows, rows)) < 0.5
    out = torch.zeros(q.shape, dtype=BF16, device=DEV)
    ops.kv4_verify_attention(q.to(DEV), kb.to(DEV), vb.to(DEV), _dev(cache), _dev(slots),
                             _dev(np.array([[0, keys, 0, rows]], np.int32)), _dev(mask), rows, out, heads, SCALE)
    k, v = (torch.cat([torch.from_numpy(a), b.double().view(rows, kv_heads, 128)])
            for a, b in zip(plain.get(cache, slots), (kb, vb)))
    seen = torch.cat([torch.ones((rows, keys), dtype=torch.bool), torch.from_numpy(mask)], 1)
    o, tol = _expected(q.double().view(rows, heads, 128), k, v, seen)
    plain.close(out.double().cpu().view(rows, heads, 128), o, tol)


@pytest.mark.parametrize("rows,keys", [(1, 70), (20, 70), (40, 130), (100, 70)])
def test_infinite_queries_are_nan(rows, keys):
    """A query with an infinity whose logits are all the same infinity: NaN, as the softmax of such a row, and not
    the zeros of a row without keys. The other queries stay right."""
    rng = np.random.default_rng(rows)
    heads, n_slots = 2, 160
    cache = _cache(rng, n_slots, heads)  # channel 5 of K is 4 everywhere
    q = _queries(rng, rows, heads, 1.0)
    q[0, 5], q[rows // 2, 128 + 32 + 5] = -math.inf, math.inf
    plan = make_plan([SeqRows(batch=0, k_end=keys, rows=np.arange(rows))],
                     np.arange(n_slots // 32, dtype=np.int32)[None], 5, device=DEV)
    out = torch.zeros(q.shape, dtype=BF16, device=DEV)
    ops.kv4_attention(q.to(DEV), _dev(cache), plan, out, heads, SCALE)
    got = out.double().cpu().view(rows, heads, 128)
    k, v = (torch.from_numpy(x) for x in plain.get(cache, np.arange(keys)))
    odd = torch.zeros((rows, heads), dtype=torch.bool)
    odd[0, 0] = odd[rows // 2, 1] = True
    assert got[odd].isnan().all()
    o, tol = _expected(torch.where(odd[..., None], 0.0, q.double().view(rows, heads, 128)), k, v)
    plain.close(got[~odd], o[~odd], tol[~odd])


@pytest.mark.parametrize("lowest", [0, 2, 120])
@pytest.mark.parametrize("rows,keys", [(1, 70), (20, 70), (40, 130), (100, 70)])
def test_tiny_keys_and_huge_queries(lowest, rows, keys):
    """Groups at the smallest scales, whose values are below the smallest normal bf16, times queries as large as
    that makes ordinary logits."""
    rng = np.random.default_rng(rows + lowest)
    heads, n_slots = 2, 160
    cache = plain.random_cache(rng, n_slots, heads)
    cache[..., 2048:2112] = rng.integers(lowest, lowest + 2, cache[..., 2048:2112].shape)
    cache[..., 2112:] = 127
    q = torch.from_numpy(0.3 * rng.standard_normal((rows, heads * 128)) * 2.0 ** (126 - lowest)).to(BF16)
    plan = make_plan([SeqRows(batch=0, k_end=keys, rows=np.arange(rows))],
                     np.arange(n_slots // 32, dtype=np.int32)[None], 5, device=DEV)
    out = torch.zeros(q.shape, dtype=BF16, device=DEV)
    ops.kv4_attention(q.to(DEV), _dev(cache), plan, out, heads, SCALE)
    k, v = (torch.from_numpy(x) for x in plain.get(cache, np.arange(keys)))
    o, tol = _expected(q.double().view(rows, heads, 128), k, v)
    plain.close(out.double().cpu().view(rows, heads, 128), o, tol)
