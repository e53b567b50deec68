"""The operators of the 4-bit K/V cache as measurable cases, with their plain forms.

kinds
  append   fdl.ops.kv4_append: rotate K (and Q) by the row's position, quantise K and V to 4 bits and
           write them to their cache slots; then fdl.ops.kv4_read of the written rows
  attend   fdl.ops.kv4_attention: block-table attention over the 4-bit cache (single tokens of long
           sequences, masked blocks, full recomputes; grouped-query heads), with the raw-logit
           importance where the case has it
  verify   fdl.ops.kv4_verify_attention: gathered cache keys in 4 bits and the block's own keys in
           bf16 under the Flash-Verify mask

The cache is uint8 [n_slots / 16, n_kv_heads, 2176]: per 16 slots and head the K codes (64 bytes a
slot, channel c in half c % 2 of byte c / 2), the V codes (word w of a slot, channels 8 w .. 8 w + 7, at
(slot / 4, w, slot % 4)), and the scale bytes of K, then of V, [4 groups of 32 channels][16 slots]. A
code is a sign bit and an index into 0 .5 1 1.5 2 3 4 6; scale byte b stands for 2^(b - 127), 255 for NaN.

`own` False: the plain forms in elementary torch operations. `own` True: the framework's calls.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda:0"
HD = 128                    # head dim
CELL, CELL_BYTES = 16, 2176
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
SCALE = 1.0 / math.sqrt(HD)
THETA = 500000.0
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a decode step of eight sequences, one token each (latency): projections made elsewhere, both
        # Q and K rotated on the way
        dict(name="append_token", kind="append", rows=8, pad=0, heads=32, kv_heads=8, pages=64,
             rope=True, shape=1),
        # the block step of eight sequences: 32 masked and 32 tracked rows each at scattered slots; the
        # fused projection has rotated K already
        dict(name="append_block", kind="append", rows=512, pad=0, heads=0, kv_heads=32, pages=192,
             rope=False, shape=2),
        # prompts of uneven length entering the cache, with padding rows behind the last one
        dict(name="append_prompts", kind="append", rows=7919, pad=273, heads=32, kv_heads=8, pages=260,
             rope=True, shape=3),
        # one sequence, one token (latency)
        dict(name="token_one", kind="attend", heads=32, kv_heads=8, seqs=1, keys_lo=2011, keys_hi=2011,
             rows_lo=1, rows_hi=1, full=0, empty=0, page_log2=5, imp=0, shape=1),
        # single-token decode of a serving batch with uneven, mostly long contexts
        dict(name="token_batch", kind="attend", heads=32, kv_heads=8, seqs=24, keys_lo=1000, keys_hi=32768,
             rows_lo=1, rows_hi=1, full=0, empty=0, page_log2=5, imp=0, shape=2),
        # a masked block of 32 rows over a very long context
        dict(name="block_long", kind="attend", heads=32, kv_heads=32, seqs=1, keys_lo=65501, keys_hi=65501,
             rows_lo=32, rows_hi=32, full=0, empty=0, page_log2=8, imp=32, shape=3),
        # the decode step of eight sequences, importance of the masked rows (a layer's call)
        dict(name="block_batch", kind="attend", heads=32, kv_heads=32, seqs=8, keys_lo=768, keys_hi=768,
             rows_lo=64, rows_hi=64, full=0, empty=0, page_log2=5, imp=32, shape=4),
        # a serving batch: 32 sequences of uneven length, a few recomputed in full, one admitted
        # without keys yet
        dict(name="mixed", kind="attend", heads=32, kv_heads=32, seqs=32, keys_lo=512, keys_hi=1536,
             rows_lo=1, rows_hi=96, full=6, empty=1, page_log2=5, imp=32, shape=5),
        # the first step of eight prompts: every row over every key
        dict(name="recompute", kind="attend", heads=32, kv_heads=32, seqs=8, keys_lo=1024, keys_hi=1024,
             rows_lo=1, rows_hi=1, full=8, empty=0, page_log2=5, imp=0, shape=6),
        # the verify forward of one sequence (latency)
        dict(name="verify_one", kind="verify", heads=32, kv_heads=32, seqs=1, keys_lo=320, keys_hi=320,
             block=32, dense=False, shape=1),
        # the verify forward of sixteen sequences, the mask in closed form
        dict(name="verify_batch", kind="verify", heads=32, kv_heads=32, seqs=16, keys_lo=1024, keys_hi=1024,
             block=32, dense=False, shape=2),
        # wide blocks of uneven sequences, the mask as an array, grouped-query heads
        dict(name="verify_wide", kind="verify", heads=32, kv_heads=8, seqs=6, keys_lo=700, keys_hi=2900,
             block=128, dense=True, shape=3),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "verify"])
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 4), (16, 16), (28, 4), (8, 1)])
    if kind == "append":
        rows = _log(rng, 1, 7919)
        return dict(kind=kind, rows=rows, pad=rng.choice([0, 0, rng.randint(1, 40)]),
                    heads=rng.choice([0, heads]), kv_heads=kv_heads, pages=rows // 32 + 2 + rng.randint(0, 64),
                    rope=rng.random() < 0.7, shape=rng.randrange(1 << 20))
    if kind == "verify":
        lo = _log(rng, 70, 1500)
        block = rng.choice([16, 32, 32, 64, 128])
        lo = max(lo, 2 * block + 1)
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, seqs=_log(rng, 1, 16), keys_lo=lo,
                    keys_hi=_log(rng, lo, 2900), block=block, dense=rng.random() < 0.4,
                    shape=rng.randrange(1 << 20))
    regime = rng.choice(["token", "block", "recompute"])
    imp = rng.choice([0, 0, 1])
    page_log2 = rng.choice([4, 5, 5, 6, 8])
    if regime == "token":
        seqs = _log(rng, 1, 24)
        lo = _log(rng, 1, 16000)
        return dict(kind="attend", heads=heads, kv_heads=kv_heads, seqs=seqs, keys_lo=lo,
                    keys_hi=_log(rng, lo, 32768), rows_lo=1, rows_hi=1, full=0,
                    empty=rng.choice([0, 0, 1]) if seqs > 1 else 0, page_log2=page_log2, imp=imp,
                    shape=rng.randrange(1 << 20))
    seqs = _log(rng, 1, 32)
    lo = _log(rng, 100, 1200)
    rows_lo = rng.randint(1, 64)
    full = 0 if regime == "block" else min(seqs, rng.choice([1, 2, 6, 8]))
    return dict(kind="attend", heads=heads, kv_heads=kv_heads, seqs=seqs, keys_lo=lo,
                keys_hi=rng.randint(lo, 1536) if full else _log(rng, lo, 4000), rows_lo=rows_lo,
                rows_hi=rng.randint(rows_lo, 120), full=full, empty=rng.choice([0, 0, 1]) if seqs > full else 0,
                page_log2=page_log2, imp=32 * imp, shape=rng.randrange(1 << 20))


# ------------------------------------------------------------------------------ sizes of a case

def _sizes(case):
    """Per sequence (keys, rows, importance rows) of an attend case, fixed by the case alone."""
    rng = np.random.default_rng(case["shape"])
    out = []
    for i in range(case["seqs"]):
        keys = int(rng.integers(case["keys_lo"], case["keys_hi"] + 1))
        rows = int(rng.integers(case["rows_lo"], case["rows_hi"] + 1))
        if i < case["full"]:
            rows = keys
        elif i >= case["seqs"] - case["empty"]:
            keys = 0
        out.append((keys, rows, min(case["imp"], rows)))
    return out


def _verify_sizes(case):
    """Per sequence (cache keys, fill rows T, candidates S) of a verify case."""
    rng = np.random.default_rng(case["shape"])
    out = []
    for _ in range(case["seqs"]):
        keys = int(rng.integers(case["keys_lo"], case["keys_hi"] + 1))
        s = int(rng.integers(1, case["block"] // 2 + 1))
        out.append((keys, 2 * case["block"] - 2 * s, s))
    return out


def _rotated_by(case):
    return case["rows"] if case["rope"] else 0


def work(case):
    hkv, h = case["kv_heads"], case["heads"]
    if case["kind"] == "append":
        rows = case["rows"]
        n = rows * hkv * (4 * HD + 136)                 # K, V in; codes and scales out
        n += rows * hkv * (4 * HD + 136)                # read back
        n += 4 * rows * h * HD + 8 * _rotated_by(case) * HD
        return {"bytes": n, "flops": 3 * _rotated_by(case) * (h + hkv) * HD}
    n = flops = 0
    if case["kind"] == "attend":
        for keys, rows, imp in _sizes(case):
            n += keys * hkv * 136 + 4 * rows * h * HD + (4 * h * keys if imp else 0)
            flops += 4 * rows * keys * h * HD
    else:
        for keys, t, s in _verify_sizes(case):
            rows = t + 2 * s
            n += (keys - t - s) * hkv * 136 + 4 * rows * (h + hkv) * HD
            flops += 4 * rows * (keys - s + rows - t) * h * HD
    return {"bytes": n, "flops": flops}


# ------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _channels(gen, heads):
    """A spread per channel: a few channels of a head are several times as large as the rest."""
    c = torch.exp(0.5 * torch.randn((heads, HD), generator=gen, device=DEV))
    c[:, torch.randint(0, HD, (3,), generator=gen, device=DEV)] *= 4.0
    return c


def _rows(gen, n, heads, spread):
    x = torch.randn((n, heads, HD), generator=gen, device=DEV)
    return (x * spread).reshape(n, heads * HD).to(BF16)


def _cache(gen, n_slots, kv_heads):
    """A cache whose slots hold quantised rows."""
    cache = torch.empty((n_slots // CELL, kv_heads, CELL_BYTES), dtype=torch.uint8, device=DEV)
    ks, vs = _channels(gen, kv_heads), _channels(gen, kv_heads)
    step = max(CELL, (1 << 19) // kv_heads // CELL * CELL)
    for s0 in range(0, n_slots, step):
        n = min(step, n_slots - s0)
        slot = torch.arange(s0, s0 + n, device=DEV)
        k = _rows(gen, n, kv_heads, ks).float().view(n, kv_heads, HD)
        v = _rows(gen, n, kv_heads, vs).float().view(n, kv_heads, HD)
        _store(cache, slot, k, v)
    return cache


def _queries(gen, n, heads):
    return _rows(gen, n, heads, 1.3 * torch.ones((heads, 1), device=DEV))


def _pages(rng, keys, page_log2):
    """A shuffled page table [n_seq][max_pages] and the pool's slots."""
    need = [-((-k) >> page_log2) for k in keys]
    perm = rng.permutation(sum(need) + 2)
    table = np.zeros((len(keys), max(max(need), 1)), dtype=np.int32)
    at = 0
    for j, n in enumerate(need):
        table[j, :n] = perm[at:at + n]
        at += n
    return table, len(perm) << page_log2


def _slots(table, j, n, page_log2):
    p = np.arange(n, dtype=np.int64)
    return (table[j, p >> page_log2].astype(np.int64) << page_log2) | (p & ((1 << page_log2) - 1))


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def prepare(case, seed):
    gen = _gen(seed)
    rng = np.random.default_rng(seed)
    hkv, h = case["kv_heads"], case["heads"]
    st = dict(case=case)
    if case["kind"] == "append":
        rows, total = case["rows"], case["rows"] + case["pad"]
        n_slots = 32 * case["pages"]
        # K, V (and Q) are column ranges of one product's rows
        x = torch.cat([_rows(gen, total, hkv, _channels(gen, hkv)) for _ in range(2)] +
                      ([_queries(gen, total, h)] if h else []), 1)
        st["k"], st["v"] = x[:, :hkv * HD], x[:, hkv * HD:2 * hkv * HD]
        st["q"] = x[:, 2 * hkv * HD:] if h else None
        st["q_out"] = torch.zeros((total, h * HD), dtype=BF16, device=DEV) if h else None
        st["cache"] = torch.zeros((n_slots // CELL, hkv, CELL_BYTES), dtype=torch.uint8, device=DEV)
        if rows > 1024:    # prompts: consecutive positions in shuffled pages
            slot = _slots(rng.permutation(case["pages"])[None], 0, rows, 5)
        else:
            slot = np.sort(rng.choice(n_slots, rows, replace=False))
        slot = np.concatenate([slot, np.full(case["pad"], -1)])
        st["slot"] = _dev(slot)
        st["sin"] = st["cos"] = st["rope_row"] = None
        if case["rope"]:
            length = 8192
            freq = 1.0 / THETA ** (np.arange(0, HD, 2) / HD)
            ang = np.outer(np.arange(length), freq)
            ang = np.concatenate([ang, ang], 1)
            st["sin"], st["cos"] = _dev(np.sin(ang).astype(np.float32)), _dev(np.cos(ang).astype(np.float32))
            st["rope_row"] = _dev(np.concatenate([rng.integers(0, length - rows) + np.arange(rows)
                                                  if rows > 1024 else rng.integers(0, length, rows),
                                                  np.full(case["pad"], -1)]))
        return st
    if case["kind"] == "attend":
        sizes = _sizes(case)
        table, n_slots = _pages(rng, [k for k, _, _ in sizes], case["page_log2"])
        n_rows = sum(r for _, r, _ in sizes)
        order = rng.permutation(n_rows)          # the step's packed rows of each sequence
        st["q"] = _queries(gen, n_rows, h)
        st["out"] = torch.zeros_like(st["q"])
        st["cache"] = _cache(gen, n_slots, hkv)
        st["imp"] = torch.zeros((h, n_slots), device=DEV) if case["imp"] else None
        st["seqs"], at = [], 0
        for j, (keys, rows, imp) in enumerate(sizes):
            st["seqs"].append(dict(batch=j, k_end=keys, rows=order[at:at + rows].astype(np.int32), n_imp=imp))
            at += rows
        st["tables"] = [(_dev(_slots(table, j, s["k_end"], case["page_log2"])), _dev(s["rows"].astype(np.int64)))
                        for j, s in enumerate(st["seqs"])]
        if own:
            schedule = _package()[1]
            st["plan"] = schedule.make_plan([schedule.SeqRows(**s) for s in st["seqs"]], table,
                                            case["page_log2"], device=DEV)
        return st
    sizes = _verify_sizes(case)
    block = 2 * case["block"]
    table, n_slots = _pages(rng, [k for k, _, _ in sizes], 5)
    n_rows = block * len(sizes)
    st["q"] = _queries(gen, n_rows, h)
    st["k"], st["v"] = (_rows(gen, n_rows, hkv, _channels(gen, hkv)) for _ in range(2))
    st["out"] = torch.zeros_like(st["q"])
    st["cache"] = _cache(gen, n_slots, hkv)
    keys, vblocks, masks = [], [], []
    at = 0
    for j, (n, t, s) in enumerate(sizes):
        # the cache keys are the sequence's slots but those of the block's own rows, decoded ones first
        # in order of importance
        pos = rng.permutation(n)[:n - t - s]
        keys.append(_slots(table, j, n, 5)[pos])
        vblocks.append((at, at + len(pos), block * j, block * (j + 1)))
        at += len(pos)
        masks.append(_mask(t, s) if case["dense"] else (t, s))
    st["block_rows"] = block
    st["key_slots"] = _dev(np.concatenate(keys))
    st["vblocks"] = _dev(np.asarray(vblocks, np.int32))
    st["mask"] = _dev(np.concatenate(masks)) if case["dense"] else _dev(np.asarray(masks, np.int32))
    st["host"] = [(v, t, s) for v, (_, t, s) in zip(vblocks, sizes)]
    return st


def _mask(t, s):
    """[t + 2 s, t + 2 s]: fill rows see no draft; draft i sees drafts j <= i and masks j > i; mask i
    sees drafts j < i and masks j >= i; all else is seen."""
    m = np.ones((t + 2 * s, t + 2 * s), dtype=bool)
    i, j = np.arange(s)[:, None], np.arange(s)[None]
    m[:t, t:t + s] = False
    m[t:t + s, t:t + s] = j <= i
    m[t:t + s, t + s:] = j > i
    m[t + s:, t:t + s] = j < i
    m[t + s:, t + s:] = j >= i
    return m


# ------------------------------------------------------------------------------- plain forms

def _regions(cache):
    """Views of the cells: K codes [c, h, 16, 64], V codes [c, h, 4, 16, 4, 4], scales [c, h, 4, 16]."""
    return (cache[..., :1024].unflatten(-1, (16, 64)), cache[..., 1024:2048].unflatten(-1, (4, 16, 4, 4)),
            cache[..., 2048:2112].unflatten(-1, (4, 16)), cache[..., 2112:].unflatten(-1, (4, 16)))


def _quantise(x):
    """Bytes of two codes [..., 64] and scale bytes [..., 4] of float32 rows [..., 128]."""
    g = x.double().unflatten(-1, (4, 32))
    top = g.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    f, e = torch.frexp(torch.where(bad, 1.0, top))
    e = torch.where(top > 0, e - 3 + (f > 0.875).int(), -127).clamp(-127, 125)
    y = torch.ldexp(torch.where(bad, 0.0, g), -e)
    m = y.abs()
    code = ((m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int() + (m > 2.5).int()
            + (m >= 3.5).int() + (m > 5.0).int())
    code = (code + 8 * torch.signbit(y).int()).flatten(-2)
    scale = torch.where(bad, 255, e + 127).squeeze(-1)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8), scale.to(torch.uint8)


def _store(cache, slot, k, v):
    """Writes float32 rows [n, heads, 128] at their slots."""
    kr, vr, ksr, vsr = _regions(cache)
    cell, s = slot // CELL, slot % CELL
    codes, scales = _quantise(k)
    kr[cell, :, s] = codes
    ksr[cell, :, :, s] = scales
    codes, scales = _quantise(v)
    vr[cell, :, s // 4, :, s % 4] = codes.unflatten(-1, (16, 4))
    vsr[cell, :, :, s] = scales


def _values(codes, scales, dtype):
    """What codes [..., 64] and scales [..., 4] stand for, [..., 128]."""
    lut = torch.tensor(FP4 + tuple(-f for f in FP4), dtype=dtype, device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.to(dtype) - 127))
    return (lut[c.long()].unflatten(-1, (4, 32)) * s.unsqueeze(-1)).flatten(-2)


def _load(cache, slot, dtype=F32):
    """K and V rows [n, heads, 128] of the slots."""
    kr, vr, ksr, vsr = _regions(cache)
    cell, s = slot // CELL, slot % CELL
    return (_values(kr[cell, :, s], ksr[cell, :, :, s], dtype),
            _values(vr[cell, :, s // 4, :, s % 4].flatten(-2), vsr[cell, :, :, s], dtype))


def _rotate(x, sin, cos):
    """x [n, heads, 128] float64, tables [n, 128]."""
    lo, hi = x[..., :64], x[..., 64:]
    sin, cos = sin.double()[:, None], cos.double()[:, None]
    return torch.cat([lo * cos[..., :64] - hi * sin[..., :64], hi * cos[..., 64:] + lo * sin[..., 64:]], -1)


def _softmax_rows(q, k, v, seen=None):
    """q [rows, h, 128], k and v [keys, hkv, 128] float32 -> raw logits [h, rows, keys], out [rows, h, 128]."""
    rows, h, _ = q.shape
    hkv = k.shape[1]
    qh = q.view(rows, hkv, h // hkv, HD).permute(1, 2, 0, 3).reshape(hkv, -1, HD)
    raw = torch.matmul(qh, k.permute(1, 2, 0).contiguous()).view(h, rows, -1)
    s = raw * SCALE
    if seen is not None:
        s = torch.where(seen, s, float("-inf"))
    s = torch.exp(s - s.amax(-1, keepdim=True))
    s = s / s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(hkv, -1, s.shape[-1]), v.transpose(0, 1).contiguous())
    return raw, o.view(h, rows, HD).transpose(0, 1)


def _run_plain(st):
    case = st["case"]
    hkv, h = case["kv_heads"], case["heads"]
    if case["kind"] == "append":
        rows = case["rows"]
        slot = st["slot"][:rows]
        k = st["k"][:rows].view(rows, hkv, HD).double()
        v = st["v"][:rows].view(rows, hkv, HD).float()
        if case["rope"]:
            sin, cos = st["sin"][st["rope_row"][:rows]], st["cos"][st["rope_row"][:rows]]
            k = _rotate(k, sin, cos)
        if h:
            q = st["q"][:rows].view(rows, h, HD).double()
            q = _rotate(q, sin, cos) if case["rope"] else q
            st["q_out"][:rows] = q.reshape(rows, -1).float().to(BF16)
        _store(st["cache"], slot, k.float(), v)
        got = [torch.zeros((rows + case["pad"], hkv * HD), dtype=BF16, device=DEV) for _ in range(2)]
        for g, x in zip(got, _load(st["cache"], slot)):
            g[:rows] = x.reshape(rows, -1).to(BF16)
        return dict(k=got[0], v=got[1], q=st["q_out"], cache=st["cache"])
    if case["kind"] == "attend":
        for s, (slot, rows) in zip(st["seqs"], st["tables"]):
            if s["k_end"] == 0:
                st["out"][rows] = 0
                continue
            k, v = _load(st["cache"], slot)
            raw, o = _softmax_rows(st["q"][rows].float().view(-1, h, HD), k, v)
            st["out"][rows] = o.reshape(-1, h * HD).to(BF16)
            if s["n_imp"]:
                st["imp"][:, slot] = raw[:, :s["n_imp"]].sum(1)
        return dict(out=st["out"], imp=st["imp"])
    for (k0, k1, q0, q1), t, n in st["host"]:
        k, v = _load(st["cache"], st["key_slots"][k0:k1])
        kb, vb = (st[x][q0:q1].float().view(-1, hkv, HD) for x in ("k", "v"))
        seen = torch.ones((q1 - q0, k1 - k0 + q1 - q0), dtype=torch.bool, device=DEV)
        seen[:, k1 - k0:] = st["mask"][q0:q1] if case["dense"] else _dev(_mask(t, n))
        _, o = _softmax_rows(st["q"][q0:q1].float().view(-1, h, HD), torch.cat([k, kb]), torch.cat([v, vb]), seen)
        st["out"][q0:q1] = o.reshape(-1, h * HD).to(BF16)
    return st["out"]


def _package():
    pkg = str(Path(__file__).resolve().parent.parent / "flash-dllm_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from fdl import lib, ops, schedule
    return ops, schedule, lib


def run(st):
    if not own:
        return _run_plain(st)
    ops, _, lib = _package()
    case = st["case"]
    if case["kind"] == "append":
        ops.kv4_append(st["k"], st["v"], st["cache"], st["slot"], rope_sin=st["sin"], rope_cos=st["cos"],
                       rope_row=st["rope_row"], q=st["q"], q_out=st["q_out"])
        k, v = ops.kv4_read(st["cache"], st["slot"])
        return dict(k=k, v=v, q=st["q_out"], cache=st["cache"])
    if case["kind"] == "attend":
        ops.kv4_attention(st["q"], st["cache"], st["plan"], st["out"], case["heads"], SCALE,
                          lib.IMP_RAW_LOGIT if case["imp"] else lib.IMP_NONE, st["imp"])
        return dict(out=st["out"], imp=st["imp"])
    ops.kv4_verify_attention(st["q"], st["k"], st["v"], st["cache"], st["key_slots"], st["vblocks"],
                             st["mask"], st["block_rows"], st["out"], case["heads"], SCALE)
    return st["out"]


# ------------------------------------------------------------------------------ in 64 bits

_CODE = [s * f for s in (1.0, -1.0) for f in FP4]


def _byte_rows(cache, slot):
    """float64 K and V [n, heads, 128] of slots, byte by byte from the layout's definition."""
    flat = cache.view(-1, CELL_BYTES)
    heads = cache.shape[1]
    base = (slot // CELL)[:, None] * heads + torch.arange(heads, device=cache.device)
    rows = flat[base.flatten()].view(len(slot), heads, CELL_BYTES)
    s = (slot % CELL)[:, None]
    ch = torch.arange(HD, device=cache.device)[None]
    at_k = 64 * s + ch // 2
    at_v = 1024 + 256 * (s // 4) + 16 * (ch // 8) + 4 * (s % 4) + ch % 8 // 2
    out = []
    for at, at_s in ((at_k, 2048), (at_v, 2112)):
        at_s = at_s + 16 * (ch // 32) + s
        pick = lambda a: rows.gather(2, a[:, None].expand(-1, heads, -1)).long()  # noqa: E731
        code = (pick(at) >> (4 * (ch % 2))) & 15
        scale = pick(at_s).double()
        scale = torch.where(scale == 255, float("nan"), 2.0 ** (scale - 127))
        out.append(torch.tensor(_CODE, dtype=F64, device=cache.device)[code] * scale)
    return out


def _attend64(q, k, v, seen=None):
    """One K/V head: q [m, 128], k and v [n, 128] float64 -> logits before scaling, out."""
    raw = q @ k.T
    s = raw * SCALE
    if seen is not None:
        s = s.masked_fill(~seen, -math.inf)
    return raw, torch.softmax(s, -1) @ v


def _nearest(x):
    """The 4-bit values of float64 rows [n, heads, 128] and their (code, scale byte)."""
    grid = torch.tensor(FP4, dtype=F64, device=x.device)
    g = x.reshape(*x.shape[:-1], 4, 32)
    top = g.abs().amax(-1)
    e = torch.full_like(top, -127.0)
    pos = top > 0
    e[pos] = torch.ceil(torch.log2(top[pos] / 7))
    for _ in range(2):                     # log2 may be off by an ulp at the limit
        e = torch.where(pos & (top > 7 * 2.0 ** e), e + 1, e)
        e = torch.where(pos & (top <= 7 * 2.0 ** (e - 1)), e - 1, e)
    e = e.clamp(-127, 125)
    y = g.abs() / 2.0 ** e.unsqueeze(-1)
    lo = (torch.bucketize(y, grid, right=True) - 1).clamp(0, 7)
    hi = (lo + 1).clamp(max=7)
    dl, dh = y - grid[lo], grid[hi] - y
    up = (hi > lo) & ((dh < dl) | ((dh == dl) & (hi % 2 == 0)))
    code = torch.where(up, hi, lo)
    neg = torch.signbit(g)
    val = grid[code] * 2.0 ** e.unsqueeze(-1) * torch.where(neg, -1.0, 1.0)
    return val.reshape(x.shape), (code + 8 * neg).reshape(x.shape), (e + 127).long()


def exact(case, seed):
    st = prepare(case, seed)
    hkv, h = case["kv_heads"], case["heads"]
    if case["kind"] == "append":
        rows, total = case["rows"], case["rows"] + case["pad"]
        turn = torch.zeros((rows, 64), dtype=torch.complex128, device=DEV)
        if case["rope"]:
            r = st["rope_row"][:rows]
            turn = torch.complex(st["cos"][r, :64].double(), st["sin"][r, :64].double())

        def rotated(x, heads):
            x = x[:rows].double().view(rows, heads, HD)
            if not case["rope"]:
                return x
            z = torch.complex(x[..., :64], x[..., 64:])
            t = turn[:, None]
            return torch.cat([z.real * t.real - z.imag * t.imag, z.imag * t.real + z.real * t.imag], -1)

        cache = torch.zeros_like(st["cache"])
        flat = cache.view(-1, CELL_BYTES)
        slot = st["slot"][:rows]
        base = (slot // CELL)[:, None] * hkv + torch.arange(hkv, device=DEV)
        s = (slot % CELL)[:, None, None]
        byte, grp = torch.arange(64, device=DEV), torch.arange(4, device=DEV)
        res = []
        for x, at, at_s in ((rotated(st["k"], hkv).float().double(), 64 * s + byte, 2048),
                            (st["v"][:rows].double().view(rows, hkv, HD),
                             1024 + 256 * (s // 4) + 16 * (byte // 4) + 4 * (s % 4) + byte % 4, 2112)):
            val, code, scale = _nearest(x)
            pair = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)
            flat[base[..., None].expand_as(pair), at.expand_as(pair)] = pair
            flat[base[..., None].expand_as(scale), (at_s + 16 * grp + s).expand_as(scale)] = scale.to(torch.uint8)
            full = torch.zeros((total, hkv * HD), dtype=F64, device=DEV)
            full[:rows] = val.view(rows, -1)
            res.append(full)
        q = None
        if h:
            q = torch.zeros((total, h * HD), dtype=F64, device=DEV)
            q[:rows] = rotated(st["q"], h).reshape(rows, -1)
        return dict(k=res[0], v=res[1], q=q, cache=cache)
    g = h // hkv
    out = torch.zeros(st["out"].shape, dtype=F64, device=DEV)
    o4 = out.view(-1, hkv, g, HD)
    q4 = st["q"].view(-1, hkv, g, HD)
    if case["kind"] == "attend":
        imp = torch.zeros(st["imp"].shape, dtype=F64, device=DEV) if case["imp"] else None
        for s, (slot, rows) in zip(st["seqs"], st["tables"]):
            if s["k_end"] == 0:
                continue
            k, v = _byte_rows(st["cache"], slot)
            for a in range(hkv):
                for b in range(g):
                    raw, o4[rows, a, b] = _attend64(q4[rows, a, b].double(), k[:, a], v[:, a])
                    if s["n_imp"]:
                        imp[a * g + b, slot] = raw[:s["n_imp"]].sum(0)
        return dict(out=out, imp=imp)
    for (k0, k1, q0, q1), t, n in st["host"]:
        k, v = _byte_rows(st["cache"], st["key_slots"][k0:k1])
        k = torch.cat([k, st["k"][q0:q1].double().view(-1, hkv, HD)])
        v = torch.cat([v, st["v"][q0:q1].double().view(-1, hkv, HD)])
        seen = torch.cat([torch.ones((q1 - q0, k1 - k0), dtype=torch.bool, device=DEV), _dev(_mask(t, n))], 1)
        for a in range(hkv):
            for b in range(g):
                o4[q0:q1, a, b] = _attend64(q4[q0:q1, a, b].double(), k[:, a], v[:, a], seen)[1]
    return out
