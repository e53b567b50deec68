"""The queries that fdl_kv4_append rotates: rounded to bf16 once, bit for bit."""
import numpy as np
import pytest
import torch

from fdl import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def _bf16_bits(d):
    """Bits of float64 values rounded to bf16 once, to nearest, ties to even (no subnormals, no overflow)."""
    b = np.abs(d).view(np.uint64)
    keep = np.uint64(45)  # 52 - 7 bits go
    b = b + (np.uint64(1) << np.uint64(44)) - np.uint64(1) + (b >> keep & np.uint64(1)) >> keep
    expo = (b >> np.uint64(7)).astype(np.int64) - 1023 + 127
    assert ((expo > 0) & (expo < 255))[d != 0].all()
    out = np.where(d == 0, 0, expo << 7 | (b & np.uint64(127)).astype(np.int64))
    return (out | np.where(np.signbit(d), 0x8000, 0)).astype(np.int64)


def _append(q, sin, cos, row):
    n, heads = q.shape[0], q.shape[1] // 128
    k = torch.zeros((n, 128), dtype=BF16, device=DEV)
    got = torch.zeros((n, heads * 128), dtype=BF16, device=DEV)
    ops.kv4_append(k, k, ops.kv4_cache(-(-n // 16) * 16, 1, DEV), torch.arange(n, device=DEV),
                   rope_sin=torch.from_numpy(sin).to(DEV), rope_cos=torch.from_numpy(cos).to(DEV),
                   rope_row=torch.from_numpy(row).to(DEV), q=q.to(DEV), q_out=got)
    return got.view(torch.int16).cpu().numpy().astype(np.int64) & 0xffff


def _rotated(q, sin, cos):
    x = q.double().numpy().reshape(len(q), -1, 128)
    lo, hi = x[..., :64], x[..., 64:]
    s, c = sin.astype(np.float64)[:, None], cos.astype(np.float64)[:, None]
    return np.concatenate([lo * c[..., :64] - hi * s[..., :64], hi * c[..., 64:] + lo * s[..., 64:]],
                          -1).reshape(len(q), -1)


def test_values_next_to_the_middle_of_two_bf16():
    """1 + 2^-8, half way between two bf16 values, and 2^-40 (less than 32 bits see) to either side, at several
    exponents and signs: up, down, and to even at the middle itself."""
    q = torch.zeros((6, 128), dtype=BF16)
    sin, cos = np.zeros((6, 128), np.float32), np.zeros((6, 128), np.float32)
    for r, (mid, off) in enumerate([(1 + 2.0 ** -8, 2.0 ** -40), (1 + 2.0 ** -8, -2.0 ** -40), (1 + 2.0 ** -8, 0.0),
                                    (1 + 3 * 2.0 ** -8, 2.0 ** -40), (1 + 3 * 2.0 ** -8, -2.0 ** -40),
                                    (1 + 3 * 2.0 ** -8, 0.0)]):
        q[r, :64] = torch.tensor([1.0, -1.0, 2.0 ** 20, -2.0 ** -30]).repeat(16)
        q[r, 64:] = -q[r, :64]
        cos[r], sin[r, :64], sin[r, 64:] = mid, off, -off  # lo c - hi s = lo (mid + off); hi c + lo s = hi (mid + off)
    want = _rotated(q, sin, cos)
    assert (want[0] != want[2]).all() and (want[1] != want[2]).all()
    got = _append(q, sin, cos, np.arange(6))
    assert np.array_equal(got, _bf16_bits(want))


def test_random_rotations():
    rng = np.random.default_rng(0)
    n = 8192
    q = torch.from_numpy(rng.standard_normal((n, 8 * 128))).to(BF16)
    ang = np.outer(rng.integers(0, 32768, n), 1.0 / 500000.0 ** (np.arange(0, 128, 2) / 128))
    ang = np.concatenate([ang, ang], 1)
    sin, cos = np.sin(ang).astype(np.float32), np.cos(ang).astype(np.float32)
    got = _append(q, sin, cos, np.arange(n))
    want = _rotated(q, sin, cos)
    bits = _bf16_bits(np.where(np.abs(want) < 1e-30, 1.0, want))
    assert np.array_equal(got[np.abs(want) >= 1e-30], bits[np.abs(want) >= 1e-30])
