"""PAGED_ATTN of infinite and undefined values in rows of one workgroup and in rows whose parts are joined: what the formula
gives in IEEE arithmetic, in 64 bits. An infinite value under a weight makes its dim infinite and no other."""
import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import half_step, make_attention, run_attention

pytestmark = pytest.mark.gpu


def formula(q, cache, table, scale, base, neox):
    """(out [B, H, hd], a bound on what fp32 may be off where it is finite). Products and sums one by one: a BLAS may leave
    zeros out."""
    B, H, hd = q.shape
    R, KV = cache.shape[2], cache.shape[1] // 2
    out, off = np.zeros((B, H, hd)), np.zeros((B, H, hd))
    with np.errstate(invalid="ignore", over="ignore"):
        for b in range(B):
            n = int(table[b, 0])
            if n == 0:
                continue
            pos = np.arange(n)
            rows = cache[table[b, 1 + pos // R].astype(np.int64), :, pos % R].astype(np.float64)
            qr = ref.rotate(q[b][None], [n - 1], base, neox)[0]
            for h in range(H):
                k, v = rows[:, h // (H // KV)], rows[:, KV + h // (H // KV)]
                s = scale * (k * qr[h]).sum(-1)
                if np.isnan(s).any() or np.isposinf(s).any():
                    out[b, h] = np.nan
                    continue
                alive = ~np.isneginf(s)
                if not alive.any():
                    continue
                p = np.where(alive, np.exp(np.where(alive, s, 0) - s[alive].max()), 0)
                p /= p.sum()
                out[b, h] = (p[:, None] * v).sum(0)
                # as paged_ref.attention counts it, over the keys that have a weight and the values that are finite
                w = np.where(np.isfinite(v), np.abs(v), 0)
                eps = (16 + 8 * (base != 0)) * 2.0 ** -24 * abs(scale) * (np.abs(k[alive]) * np.abs(qr[h])).sum(-1).max() \
                    + 2.0 ** -22 * np.abs(s[alive]).max()
                off[b, h] = (2.2 * eps + 32 * 2.0 ** -24) * (p @ w) + n * 2.0 ** -33 * w.max(0)
    return out, off


def check(got, q, cache, table, scale, base, neox):
    want, off = formula(q[0], cache, table, scale, base, neox)
    print(f"  {np.isnan(want).sum()} undefined, {np.isinf(want).sum()} infinite of {want.size}", flush=True)
    finite = np.isfinite(want)
    assert np.array_equal(got[~finite].astype(np.float64), want[~finite], equal_nan=True)
    tol = half_step(np.where(finite, want, 0), q.dtype.type) * (1 + 2.0 ** -10) + off
    with np.errstate(invalid="ignore"):
        d = np.abs(got.astype(np.float64) - want)
    assert (d[finite] <= tol[finite]).all()
    return want


def at(table, b, pos, R):
    return table[b, 1 + np.asarray(pos) // R].astype(np.int64), np.asarray(pos) % R


SHAPES = [  # lengths, H, KV, hd, R
    ([200, 129, 1, 0, 333], 4, 4, 64, 16), ([500, 70], 8, 2, 128, 16), ([260, 40], 6, 3, 48, 16), ([300, 17], 4, 2, 80, 64),
    ([130, 1], 8, 4, 256, 16), ([90, 200], 2, 1, 136, 32), ([9000, 3], 16, 1, 128, 64), ([12000, 200], 5, 1, 64, 16),
    ([7001], 2, 1, 24, 16), ([3000, 0], 10, 2, 256, 16)]
ROPES = [(0.0, False), (1e4, False), (1e4, True)]


@pytest.mark.parametrize("dtype", [np.float32])
@pytest.mark.parametrize("base,neox", ROPES, ids=["plain", "pairs", "halves"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0][0]}-{s[1]}-{s[2]}-{s[3]}")
def test_infinite_values(ctx, vk, shape, base, neox, dtype):
    """Infinite and undefined values here and there; a dim with both signs is undefined."""
    lengths, H, KV, hd, R = shape
    print(f"[infinite values] {shape} {base} {neox} {dtype.__name__}", flush=True)
    r = np.random.default_rng(hd + H + 1)
    q, cache, table = make_attention(r, lengths, H, KV, hd, R, dtype)
    for b, n in enumerate(lengths):
        for kv in range(KV if n else 0):
            dims = r.permutation(hd)
            for d, x in [(dims[0], np.inf), (dims[1], -np.inf), (dims[2], np.nan), (dims[3], np.inf), (dims[3], -np.inf)]:
                page, row = at(table, b, r.integers(n), R)
                cache[page, KV + kv, row, d] = x
            page, row = at(table, b, n - 1, R)
            cache[page, KV + kv, row, dims[4]] = np.inf
    got = run_attention(ctx, vk, q, cache, table, hd ** -0.5, base, neox)
    want = check(got, q, cache, table, hd ** -0.5, base, neox)
    assert np.isinf(want).any() and np.isfinite(want).mean() > 0.5
