"""PAGED_ATTN of infinite and undefined keys, queries and values, with and without a rotation, in both types, in rows of one
workgroup and in rows whose parts are joined: what the formula gives in IEEE arithmetic, in 64 bits. A key whose score is -inf
has no weight, a score of +inf or NaN leaves its head undefined, a row of scores that are all -inf is zero, and an infinite
value under a weight makes its dim infinite and no other."""
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


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("base,neox", ROPES, ids=["plain", "pairs", "halves"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0][0]}-{s[1]}-{s[2]}-{s[3]}")
def test_infinite_keys(ctx, vk, shape, base, neox, dtype):
    """Infinite elements of keys, most of them against the sign of the first query head's element: that head's scores of them
    are -inf, others' are of either sign."""
    lengths, H, KV, hd, R = shape
    print(f"[infinite keys] {shape} {base} {neox} {dtype.__name__}", flush=True)
    r = np.random.default_rng(hd + H)
    q, cache, table = make_attention(r, lengths, H, KV, hd, R, dtype)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        qr = ref.rotate(q[0, b][None], [n - 1], base, neox)[0]
        for kv in range(KV):
            for pos in r.permutation(n)[:max(1, n // 7)]:
                page, row = at(table, b, pos, R)
                for d in r.permutation(hd)[:r.integers(1, 4)]:
                    cache[page, kv, row, d] = -np.sign(qr[kv * (H // KV), d]) * np.inf
    got = run_attention(ctx, vk, q, cache, table, hd ** -0.5, base, neox)
    check(got, q, cache, table, hd ** -0.5, base, neox)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
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


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("base,neox", ROPES, ids=["plain", "pairs", "halves"])
@pytest.mark.parametrize("n", [1, 40, 129, 4000])
def test_rows_whose_every_score_is_minus_infinity(ctx, vk, n, base, neox, dtype):
    """Zeros, whatever the values are; with one finite score the row is that key's value. The queries of the last head are the
    smallest numbers of 16 bits, which a rotation makes smaller still."""
    H, hd, R = 4, 64, 16
    print(f"[no weight] {n} {base} {neox} {dtype.__name__}", flush=True)
    r = np.random.default_rng(n)
    q, cache, table = make_attention(r, [n, n], H, H, hd, R, dtype)
    q[0, :, H - 1] = np.sign(r.standard_normal((2, hd))) * 2.0 ** -24
    pos = np.arange(n)
    for b in range(2):
        qr = ref.rotate(q[0, b][None], [n - 1], base, neox)[0]
        for h in range(H):
            d = r.integers(0, hd, n)
            page, row = at(table, b, pos, R)
            cache[page, h, row, d] = -np.sign(qr[h, d]) * np.inf
            cache[page[n // 2], H + h, row[n // 2], 5] = np.inf
    page, row = at(table, 1, n // 3, R)
    cache[page, :, row] = (1.3 * r.standard_normal((2 * H, hd))).astype(dtype)
    at_half = at(table, 1, n // 2, R)
    cache[at_half[0], H:, at_half[1], 5] = 1  # a weight of 0 makes an infinite value undefined: none in this row
    got = run_attention(ctx, vk, q, cache, table, hd ** -0.5, base, neox)
    want = check(got, q, cache, table, hd ** -0.5, base, neox)
    assert not want[0].any() and np.array_equal(got[1].astype(np.float64), cache[page, H:, row].astype(np.float64))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("base", [0.0, 1e4], ids=["plain", "rotated"])
def test_infinite_queries(ctx, vk, base, dtype):
    """One infinite element: the rotation makes it two, and scores infinite of either sign. Keys that stand against both give a
    row without weight; others leave the head undefined."""
    H, hd, R, n = 2, 64, 16, 300
    r = np.random.default_rng(17)
    q, cache, table = make_attention(r, [n], H, H, hd, R, dtype)
    q[0, 0, :, 6] = np.inf
    c, s = np.cos((n - 1) * 1e4 ** (-6 / 64)), np.sin((n - 1) * 1e4 ** (-6 / 64))
    signs = (c, s) if base else (1, 0)
    page, row = at(table, 0, np.arange(n), R)
    for i, sign in enumerate(signs):
        if sign:
            cache[page, 0, row, 6 + i] = -np.sign(sign) * (0.25 + np.abs(cache[page, 0, row, 6 + i]))
    got = run_attention(ctx, vk, q, cache, table, 0.125, base, False)
    assert not got[0, 0].any() and np.isnan(got[0, 1]).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_infinite_values_under_small_weights(ctx, vk, dtype):
    """Weights down to 2^-100 of the largest are numbers of 32 bits: an infinite value under one is infinite."""
    hd, R, n = 64, 16, 400
    r = np.random.default_rng(23)
    q, cache, table = make_attention(r, [n] * 4, 2, 2, hd, R, dtype)
    q[..., :] = 0
    q[..., 0] = 1.0
    page = np.stack([at(table, b, np.arange(n), R)[0] for b in range(4)])
    row = np.arange(n) % R
    for b, drop in enumerate([20, 40, 60, 69]):  # 2^-29, 2^-58, 2^-87, 2^-99.5
        cache[page[b], 0, row, 0] = -drop
        cache[page[b, 7], 0, row[7], 0] = 0
        cache[page[b], 1, row, 0] = 0
        cache[page[b, 200], 2, row[200], 9] = np.inf
        cache[page[b, 3], 2, row[3], 10] = -np.inf
    got = run_attention(ctx, vk, q, cache, table, 1.0, 0.0, False)
    assert np.isposinf(got[:, 0, 9]).all() and np.isneginf(got[:, 0, 10]).all()
    check(got, q, cache, table, 1.0, 0.0, False)
