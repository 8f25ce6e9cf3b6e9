"""ADJUST_LOGITS against the rules in 64 bits, token by token (paged_ref.adjust): one rounding to the logits' type beside a
few fp32 roundoffs of the terms; masked places and untouched logits exactly."""
import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import Bag, half_step, rows4

pytestmark = pytest.mark.gpu


def make(r, B, V, T, N, dtype):
    x = (3 * r.standard_normal((B, V))).astype(dtype)
    history = r.integers(0, V, (B, 1 + T)).astype(np.uint32)
    if T:
        history[:, 1:][r.random((B, T)) < 0.4] = r.integers(0, V)  # one token again and again
        history[:, 1:][r.random((B, T)) < 0.05] = V                # and ids that the vocabulary does not have
        history[:, T] = 0xFFFFFFFF
    history[:, 0] = r.integers(0, T + 1, B)
    rules = np.zeros((B, 4 + 2 * N), np.uint32)
    rules[:, :3] = np.stack([r.uniform(0.5, 2, B), r.uniform(-1, 1, B), r.uniform(-1, 1, B)], 1).astype(np.float32).view(np.uint32)
    rules[:, 3] = r.integers(0, N + 1, B)
    rules[:, 4::2] = r.integers(0, min(V, 2 * N + 1), (B, N))      # several biases of one token
    rules[:, 5::2] = r.uniform(-5, 5, (B, N)).astype(np.float32).view(np.uint32)
    if N:
        rules[::3, 4] = V + 1
    mask = r.integers(0, 1 << 32, (B, -(-V // 32)), dtype=np.uint32)
    return x, history, rules, mask


def run(ctx, vk, x, history, rules, mask, pad=0):
    with Bag(ctx) as bag:
        srcs = [bag.view(rowsx(x), None, pad) if pad else bag.put(rowsx(x))]
        srcs += [None if a is None else bag.view(rows4(a), None, pad) if pad else bag.put(rows4(a)) for a in (history, rules, mask)]
        t = bag.op("adjust_logits", (1, 1, *x.shape), vk.F16 if x.dtype == np.float16 else vk.F32, vk.OP_ADJUST_LOGITS, srcs)
        return ctx.download(t)[0, 0]


def rowsx(x):
    return x.reshape(1, 1, *x.shape)


def check(got, x, history, rules, mask):
    want = ref.adjust(x, history, rules, mask)
    masked = np.isneginf(want)
    assert np.array_equal(np.isneginf(got), masked)
    terms = np.abs(x.astype(np.float64)) + np.abs(want)
    if rules is not None:
        r = np.abs(rules[:, :3].view(np.float32).astype(np.float64))
        n = 0 if history is None else np.minimum(history[:, 0], history.shape[1] - 1)
        scale = np.maximum(r[:, 0], 1 / r[:, 0])
        terms = terms * scale[:, None] + (r[:, 1] * n + r[:, 2] + 5)[:, None]
    tol = half_step(want, x.dtype.type) * (1 + 2.0 ** -10) + 6 * 2.0 ** -24 * terms
    with np.errstate(invalid="ignore"):
        d = np.abs(got.astype(np.float64) - want)
    assert (d[~masked] <= tol[~masked]).all()
    if history is None and rules is None:
        assert np.array_equal(got[~masked], x[~masked])


@pytest.mark.parametrize("pad", [0, 3], ids=["packed", "padded"])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("B,V,T,N", [(1, 1, 0, 0), (1, 7, 1, 1), (3, 31, 5, 2), (2, 32, 300, 9), (5, 33, 40, 40), (1, 32000, 128, 4),
                                     (2, 32001, 1000, 300), (7, 1000, 4097, 17), (4, 50257, 64, 1), (130, 9001, 33, 5),
                                     (300, 20000, 10, 3)])
def test_adjust_logits(ctx, vk, B, V, T, N, dtype, pad):
    print(f"[adjust_logits] B={B} V={V} T={T} N={N} {dtype.__name__} pad={pad}", flush=True)
    x, history, rules, mask = make(np.random.default_rng(V + T), B, V, T, N, dtype)
    for h, u, k in ((history, rules, mask), (None, rules, None), (history, rules, None), (None, None, mask), (None, None, None)):
        check(run(ctx, vk, x, h, u, k, pad), x, h, u, k)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("V,T,N", [(40000, 70000, 5), (40000, 20, 33000), (100, 65534, 3), (100, 65535, 3)])
def test_adjust_logits_past_16_bits(ctx, vk, V, T, N, dtype):
    """Histories and biases longer than a half word counts: one token used more than 65535 times."""
    print(f"[adjust_logits] V={V} T={T} N={N} {dtype.__name__}", flush=True)
    r = np.random.default_rng(N)
    x, history, rules, mask = make(r, 2, V, T, N, dtype)
    history[0] = 7 % V
    history[0, 0] = T
    rules[:, 1] = np.float32(1e-4).view(np.uint32)
    rules[:, 3] = N
    check(run(ctx, vk, x, history, rules, mask), x, history, rules, mask)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_adjust_logits_of_rows_that_nothing_is_left_of(ctx, vk, dtype):
    """All masked; NaN and infinities in masked places give -inf like any other; -inf logits stay; counts past a row end with it;
    rules that change nothing."""
    V, T = 100, 6
    x = np.linspace(-4, 4, 4 * V).reshape(4, V).astype(dtype)
    x[0, ::3], x[0, 1::3] = np.nan, np.inf
    x[1, 5], x[2, 6], x[1, 7] = np.nan, -np.inf, np.inf
    history = np.tile(np.array([T, 1, 5, 5, 6, 9, 200], np.uint32), (4, 1))
    history[3, 0] = 0xFFFFFFFF
    rules = np.zeros((4, 6), np.uint32)
    rules[:, :3] = np.array([1.0, 0.0, 0.0], np.float32).view(np.uint32)
    rules[3, :3] = np.array([2.0, 0.5, 0.25], np.float32).view(np.uint32)
    rules[3, 3], rules[3, 4] = 0xFFFFFFFF, 9
    rules[3, 5] = np.float32(1.5).view(np.uint32)
    mask = np.full((4, 4), 0xFFFFFFFF, np.uint32)
    mask[0] = 0
    mask[1, 0] &= ~np.uint32(1 << 5)
    got = run(ctx, vk, x, history, rules, mask)
    assert np.isneginf(got[0]).all()
    assert np.isneginf(got[1, 5]) and np.isposinf(got[1, 7]) and np.array_equal(np.delete(got[1], 5), np.delete(x[1], 5))
    assert np.array_equal(got[2], x[2])
    check(got[3:], x[3:], history[3:], rules[3:], mask[3:])


def test_arg_max_after_a_mask(ctx, vk):
    """The token that is chosen is one that the grammar allows."""
    r = np.random.default_rng(4)
    x, history, rules, mask = make(r, 6, 32000, 50, 8, np.float16)
    with Bag(ctx) as bag:
        srcs = [bag.put(rowsx(x))] + [bag.put(rows4(a)) for a in (history, rules, mask)]
        t = bag.op("adjust_logits", (1, 1, *x.shape), vk.F16, vk.OP_ADJUST_LOGITS, srcs)
        ids = ctx.download(bag.op("arg_max", (1, 1, 6, 1), vk.U32, vk.OP_ARG_MAX, [t])).reshape(6)
        y = ctx.download(t)[0, 0]
    assert ((mask[np.arange(6), ids // 32] >> (ids % 32).astype(np.uint32)) & 1).all()
    assert np.array_equal(y[np.arange(6), ids], y.max(1))
