"""Edges of the operators of batched generation: sources that no call has written yet under stream capture, a table in place
whose first columns hold anything, penalties by quotients of any size, rotations as near as 32 bits allow, rows without a token,
and how many (sequence, key head) pairs share the GPU."""
import ctypes

import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import Bag, check_attention, make_attention, rows4, run_attention, table_step
from test_zz_no_alloc import _hip_runtime

pytestmark = pytest.mark.gpu

NONE = ref.NONE


@pytest.mark.parametrize("which", ["history", "rules", "mask"])
def test_adjust_logits_of_a_source_that_never_ran_is_refused_under_capture(ctx, vk, which):
    """History, rules or mask that an operator has yet to write have no memory: the call under capture is refused, makes
    none, though the context has a free piece of that size, and leaves the capture as it was."""
    print(f"[capture] {which}", flush=True)
    H, L = _hip_runtime(), vk.lib()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    vk.check("stream", L.vkllm_hip_context_stream(ctx.vp, ctypes.byref(stream)))
    B, V, width = 2, 100, {"history": 9, "rules": 6, "mask": 4}[which]
    with Bag(ctx) as bag:
        x = bag.put(np.linspace(-3, 3, B * V).reshape(1, 1, B, V).astype(np.float16))
        rules = np.zeros((B, 4), np.uint32)
        rules[:, 0] = np.float32(1).view(np.uint32)
        srcs = {"history": None, "rules": bag.put(rows4(rules)), "mask": None}
        never = ctx.tensor([1, 1, B, width], vk.U32, op=vk.OP_PAGE_TABLE, srcs=[bag.put(rows4(np.zeros((1, B))))],
                           params=vk.PageTableParams(16, 4))
        srcs[which] = never
        y = ctx.tensor([1, 1, B, V], vk.F16, op=vk.OP_ADJUST_LOGITS, srcs=[x, *srcs.values()])
        bag.made += [never, y]
        ctx.upload(y, np.zeros((1, 1, B, V), np.float16))
        ctx.free(ctx.tensor([1, 1, B, width], vk.U32))
        assert not never.contents.data.dev
        assert H.hipStreamBeginCapture(stream, 0) == 0
        rc = L.vkllm_op_adjust_logits_run(ctx.vp, ctx.cmds, y)
        end = H.hipStreamEndCapture(stream, ctypes.byref(graph))
        if graph.value:
            H.hipGraphDestroy(graph)
        assert rc == vk.ERR_ARGS and end == 0 and not never.contents.data.dev
        first = np.zeros((B, width), np.uint32)
        if which == "rules":
            first[:, 0] = np.float32(1).view(np.uint32)
        ctx.upload(never, rows4(first))
        vk.check("adjust_logits", ctx.run_op("adjust_logits", y))
        got = ctx.download(y)
        assert np.isneginf(got).all() if which == "mask" else np.array_equal(got, ctx.download(x))


@pytest.mark.parametrize("B,P,R,pages", [(1, 3, 16, 9), (5, 7, 16, 40), (70, 300, 4, 9000), (300, 600, 16, 70000)])
def test_page_table_in_place_over_anything(ctx, vk, B, P, R, pages):
    """A table in place needs no more of its first contents than a length of 0 in every row: whatever the columns hold, the
    first step leaves the pages of the rows that grew and nothing behind them, also in rows whose wanted length is over the
    table's width, and in those that do not fit."""
    print(f"[page_table] B={B} P={P} R={R} pages={pages}", flush=True)
    r = np.random.default_rng(B)
    old = r.integers(0, 1 << 32, (B, 1 + P), dtype=np.uint32)
    old[:, 1:][r.random((B, P)) < 0.5] = r.integers(0, pages)
    old[:, 0] = 0
    want = r.integers(0, P * R + 1, B)
    want[r.random(B) < 0.4] = P * R + 1 + r.integers(0, 1000)
    want[0] = P * R + 1
    for in_place in (True, False):
        got = table_step(ctx, vk, old, want, R, pages, in_place)
        assert np.array_equal(got, ref.page_table(old, want, R, pages)), in_place


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rep", [1.1, 1.3, 3.0, 1e-39, 2e-42, 3e38, 1.0 / 3.0], ids=str)
def test_penalties_are_quotients(ctx, vk, rep, dtype):
    """x / repetition and x * repetition as 32 bits round them, once (and once more to 16): also where 1 / repetition is no
    number of 32 bits."""
    print(f"[adjust_logits] repetition {rep} {dtype.__name__}", flush=True)
    B, V = 3, 4099
    r = np.random.default_rng(11)
    x = (r.standard_normal((1, 1, B, V)) * np.exp(r.uniform(-12, 4, (1, 1, B, V)))).astype(dtype)
    history = np.concatenate((np.full((B, 1), V), np.tile(np.arange(V), (B, 1))), 1)
    rules = np.zeros((B, 4), np.uint32)
    rules[:, 0] = np.float32(rep).view(np.uint32)
    with Bag(ctx) as bag:
        t = bag.op("adjust_logits", x.shape, vk.F16 if dtype == np.float16 else vk.F32, vk.OP_ADJUST_LOGITS,
                   [bag.put(x), bag.put(rows4(history)), bag.put(rows4(rules))])
        got = ctx.download(t)
    x32 = x.astype(np.float32)
    with np.errstate(over="ignore", under="ignore"):
        want = np.where(x32 > 0, x32 / np.float32(rep), x32 * np.float32(rep)).astype(dtype)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("neox", [False, True], ids=["pairs", "halves"])
def test_rotations_in_32_bits(ctx, vk, neox):
    """Rotated fp32 keys are as near to 64 bits as 32-bit arithmetic on the rounded cosine and sine comes, in the mean of
    squares over 2^18 pairs. An angle that is a 32-bit fraction of a turn is off by up to 2 pi 2^-26 more, which makes it 1.4
    times as much (in numpy); rounded cosines and sines that the fraction's rest corrects, which rounds them once more, 1.07. The
    bar lies between."""
    T, KV, hd, R = 512, 8, 128, 16
    print(f"[update_pages] rotations {neox}", flush=True)
    r = np.random.default_rng(41)
    k, v = (r.standard_normal((1, T, KV, hd)).astype(np.float32) for _ in range(2))
    positions = r.integers(0, 100000, T).astype(np.uint32)
    with Bag(ctx) as bag:
        t = bag.op("update_pages", (T // R, 2 * KV, R, hd), vk.F32, vk.OP_UPDATE_PAGES,
                   [bag.put(k), bag.put(v), bag.put(rows4(np.stack([np.arange(T), positions], 1)))],
                   vk.UpdatePagesParams(1e4, neox))
        got = ctx.download(t)
    got = got[np.arange(T) // R, :KV, np.arange(T) % R]
    angle = (positions.astype(np.float64)[:, None] * 1e4 ** (-np.arange(0, hd, 2) / hd))[:, None]
    c, s = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    a, b = (k[0][..., :hd // 2], k[0][..., hd // 2:]) if neox else (k[0][..., 0::2], k[0][..., 1::2])
    pair = c * a - s * b, s * a + c * b  # three roundings each
    near = np.concatenate(pair, -1) if neox else np.stack(pair, -1).reshape(T, KV, hd)
    want = ref.rotate(k[0], positions, 1e4, neox)
    rms = lambda e: float(np.sqrt((e.astype(np.float64) ** 2).mean()))  # noqa: E731
    print(f"  {rms(got - want):.3e}, nearest cosines and sines {rms(near - want):.3e}", flush=True)
    assert rms(got - want) <= 1.2 * rms(near - want)


def test_a_token_in_every_row(ctx, vk):
    """With counts of 1 in all rows token b is row b's, whichever rows have no sequence; those get no slot. With counts of 0 there
    the tokens behind move up."""
    table = np.array([[20, 4, 9], [0, NONE, NONE], [3, 7, NONE], [0, NONE, NONE], [16, 2, NONE]], np.uint32)
    lengths = table[:, 0]
    for counts, want in ((np.ones(5), [[9 * 16 + 3, 19], [NONE, 0], [7 * 16 + 2, 2], [NONE, 0], [2 * 16 + 15, 15]]),
                         (lengths > 0, [[9 * 16 + 3, 19], [7 * 16 + 2, 2], [2 * 16 + 15, 15], [NONE, 0], [NONE, 0]])):
        with Bag(ctx) as bag:
            t = bag.op("slot_map", (1, 1, 5, 2), vk.U32, vk.OP_SLOT_MAP,
                       [bag.put(rows4(table)), bag.put(rows4(lengths[None])), bag.put(rows4(counts[None]))], vk.SlotMapParams(16))
            assert ctx.download(t)[0, 0].tolist() == want


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("lengths,H,KV", [([8200], 8, 8), ([6400], 10, 10), ([6300], 11, 11), ([5600], 48, 12), ([3000, 2900], 24, 6),
                                          ([5600], 96, 12), ([2900], 120, 24), ([2800], 130, 26), ([2700, 0, 2600], 65, 13)],
                         ids=lambda v: str(v))
def test_rows_on_one_workgroup_a_cu(ctx, vk, lengths, H, KV, dtype):
    """Numbers of (sequence, key head) pairs at both sides of where rows of 128 dims go to half of the workgroups."""
    print(f"[paged_attn] {lengths} {H} {KV} {dtype.__name__}", flush=True)
    q, cache, table = make_attention(np.random.default_rng(H + KV), lengths, H, KV, 128, 16, dtype)
    got = run_attention(ctx, vk, q, cache, table, 128 ** -0.5, 1e4, True)
    check_attention(got, q, cache, table, 128 ** -0.5, 1e4, True)


def test_page_table_of_the_most_rows_and_pages(ctx, vk):
    """4096 rows and 524288 pages at once: the most that the kernel's LDS is asked for."""
    B, P, R, pages = 4096, 150, 16, 524288
    print(f"[page_table] B={B} P={P} pages={pages}", flush=True)
    r = np.random.default_rng(3)
    table = np.full((B, 1 + P), NONE, np.uint32)
    table[:, 0] = r.integers(0, P * R + 1, B)
    order, at = r.permutation(pages), 0
    for b in range(B):
        n = -(-int(table[b, 0]) // R)
        table[b, 1:1 + n] = order[at:at + n]
        at += n
    want = np.where(r.random(B) < 0.5, r.integers(0, P * R + 1, B), table[:, 0] + 1)
    want[7], want[8] = P * R + 5, 0
    new = ref.page_table(table, want, R, pages)
    for in_place in (False, True):
        assert np.array_equal(table_step(ctx, vk, table, want, R, pages, in_place), new), in_place


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_paged_attn_of_the_most_rows_and_heads(ctx, vk, dtype):
    """4096 rows of 16 heads of 256 dims on one key head: the most that the kernel's LDS is asked for."""
    print(f"[paged_attn] 4096 rows {dtype.__name__}", flush=True)
    r = np.random.default_rng(4)
    lengths = np.where(r.random(4096) < 0.9, 0, r.integers(1, 40, 4096))
    lengths[-1] = 300
    q, cache, table = make_attention(r, lengths.tolist(), 16, 1, 256, 16, dtype)
    got = run_attention(ctx, vk, q, cache, table, 1 / 16, 1e4, False)
    check_attention(got, q, cache, table, 1 / 16, 1e4, False)
    assert not got[lengths == 0].any()
