"""The operators over a paged cache against their definitions in 64 bits (paged_ref.py): PAGE_TABLE, SLOT_MAP, UPDATE_PAGES,
PAGED_ATTN. Whole numbers are equal; values round once, to half a step of their type, beside what their fp32 sums may be off."""
import ctypes

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

NONE = ref.NONE


class Bag:
    """Tensors that are freed together."""

    def __init__(self, ctx):
        self.ctx, self.made = ctx, []

    def put(self, arr):
        self.made.append(self.ctx.tensor_from(arr))
        return self.made[-1]

    def view(self, arr, axes=None, pad=0):
        """arr on the device as a view: stored in the order `axes`, its last stored axis `pad` longer (filled with NaN)."""
        V = __import__("pyvkllm")
        axes = axes or (0, 1, 2, 3)
        stored = np.ascontiguousarray(np.transpose(arr, axes))
        wide = np.full((*stored.shape[:-1], stored.shape[-1] + pad), np.nan if arr.dtype.kind == "f" else 0x55555555, arr.dtype)
        wide[..., :stored.shape[-1]] = stored
        base = self.put(wide)
        t = V.TensorP()
        V.check("copy_ref", V.lib().vkllm_tensor_copy_ref(self.ctx.vp, base, ctypes.byref(t)))
        self.made.append(t)
        t.contents.shapes[3] = stored.shape[-1]
        back = [list(axes).index(i) for i in range(4)]
        V.check("permute", V.lib().vkllm_tensor_permute(self.ctx.vp, t, (ctypes.c_uint32 * 4)(*back)))
        assert tuple(t.contents.shapes) == arr.shape
        return t

    def op(self, name, shape, dtype, op, srcs, params=None, first=None):
        V = __import__("pyvkllm")
        t = self.ctx.tensor(list(shape), dtype, op=op, srcs=srcs, params=params)
        self.made.append(t)
        if first is not None:
            self.ctx.upload(t, first)
        V.check(name, self.ctx.run_op(name, t))
        return t

    def __enter__(self):
        return self

    def __exit__(self, *a):
        for t in reversed(self.made):
            self.ctx.free(t)


def rows4(a):
    return np.ascontiguousarray(a.astype(np.uint32)).reshape(1, 1, *a.shape)


# ---- tables and maps -----------------------------------------------------------------------------------------------
def table_step(ctx, vk, old, want, R, pages, in_place):
    with Bag(ctx) as bag:
        lengths = bag.put(rows4(want[None, :]))
        if in_place:
            t = bag.op("page_table", (1, 1, *old.shape), vk.U32, vk.OP_PAGE_TABLE, [lengths], vk.PageTableParams(R, pages),
                       first=old)
        else:
            t = bag.op("page_table", (1, 1, *old.shape), vk.U32, vk.OP_PAGE_TABLE, [lengths, bag.put(rows4(old))],
                       vk.PageTableParams(R, pages))
        return ctx.download(t)[0, 0]


@pytest.mark.parametrize("in_place", [False, True], ids=["new", "in_place"])
@pytest.mark.parametrize("B,P,R,pages", [(1, 1, 1, 1), (1, 4, 16, 3), (3, 5, 7, 11), (7, 9, 16, 31), (33, 40, 16, 32),
                                         (64, 70, 3, 2100), (257, 33, 16, 4097), (1025, 5, 32, 3000), (4096, 6, 1, 9000)])
def test_page_table_over_many_steps(ctx, vk, B, P, R, pages, in_place):
    """Sequences begin, grow, shrink and end; every second step asks for more than there is. Each step's table is the next
    step's first, so pages are neither lost nor held twice."""
    print(f"[page_table] B={B} P={P} R={R} pages={pages}", flush=True)
    r = np.random.default_rng(B + P)
    table = np.full((B, 1 + P), NONE, np.uint32)
    table[:, 0] = 0
    for step in range(6):
        old = table[:, 0].astype(np.int64)
        want = np.where(r.random(B) < 0.6, old + r.integers(0, R + 2, B), r.integers(0, P * R + 3, B))
        if step % 2 == 0:
            want = np.where(r.random(B) < 0.5, want // 3, want)
        want[r.random(B) < 0.15] = 0
        got = table_step(ctx, vk, table, want, R, pages, in_place)
        table = ref.page_table(table, want, R, pages)
        assert np.array_equal(got, table), f"step {step}"
        held = [int(i) for b in range(B) for i in table[b, 1:1 + -(-int(table[b, 0]) // R)]]
        assert len(set(held)) == len(held) and all(i < pages for i in held)


@pytest.mark.parametrize("pages", [131072, 524288])
def test_page_table_of_a_large_cache(ctx, vk, pages):
    """More free pages than the list holds at a time, from a fragmented pool, and one row that takes most of it."""
    print(f"[page_table] pages={pages}", flush=True)
    R, P = 16, pages - 3000
    r = np.random.default_rng(2)
    table = np.full((3, 1 + P), NONE, np.uint32)
    table[:, 0] = 0, 4000 * R - 3, 900 * R
    order = r.permutation(pages)
    table[1, 1:4001], table[2, 1:901] = order[:4000], order[4000:4900]
    want = np.array([(pages - 4250) * R - 5, 4000 * R + 40, 100 * R])
    assert np.array_equal(table_step(ctx, vk, table, want, R, pages, False), ref.page_table(table, want, R, pages))
    want[0] = P * R  # the first row's demand does not fit, and with it the second's
    want[1] = 4800 * R
    new = ref.page_table(table, want, R, pages)
    assert np.array_equal(table_step(ctx, vk, table, want, R, pages, True), new)


def test_page_table_with_shared_and_absent_pages(ctx, vk):
    """Two rows hold a prefix of the same pages; one lets go of it. Ids that the cache does not have, and a length past the
    row's end, are carried along."""
    R, pages = 16, 12
    table = np.array([[40, 3, 5, 7, NONE], [48, 3, 5, 8, NONE], [33, 99, 0xFFFFFFF0, 2, NONE], [1 << 30, 0, 1, 4, 6]],
                     np.uint32)
    for want in ([0, 48, 33, 64], [40, 64, 50, 10], [17, 0, 0, 1 << 31], [64, 64, 64, 64]):
        want = np.array(want)
        for in_place in (False, True):
            assert np.array_equal(table_step(ctx, vk, table, want, R, pages, in_place), ref.page_table(table, want, R, pages))


@pytest.mark.parametrize("B,T", [(1, 1), (1, 40), (5, 64), (256, 256), (256, 3000), (300, 77), (4096, 5000)])
def test_slot_map(ctx, vk, B, T):
    print(f"[slot_map] B={B} T={T}", flush=True)
    R, P = 16, 12
    r = np.random.default_rng(B + T)
    table = r.permutation(B * P).astype(np.uint32).reshape(B, P)
    lengths = r.integers(0, P * R + 1, B)
    counts = np.minimum(r.integers(0, max(2, 2 * T // B), B), lengths)
    counts[r.random(B) < 0.3] = 0
    held = np.where(r.random(B) < 0.2, lengths - counts, lengths)  # rows that could not grow
    if B > 4:
        counts[1], lengths[2], held[3] = lengths[1] + 7, 1 << 31, 1 << 31  # more new tokens than tokens; lengths past the table
        table[4, 0] = NONE
    table = np.concatenate((held[:, None].astype(np.uint32), table), 1)
    with Bag(ctx) as bag:
        t = bag.op("slot_map", (1, 1, T, 2), vk.U32, vk.OP_SLOT_MAP,
                   [bag.put(rows4(table)), bag.put(rows4(lengths[None])), bag.put(rows4(counts[None]))], vk.SlotMapParams(R))
        got = ctx.download(t)[0, 0]
    assert np.array_equal(got, ref.slot_map(table, lengths, counts, T, R))


def test_slot_map_of_counts_past_32_bits(ctx, vk):
    table = np.array([[20, 1, 2], [20, 3, 4], [20, 5, 6]], np.uint32)
    lengths, counts = np.array([20, 20, 20]), np.array([3, 0xFFFFFFFF, 0xFFFFFFFF])
    with Bag(ctx) as bag:
        t = bag.op("slot_map", (1, 1, 9, 2), vk.U32, vk.OP_SLOT_MAP,
                   [bag.put(rows4(table)), bag.put(rows4(lengths[None])), bag.put(rows4(counts[None]))], vk.SlotMapParams(16))
        got = ctx.download(t)[0, 0]
    assert np.array_equal(got[:3], [[33, 17], [34, 18], [35, 19]])
    assert np.array_equal(got[3:], [[NONE, 0]] * 6)


# ---- rows into pages -----------------------------------------------------------------------------------------------
def half_step(x, dtype):
    """Half the distance of neighbouring values of `dtype` at |x|."""
    info = np.finfo(dtype)
    return np.maximum(np.abs(x) * (info.eps / 2), float(info.smallest_subnormal) / 2)


ROWS = [  # T, KV, hd, R, pages, base, neox, view of k and v (axes, pad)
    (1, 32, 128, 16, 9, 1e4, False, None), (1, 1, 8, 1, 1, 1e4, True, None), (5, 6, 48, 16, 4, 1e4, False, None),
    (64, 8, 128, 64, 3, 1e4, True, None), (300, 2, 80, 48, 9, 5e5, True, None), (1500, 4, 64, 16, 101, 1e4, False, None),
    (33, 3, 256, 16, 5, 1e4, True, None), (33, 3, 256, 16, 5, 0.0, True, None), (17, 5, 40, 7, 6, 1e4, True, None),
    (17, 5, 40, 7, 6, 1e4, False, ((0, 2, 1, 3), 0)), (17, 5, 40, 7, 6, 1e4, True, ((0, 1, 2, 3), 3)),
    (9, 4, 24, 16, 2, 1e4, False, ((0, 3, 2, 1), 1)),
]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("case", ROWS, ids=str)
def test_update_pages(ctx, vk, case, dtype):
    T, KV, hd, R, pages, base, neox, how = case
    print(f"[update_pages] {case} {dtype.__name__}", flush=True)
    r = np.random.default_rng(T + hd)
    cache = r.standard_normal((pages, 2 * KV, R, hd)).astype(dtype)
    cache[0, 0, 0, 0] = np.nan
    k, v = (r.standard_normal((1, T, KV, hd)).astype(dtype) for _ in range(2))
    v[0, 0, 0, 0] = np.inf  # values are stored as they are
    n = min(T, pages * R - (pages * R > 1))
    slots = np.full(T, NONE, np.uint32)  # tokens without a row among them, and slots that the cache does not have
    slots[r.permutation(T)[:n]] = r.permutation(pages * R)[:n]
    if T > 3:
        slots[1], slots[2] = pages * R, NONE - 1
    positions = r.integers(0, 200000, T).astype(np.uint32)
    positions[0] = 0
    with Bag(ctx) as bag:
        put = (lambda a: bag.view(a, *how)) if how else bag.put
        srcs = [put(k), put(v), bag.put(rows4(np.stack([slots, positions], 1)))]
        t = bag.op("update_pages", cache.shape, vk.F16 if dtype == np.float16 else vk.F32, vk.OP_UPDATE_PAGES, srcs,
                   vk.UpdatePagesParams(base, neox), first=cache)
        got = ctx.download(t)
    live = slots < pages * R
    page, row = slots[live].astype(np.int64) // R, slots[live].astype(np.int64) % R
    new = got[page, :, row]
    assert np.array_equal(new[:, KV:], v[0][live], equal_nan=True)
    want = ref.rotate(k[0], positions, base, neox)[live]
    # a rotated element is a sum of two products: cos and sin (2 roundoffs each with the angle's), the products and the sum
    size = np.abs(k[0][live].astype(np.float64))
    pair = size + (np.roll(size, -hd // 2, -1) if neox else size.reshape(*size.shape[:-1], -1, 2)[..., ::-1].reshape(size.shape))
    tol = half_step(want, dtype) * (1 + 2.0 ** -10) + (6 * 2.0 ** -24 * pair if base else 0)
    assert (np.abs(new[:, :KV].astype(np.float64) - want) <= tol).all()
    kept = cache.copy()
    kept[page, :, row] = new
    assert np.array_equal(got.view(np.uint8), kept.view(np.uint8))  # every other row as it was, bit for bit


# ---- attention -----------------------------------------------------------------------------------------------------
def make_attention(r, lengths, H, KV, hd, R, dtype, spare=3, P=None):
    B = len(lengths)
    need = [-(-n // R) for n in lengths]
    P = P or max(1, *need)
    pages = sum(need) + spare
    order = r.permutation(pages)
    table = np.full((B, 1 + P), NONE, np.uint32)
    table[:, 0] = lengths
    cache = (1.3 * r.standard_normal((pages, 2 * KV, R, hd))).astype(dtype)
    used = np.zeros((pages, R), bool)
    at = 0
    for b in range(B):
        table[b, 1:1 + need[b]] = order[at:at + need[b]]
        at += need[b]
        pos = np.arange(lengths[b])
        used[table[b, 1 + pos // R], pos % R] = True
    # what lies past a sequence's end, and on pages of nobody: anything
    cache[~used.repeat(2 * KV, 0).reshape(pages, 2 * KV, R)] = r.choice(np.array([np.nan, np.inf, -np.inf], dtype))
    return (1.3 * r.standard_normal((1, B, H, hd))).astype(dtype), cache, table


def run_attention(ctx, vk, q, cache, table, scale, base, neox, view=None):
    dt = vk.F16 if q.dtype == np.float16 else vk.F32
    with Bag(ctx) as bag:
        srcs = [bag.view(q, *view) if view else bag.put(q), bag.put(cache), bag.put(rows4(table))]
        t = bag.op("paged_attn", q.shape, dt, vk.OP_PAGED_ATTN, srcs, vk.PagedAttnParams(scale, base, neox),
                   first=np.full(q.shape, np.nan, q.dtype))
        got = ctx.download(t)
        vk.check("paged_attn", ctx.run_op("paged_attn", t))
        again = ctx.download(t)
    assert np.array_equal(got.view(np.uint8), again.view(np.uint8))  # the split and the join leave nothing to chance
    return got[0]


def check_attention(got, q, cache, table, scale, base, neox):
    want, off = ref.attention(q[0], cache, table, scale, base, neox)
    d = np.abs(got.astype(np.float64) - want)
    tol = half_step(want, q.dtype.type) * (1 + 2.0 ** -10) + off
    worst = np.unravel_index((d - tol).argmax(), d.shape)
    assert (d <= tol).all(), (worst, got[worst], want[worst], tol[worst])


ATTN = [  # lengths, H, KV, hd, R, base, neox, view
    ([1], 1, 1, 8, 16, 0.0, False, None),
    ([200], 6, 6, 48, 16, 1e4, False, None),
    ([0], 6, 6, 48, 16, 1e4, False, None),
    ([15, 16, 17, 0, 31, 32, 33, 1], 8, 2, 64, 16, 1e4, True, None),
    ([127, 128, 129, 63, 64, 65, 255, 257], 4, 4, 128, 16, 1e4, False, None),
    ([0, 0, 0, 500, 0, 1, 0], 32, 8, 128, 48, 1e4, True, None),
    ([1000, 3, 77], 16, 1, 128, 32, 1e4, True, None),
    ([513, 90], 34, 2, 64, 16, 1e4, False, None),           # 17 query heads to a key head: a tile of 16 and one of 1
    ([300, 0, 41], 64, 2, 80, 64, 5e5, True, None),         # two full tiles
    ([700, 129], 10, 2, 96, 16, 0.0, False, None),
    ([333, 1], 7, 1, 24, 128, 1e4, True, None),
    ([400, 401, 17], 4, 2, 136, 16, 1e4, True, None),
    ([900, 35], 8, 4, 256, 16, 1e4, False, None),
    ([260, 2], 40, 40, 128, 16, 1e4, False, None),
    ([50, 60, 70], 6, 3, 48, 16, 1e4, False, ((0, 2, 1, 3), 0)),   # queries in other orders, in rows of a wider tensor
    ([50, 60, 70], 6, 3, 48, 16, 1e4, True, ((0, 1, 2, 3), 5)),
    ([50, 60, 70], 6, 3, 48, 16, 1e4, True, ((0, 3, 2, 1), 1)),
    ([20000], 4, 1, 128, 64, 1e4, True, None),              # split over many workgroups
    ([9000, 1, 0, 12345], 8, 8, 64, 16, 1e4, False, None),
    ([3] * 300 + [0] * 20 + [400] * 5, 4, 2, 64, 16, 1e4, False, None),  # more rows than threads
    ([60000, 5], 16, 1, 64, 32, 1e4, False, None),          # joined over three levels, 16 heads a part
    ([50000, 0, 30], 1, 1, 128, 16, 1e4, True, None),       # and with several threads to the same dims
    ([700] * 65 + [0, 3000], 6, 3, 48, 16, 1e4, False, None),  # several rows to a workgroup, starts and ends counted
    # joins in which 8, 4, 2 lanes and one thread have four dims, and a thread eight
    ([7000], 2, 1, 16, 16, 1e4, True, None),
    ([6000, 1], 3, 1, 72, 32, 1e4, False, None),
    ([8000], 4, 1, 64, 16, 1e4, False, None),
    ([5000], 10, 2, 96, 16, 1e4, True, None),
    ([9000, 0], 9, 1, 128, 64, 1e4, False, None),
    ([4000, 10], 5, 1, 256, 16, 1e4, True, None),
    ([3000], 12, 1, 200, 16, 1e4, False, None),
    ([30000], 11, 1, 120, 64, 0.0, False, None),
    # long rows of 128 dims: a workgroup per CU, with and without starts counted, and more rows than lanes
    ([1100, 1080], 32, 32, 128, 16, 1e4, True, None),
    ([1500, 0, 1] + [1490] * 23, 16, 8, 128, 64, 1e4, False, None),
    ([900] * 68 + [0, 790, 1], 4, 2, 128, 16, 1e4, True, None),
    ([70000, 3], 8, 4, 128, 16, 1e4, True, None),
]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: f"{len(c[0])}x{c[0][0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{c[6]}-{c[7]}")
def test_paged_attn(ctx, vk, case, dtype):
    lengths, H, KV, hd, R, base, neox, view = case
    print(f"[paged_attn] {lengths[:8]} {case[1:]} {dtype.__name__}", flush=True)
    r = np.random.default_rng(sum(lengths) + H + hd)
    q, cache, table = make_attention(r, lengths, H, KV, hd, R, dtype)
    scale = hd ** -0.5
    got = run_attention(ctx, vk, q, cache, table, scale, base, neox, view)
    check_attention(got, q, cache, table, scale, base, neox)
    assert not got[np.array(lengths) == 0].any()


def test_paged_attn_of_4096_rows(ctx, vk):
    r = np.random.default_rng(1)
    lengths = r.integers(0, 20, 4096).tolist()
    q, cache, table = make_attention(r, lengths, 2, 1, 16, 16, np.float16)
    got = run_attention(ctx, vk, q, cache, table, 0.25, 1e4, False)
    check_attention(got, q, cache, table, 0.25, 1e4, False)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_paged_attn_with_bad_tables(ctx, vk, dtype):
    """Pages that the cache does not have (at the start, in the middle, at the end of a tile and of the row, all of them)
    count as absent; a length past the table's columns ends with them."""
    r = np.random.default_rng(7)
    q, cache, table = make_attention(r, [100, 250, 64, 33, 96, 200], 8, 4, 64, 16, dtype, P=16)
    pages = cache.shape[0]
    table[0, 1], table[1, 5], table[1, 6], table[1, 16] = NONE, pages, NONE, 1 << 31
    table[2, 4], table[3, 1:4] = pages + 1, NONE
    table[4, 0] = 0xFFFFFFFF
    table[4, 7:] = table[5, 1:11]
    cache[:] = (1.3 * r.standard_normal(cache.shape)).astype(dtype)  # row 4 reads rows past an end: nothing but numbers
    got = run_attention(ctx, vk, q, cache, table, 0.125, 1e4, False)
    check_attention(got, q, cache, table, 0.125, 1e4, False)
    assert not got[3].any()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_paged_attn_of_extreme_scores(ctx, vk, dtype):
    """One key far above the others (first, last, in the middle), scores that climb from tile to tile (every step rescales),
    scores all alike, of both signs, and a heavy tail of small weights under one large one."""
    hd, R, n = 64, 16, 3000
    r = np.random.default_rng(3)
    q, cache, table = make_attention(r, [n] * 7, 2, 2, hd, R, dtype)
    q[..., :] = 0
    q[..., 0] = 1.0
    pos = np.arange(n)
    for b, s in enumerate([np.where(pos == 0, 60.0, 0), np.where(pos == n - 1, 60.0, 0), np.where(pos == 1500, 300.0, 0),
                           pos * 0.05, -pos * 0.05, np.full(n, -200.0), np.where(pos == 7, 17.0, 0.0)]):
        page = table[b, 1 + pos // R]
        cache[page, 0, pos % R, 0] = s
        cache[page, 1, pos % R, 0] = -s
    got = run_attention(ctx, vk, q, cache, table, 1.0, 0.0, False)
    check_attention(got, q, cache, table, 1.0, 0.0, False)


def test_paged_attn_of_infinities(ctx, vk):
    """An infinite or undefined score makes its heads undefined, as the formula does, and no others; a row whose every score is
    -inf has no weight and is zero."""
    r = np.random.default_rng(5)
    q, cache, table = make_attention(r, [200, 200, 200, 200], 2, 2, 64, 16, np.float16)
    q[..., 0] = 1.0
    page = lambda b, pos: (table[b, 1 + pos // 16], pos % 16)  # noqa: E731
    p, i = page(0, 77)
    cache[p, 0, i, 0] = np.inf
    p, i = page(1, 5)
    cache[p, 1, i, 3] = np.nan
    pos = np.arange(200)
    cache[table[2, 1 + pos // 16], 0, pos % 16, 0] = -np.inf
    got = run_attention(ctx, vk, q, cache, table, 0.125, 0.0, False)
    assert np.isnan(got[0, 0]).all() and np.isnan(got[1, 1]).all() and not got[2, 0].any()
    sane = cache.copy()
    sane[~np.isfinite(sane)] = 0
    want, off = ref.attention(q[0], sane, table, 0.125, 0.0, False)
    for b, h in ((0, 1), (1, 0), (2, 1), (3, 0), (3, 1)):
        assert (np.abs(got[b, h] - want[b, h]) <= half_step(want[b, h], np.float16) * 1.001 + off[b, h]).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_paged_attn_of_an_undefined_query(ctx, vk, dtype):
    """A query that is not a number makes its head undefined, also where parts of the row are joined, and no other."""
    r = np.random.default_rng(6)
    q, cache, table = make_attention(r, [12000, 90], 4, 2, 64, 16, dtype)
    q[0, :, 2, 5] = np.nan
    got = run_attention(ctx, vk, q, cache, table, 0.125, 1e4, False)
    assert np.isnan(got[:, 2]).all()
    q[0, :, 2, 5] = 0
    want, off = ref.attention(q[0], cache, table, 0.125, 1e4, False)
    for h in (0, 1, 3):
        assert (np.abs(got[:, h] - want[:, h]) <= half_step(want[:, h], dtype) * 1.001 + off[:, h]).all()


def test_paged_attn_into_a_permuted_tensor(ctx, vk):
    """The result's own order of memory is another one: [H, B, hd] seen as [B, H, hd]."""
    r = np.random.default_rng(12)
    q, cache, table = make_attention(r, [40, 0, 300], 6, 2, 64, 16, np.float16)
    with Bag(ctx) as bag:
        t = ctx.tensor([1, 6, 3, 64], vk.F16, op=vk.OP_PAGED_ATTN, srcs=[bag.put(q), bag.put(cache), bag.put(rows4(table))],
                       params=vk.PagedAttnParams(0.125, 1e4, False))
        bag.made.append(t)
        vk.check("permute", vk.lib().vkllm_tensor_permute(ctx.vp, t, (ctypes.c_uint32 * 4)(0, 2, 1, 3)))
        vk.check("paged_attn", ctx.run_op("paged_attn", t))
        got = ctx.download(t)[0]
    check_attention(got, q, cache, table, 0.125, 1e4, False)


def test_paged_attn_past_32_bit_offsets(ctx, vk):
    """A cache of nearly 4 GiB, the most that a tensor holds: the pages in use lie at its end, past 2^31 bytes."""
    R, KV, hd = 64, 8, 128
    pages = ((1 << 32) - 256) // (2 * KV * R * hd * 2)
    r = np.random.default_rng(9)
    q, small, table = make_attention(r, [300, 64], 16, KV, hd, R, np.float16, spare=1)
    cache = ctx.tensor([pages, 2 * KV, R, hd], vk.F16)
    with Bag(ctx) as bag:
        bag.made.append(cache)
        first = pages - small.shape[0]
        assert first * 2 * KV * R * hd * 2 > 1 << 31
        part = ctx.tensor_from(small)
        bag.made.append(part)
        hip = ctypes.CDLL(sorted({line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64.so" in line})[0])
        hip.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
        assert hip.hipMemcpy(cache.contents.data.dev + first * 2 * KV * R * hd * 2, part.contents.data.dev, small.nbytes, 3) == 0
        moved = table.copy()
        moved[:, 1:][table[:, 1:] != NONE] += first
        t = bag.op("paged_attn", q.shape, vk.F16, vk.OP_PAGED_ATTN, [bag.put(q), cache, bag.put(rows4(moved))],
                   vk.PagedAttnParams(0.1, 1e4, True))
        got = ctx.download(t)[0]
        check_attention(got, q, small, table, 0.1, 1e4, True)
        # and rows written there
        k, v = (r.standard_normal((1, 3, KV, hd)).astype(np.float16) for _ in range(2))
        slots = np.array([pages * R - 1, pages * R, (first + 1) * R + 5], np.uint32)
        cache.contents.op = vk.OP_UPDATE_PAGES
        for i, s in enumerate((bag.put(k), bag.put(v), bag.put(rows4(np.stack([slots, slots], 1))))):
            cache.contents.srcs[i] = s
        vk.check("update_pages", ctx.run_op("update_pages", cache))  # no rotation: its parameters are zeros
        assert hip.hipMemcpy(part.contents.data.dev, cache.contents.data.dev + first * 2 * KV * R * hd * 2, small.nbytes, 3) == 0
        got = ctx.download(part).reshape(small.shape)
    want = small.copy()
    want[-1, :KV, R - 1], want[-1, KV:, R - 1] = k[0, 0], v[0, 0]
    want[1, :KV, 5], want[1, KV:, 5] = k[0, 2], v[0, 2]
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))


def test_tables_and_lists_that_are_views(ctx, vk):
    """A table in rows of a wider tensor, and lengths and counts that are columns of others: what lies beside them is not read."""
    r = np.random.default_rng(31)
    R, KV, H, hd = 16, 2, 4, 64
    lengths = [70, 0, 33, 129, 1]
    q, cache, table = make_attention(r, lengths, H, KV, hd, R, np.float16)
    B, pages = len(lengths), cache.shape[0]
    want = np.array([75, 17, 0, 129, 64])
    counts = np.array([5, 17, 0, 1, 63])
    with Bag(ctx) as bag:
        def column(values):
            return bag.view(values.astype(np.uint32).reshape(1, 1, 1, B), (0, 1, 3, 2), 6)

        wide = bag.view(rows4(table), None, 7)
        assert wide.contents.strides[2] == 4 * (table.shape[1] + 7) and column(want).contents.strides[3] == 28
        out = bag.op("paged_attn", q.shape, vk.F16, vk.OP_PAGED_ATTN, [bag.put(q), bag.put(cache), wide],
                     vk.PagedAttnParams(0.125, 1e4, True))
        check_attention(ctx.download(out)[0], q, cache, table, 0.125, 1e4, True)
        grown = bag.op("page_table", (1, 1, *table.shape), vk.U32, vk.OP_PAGE_TABLE, [column(want), wide],
                       vk.PageTableParams(R, pages + 20))
        new = ref.page_table(table, want, R, pages + 20)
        assert np.array_equal(ctx.download(grown)[0, 0], new)
        T = int(counts.sum())
        slots = bag.op("slot_map", (1, 1, T, 2), vk.U32, vk.OP_SLOT_MAP,
                       [bag.view(rows4(new), None, 3), column(want), column(counts)], vk.SlotMapParams(R))
        assert np.array_equal(ctx.download(slots)[0, 0], ref.slot_map(new, want, counts, T, R))
