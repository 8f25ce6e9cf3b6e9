"""What the operators over a paged cache refuse, without a GPU: their _init checks on descriptions of tensors (no memory
behind them), each wrong in one way."""
import ctypes

import pytest

OP = {"page_table": 12, "slot_map": 13, "update_pages": 14, "paged_attn": 15, "adjust_logits": 16}


class World:
    """A context without a device, and tensor structs of its own."""

    def __init__(self, vk):
        self.vk, self.keep = vk, []
        self.entries = (vk.Pipeline * 256)()
        self.context = vk.Context()
        self.context.pipelines = ctypes.cast(self.entries, ctypes.c_void_p)

    def tensor(self, shape, dtype, op=0, srcs=(), params=None):
        size = ctypes.sizeof(self.vk.Tensor)
        raw = ctypes.create_string_buffer(size + 64)
        t = ctypes.cast(raw, self.vk.TensorP)
        c = t.contents
        c.dtype, c.op = dtype, op
        c.shapes[:] = shape
        es = {self.vk.F32: 4, self.vk.F16: 2, self.vk.U32: 4, self.vk.I8: 1}[dtype]
        c.strides[:] = [shape[1] * shape[2] * shape[3] * es, shape[2] * shape[3] * es, shape[3] * es, es]
        c.bytes = shape[0] * c.strides[0]
        for i, s in enumerate(srcs):
            if s is not None:
                c.srcs[i] = s
        if params is not None:
            ctypes.memmove(ctypes.addressof(raw) + size, ctypes.byref(params), ctypes.sizeof(params))
        self.keep.append((raw, srcs))
        return t

    def init(self, op, t):
        p = ctypes.cast(ctypes.byref(self.context), ctypes.c_void_p)
        return getattr(self.vk.lib(), f"vkllm_op_{op}_init")(p, ctypes.c_void_p(16), t)


@pytest.fixture
def world(vk):
    return World(vk)


def page_table(w, shape=(1, 1, 3, 9), want=(1, 1, 1, 3), old=(1, 1, 3, 9), rows=16, pages=24, dtype=None, op=None):
    V = w.vk
    srcs = [w.tensor(want, V.U32)] + ([w.tensor(old, V.U32)] if old else [])
    return w.tensor(shape, dtype or V.U32, op or V.OP_PAGE_TABLE, srcs, V.PageTableParams(rows, pages))


@pytest.mark.parametrize("kw", [
    dict(want=(1, 1, 1, 4)), dict(want=(1, 1, 3, 1)), dict(old=(1, 1, 3, 8)), dict(shape=(1, 1, 3, 1), old=None),
    dict(shape=(1, 3, 1, 9), old=None), dict(rows=0), dict(pages=0), dict(pages=(512 << 10) + 1),
    dict(rows=1 << 20, pages=4096), dict(dtype=1), dict(op=13), dict(shape=(1, 1, 4097, 2), want=(1, 1, 1, 4097), old=None)],
    ids=str)
def test_page_table_refuses(vk, world, kw):
    assert world.init("page_table", page_table(world)) == vk.ERR_OK
    assert world.init("page_table", page_table(world, old=None)) == vk.ERR_OK
    assert world.init("page_table", page_table(world, pages=512 << 10)) == vk.ERR_OK
    assert world.init("page_table", page_table(world, **kw)) == vk.ERR_ARGS


def test_page_table_refuses_its_own_memory_and_missing_lengths(vk, world):
    t = page_table(world)
    view = world.tensor((1, 1, 3, 9), vk.U32, vk.OP_REF, [t])
    view.contents.data.is_ref = True
    t.contents.srcs[1] = view
    assert world.init("page_table", t) == vk.ERR_ARGS
    t = page_table(world)
    t.contents.srcs[0] = vk.TensorP()
    assert world.init("page_table", t) == vk.ERR_ARGS
    t = page_table(world)
    t.contents.strides[2] += 4  # rows of a wider tensor
    assert world.init("page_table", t) == vk.ERR_ARGS


def slot_map(w, shape=(1, 1, 7, 2), table=(1, 1, 3, 9), lengths=(1, 1, 1, 3), counts=(1, 1, 1, 3), rows=16, dtype=None):
    V = w.vk
    return w.tensor(shape, dtype or V.U32, V.OP_SLOT_MAP, [w.tensor(s, V.U32) for s in (table, lengths, counts)],
                    V.SlotMapParams(rows))


def test_slot_map_refuses_shared_memory(vk, world):
    for i in range(3):
        t = slot_map(world)
        view = world.tensor(tuple(t.contents.srcs[i].contents.shapes), vk.U32, vk.OP_REF, [t])
        view.contents.data.is_ref = True
        t.contents.srcs[i] = view
        assert world.init("slot_map", t) == vk.ERR_ARGS


@pytest.mark.parametrize("kw", [
    dict(shape=(1, 1, 7, 3)), dict(shape=(1, 7, 1, 2)), dict(table=(1, 1, 4, 9)), dict(lengths=(1, 1, 1, 2)),
    dict(counts=(1, 1, 3, 1)), dict(rows=0), dict(dtype=1), dict(table=(1, 1, 3, 1))], ids=str)
def test_slot_map_refuses(vk, world, kw):
    assert world.init("slot_map", slot_map(world)) == vk.ERR_OK
    assert world.init("slot_map", slot_map(world, **kw)) == vk.ERR_ARGS


def update_pages(w, cache=(24, 6, 16, 64), k=(1, 7, 3, 64), v=None, at=(1, 1, 7, 2), base=1e4, dtype=None, kd=None, vd=None):
    V = w.vk
    d = dtype or V.F16
    return w.tensor(cache, d, V.OP_UPDATE_PAGES,
                    [w.tensor(k, kd or d), w.tensor(v or k, vd or d), w.tensor(at, V.U32)], V.UpdatePagesParams(base, False))


@pytest.mark.parametrize("kw", [
    dict(cache=(24, 5, 16, 64)), dict(k=(1, 7, 4, 64)), dict(k=(1, 7, 3, 56)), dict(v=(1, 7, 2, 64)), dict(at=(1, 1, 6, 2)),
    dict(at=(1, 1, 7, 3)), dict(cache=(24, 6, 16, 60), k=(1, 7, 3, 60)), dict(cache=(24, 6, 16, 264), k=(1, 7, 3, 264)),
    dict(k=(2, 7, 3, 64)), dict(base=-1.0), dict(base=float("inf")), dict(base=float("nan")), dict(dtype=4), dict(kd=1),
    dict(vd=1)], ids=str)
def test_update_pages_refuses(vk, world, kw):
    for ok in (dict(), dict(base=0.0), dict(dtype=vk.F32), dict(cache=(24, 6, 5, 256), k=(1, 7, 3, 256))):
        assert world.init("update_pages", update_pages(world, **ok)) == vk.ERR_OK
    assert world.init("update_pages", update_pages(world, **kw)) == vk.ERR_ARGS


def test_update_pages_refuses_views_of_the_cache(vk, world):
    for i in range(3):
        t = update_pages(world)
        view = world.tensor(tuple(t.contents.srcs[i].contents.shapes), t.contents.srcs[i].contents.dtype, vk.OP_REF, [t])
        view.contents.data.is_ref = True
        t.contents.srcs[i] = view
        assert world.init("update_pages", t) == vk.ERR_ARGS
    t = update_pages(world)
    t.contents.strides[2] += 16  # rows with a gap
    assert world.init("update_pages", t) == vk.ERR_ARGS


def paged_attn(w, q=(1, 5, 6, 64), out=None, cache=(24, 6, 16, 64), table=(1, 1, 5, 9), scale=0.125, base=1e4, dtype=None,
               cd=None):
    V = w.vk
    d = dtype or V.F16
    return w.tensor(out or q, d, V.OP_PAGED_ATTN, [w.tensor(q, d), w.tensor(cache, cd or d), w.tensor(table, V.U32)],
                    V.PagedAttnParams(scale, base, False))


@pytest.mark.parametrize("kw", [
    dict(out=(1, 5, 6, 56)), dict(q=(2, 5, 6, 64)), dict(q=(1, 5, 7, 64)), dict(q=(1, 5, 2, 64)), dict(q=(1, 5, 6, 56)),
    dict(cache=(24, 6, 24, 64)), dict(cache=(24, 6, 8, 64)), dict(cache=(24, 3, 16, 64)), dict(table=(1, 1, 4, 9)),
    dict(table=(1, 1, 5, 1)), dict(q=(1, 5, 6, 60), cache=(24, 6, 16, 60)), dict(q=(1, 5, 6, 264), cache=(24, 6, 16, 264)),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(base=-2.0), dict(dtype=4), dict(cd=1),
    dict(q=(1, 4097, 6, 64), table=(1, 1, 4097, 9)), dict(cache=(2, 6, 65536, 64), table=(1, 1, 5, 32770))], ids=str)
def test_paged_attn_refuses(vk, world, kw):
    # a description that passes goes on to the workspace, which needs a device: only refusals are asked for here
    assert world.init("paged_attn", paged_attn(world, **kw)) == vk.ERR_ARGS


def test_paged_attn_refuses_shared_memory(vk, world):
    for i in range(3):
        t = paged_attn(world)
        view = world.tensor(tuple(t.contents.srcs[i].contents.shapes), t.contents.srcs[i].contents.dtype, vk.OP_REF, [t])
        view.contents.data.is_ref = True
        t.contents.srcs[i] = view
        assert world.init("paged_attn", t) == vk.ERR_ARGS


def adjust(w, x=(1, 1, 3, 100), out=None, history=(1, 1, 3, 9), rules=(1, 1, 3, 8), mask=(1, 1, 3, 4), dtype=None, xd=None,
           md=None):
    V = w.vk
    d = dtype or V.F16
    srcs = [w.tensor(x, xd or d)] + [w.tensor(s, V.U32) if s else None for s in (history, rules)]
    return w.tensor(out or x, d, V.OP_ADJUST_LOGITS, srcs + [w.tensor(mask, md or V.U32) if mask else None])


@pytest.mark.parametrize("kw", [
    dict(out=(1, 1, 3, 99)), dict(x=(1, 3, 1, 100)), dict(history=(1, 1, 2, 9)), dict(rules=None), dict(rules=(1, 1, 3, 3)),
    dict(rules=(1, 1, 3, 7)), dict(rules=(1, 1, 4, 8)), dict(mask=(1, 1, 3, 3)), dict(mask=(1, 1, 1, 4)), dict(dtype=4),
    dict(xd=1), dict(md=1), dict(x=(1, 1, 65536, 4), history=None, rules=None, mask=None)], ids=str)
def test_adjust_logits_refuses(vk, world, kw):
    for ok in (dict(), dict(history=None), dict(history=None, rules=None), dict(mask=None), dict(dtype=vk.F32),
               dict(history=None, rules=None, mask=None), dict(mask=(1, 1, 3, 5))):
        assert world.init("adjust_logits", adjust(world, **ok)) == vk.ERR_OK
    assert world.init("adjust_logits", adjust(world, **kw)) == vk.ERR_ARGS


def test_adjust_logits_refuses_shared_memory(vk, world):
    for i in range(4):
        t = adjust(world)
        view = world.tensor(tuple(t.contents.srcs[i].contents.shapes), t.contents.srcs[i].contents.dtype, vk.OP_REF, [t])
        view.contents.data.is_ref = True
        t.contents.srcs[i] = view
        assert world.init("adjust_logits", t) == vk.ERR_ARGS


def test_a_node_of_another_operator_and_missing_arguments(vk, world):
    make = {"page_table": page_table, "slot_map": slot_map, "update_pages": update_pages, "paged_attn": paged_attn,
            "adjust_logits": adjust}
    for op, fn in make.items():
        t = fn(world)
        t.contents.op = vk.OP_COPY
        assert world.init(op, t) == vk.ERR_ARGS
        t = fn(world)
        t.contents.srcs[0] = vk.TensorP()
        assert world.init(op, t) == vk.ERR_ARGS
        assert getattr(vk.lib(), f"vkllm_op_{op}_init")(None, None, t) == vk.ERR_ARGS
        assert vk.lib().vkllm_op_s(OP[op]).decode() == f"VKLLM_OP_{op.upper()}"
