"""Batched generation with the operators over a paged cache, as a program would run it: one graph a step on the weights of a
loaded model, sequences that join, end and reuse rows and pages. Each sequence's logits are those of the model's forward pass in
numpy, and those of the framework's own one-sequence token loop on the same tokens up to position head_dim - 2: with as many
cached positions as head dims the API's shape rule reads V as [N, K], transposed, so from position head_dim - 1 on the
token loop's cache is another one (tests/test_matmul_batched_gpu.py has that rule: N == K, B in its own order by shape)."""
import ctypes

import numpy as np
import pytest

from paged_ref import attention, rotate
from test_paged_gpu import Bag, rows4
from test_zz_no_alloc import _hip_runtime

pytestmark = pytest.mark.gpu

ROWS, COLUMNS, PAGE, PAGES, HISTORY = 4, 8, 16, 20, 96


class Server:
    """The graph of one step for ROWS sequences: embedding to arg max."""

    def __init__(self, ctx, vk, model):
        self.ctx, self.vk, self.L, self.made = ctx, vk, vk.lib(), []
        m, w = model.meta, model.m.weights
        D, H, V = m.embedding_length, m.head_count, m.vocab_size
        hd = D // H
        B = ROWS
        self.lengths, self.counts, self.tokens = (self.input((1, 1, 1, B), vk.U32) for _ in range(3))
        self.history, self.rules, self.mask = (self.input((1, 1, B, n), vk.U32) for n in (1 + HISTORY, 8, -(-V // 32)))
        self.table = self.op(vk.OP_PAGE_TABLE, (1, 1, B, 1 + COLUMNS), [self.lengths], vk.PageTableParams(PAGE, PAGES), vk.U32)
        ctx.upload(self.table, np.zeros((B, 1 + COLUMNS), np.uint32))
        at = self.op(vk.OP_SLOT_MAP, (1, 1, B, 2), [self.table, self.lengths, self.counts], vk.SlotMapParams(PAGE), vk.U32)
        x = self.op(vk.OP_EMBEDDING, (1, 1, B, D), [self.tokens, w.tok_embed_weights], ctypes.c_uint32(0))
        rms = vk.RmsnormParams(2.0, m.layer_norm_rms_epsilon)
        plain = vk.MatmulParams(1.0, 0)
        base = m.rope_freq_base
        self.caches = []
        for i in range(m.block_count):
            b = w.blocks.contents.data[i].contents
            n = self.op(vk.OP_RMSNORM, (1, 1, B, D), [x, b.attn_norm_weight], rms)
            q, k, v = (self.heads(self.op(vk.OP_MATMUL, (1, 1, B, D), [n, wt], plain), (1, B, H, hd)) for wt in (b.WQ, b.WK, b.WV))
            cache = self.op(vk.OP_UPDATE_PAGES, (PAGES, 2 * H, PAGE, hd), [k, v, at], vk.UpdatePagesParams(base, False))
            ctx.upload(cache, np.full((PAGES, 2 * H, PAGE, hd), np.nan, np.float16))
            self.caches.append(cache)
            o = self.op(vk.OP_PAGED_ATTN, (1, B, H, hd), [q, cache, self.table], vk.PagedAttnParams(hd ** -0.5, base, False))
            o = self.op(vk.OP_MATMUL, (1, 1, B, D), [self.heads(o, (1, 1, B, D)), b.WO], plain)
            x = self.op(vk.OP_BIN, (1, 1, B, D), [x, o], ctypes.c_int32(0))
            n = self.op(vk.OP_RMSNORM, (1, 1, B, D), [x, b.ffn_norm_weight], rms)
            u = self.op(vk.OP_FFN_UP_AND_GATE, (1, 1, B, b.WU.contents.shapes[2]), [n, b.WU, b.WG])
            x = self.op(vk.OP_BIN, (1, 1, B, D), [x, self.op(vk.OP_MATMUL, (1, 1, B, D), [u, b.WD], plain)], ctypes.c_int32(0))
        n = self.op(vk.OP_RMSNORM, (1, 1, B, D), [x, w.output_norm_weight], rms)
        self.raw = self.op(vk.OP_MATMUL, (1, 1, B, V), [n, w.output_weight], plain)
        self.logits = self.op(vk.OP_ADJUST_LOGITS, (1, 1, B, V), [self.raw, self.history, self.rules, self.mask])
        self.ids = self.op(vk.OP_ARG_MAX, (1, 1, B, 1), [self.logits], None, vk.U32)
        self.graph = ctypes.POINTER(vk.Graph)()
        vk.check("graph_new", self.L.vkllm_graph_new(ctx.vp, ctypes.byref(self.graph)))
        vk.check("set_output", self.L.vkllm_graph_set_output(ctx.vp, self.graph, self.ids))
        vk.check("graph_init", self.L.vkllm_graph_init(ctx.vp, self.graph))
        ctx.upload(self.rules, np.tile(np.array([1, 0, 0, 0, 0, 0, 0, 0], np.float32).view(np.uint32), (B, 1)))
        ctx.upload(self.mask, np.full((B, -(-V // 32)), 0xFFFFFFFF, np.uint32))
        ctx.upload(self.history, np.zeros((B, 1 + HISTORY), np.uint32))

    def input(self, shape, dtype):
        self.made.append(self.ctx.tensor(list(shape), dtype))
        return self.made[-1]

    def op(self, op, shape, srcs, params=None, dtype=None):
        self.made.append(self.ctx.tensor(list(shape), dtype or self.vk.F16, op=op, srcs=srcs, params=params))
        return self.made[-1]

    def heads(self, t, shape):
        r = self.vk.TensorP()
        self.vk.check("copy_ref", self.L.vkllm_tensor_copy_ref(self.ctx.vp, t, ctypes.byref(r)))
        self.vk.check("reshape", self.L.vkllm_tensor_reshape(self.ctx.vp, r, (ctypes.c_uint32 * 4)(*shape)))
        self.made.append(r)
        return r

    def put(self, lengths, counts, tokens):
        for t, a in ((self.lengths, lengths), (self.counts, counts), (self.tokens, tokens)):
            self.ctx.upload(t, np.asarray(a, np.uint32))

    def step(self, lengths, counts, tokens):
        self.put(lengths, counts, tokens)
        self.vk.check("graph_run", self.L.vkllm_graph_run(self.ctx.vp, self.graph))
        return self.ctx.download(self.raw)[0, 0], self.ctx.download(self.ids).reshape(-1)

    def close(self):
        self.L.vkllm_graph_free(self.ctx.vp, self.graph)
        for t in reversed(self.made):
            self.ctx.free(t)


@pytest.fixture(scope="module")
def tiny(ctx, vk, tiny_gguf):
    model = vk.Model(ctx, path=tiny_gguf)
    yield model
    model.close()


def forward(ctx, model, toks):
    """Logits [n, V] of the model after each of `toks`, without its fp16 roundings."""
    m, w = model.meta, model.m.weights
    D, H, n = m.embedding_length, m.head_count, len(toks)
    hd = D // H
    get = lambda t: ctx.download(t).astype(np.float32)[0, 0]  # noqa: E731
    rms = lambda x, wt: x * get(wt)[0] / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + m.layer_norm_rms_epsilon)  # noqa: E731
    x = get(w.tok_embed_weights)[toks]
    later = np.triu(np.ones((n, n), bool), 1)
    for i in range(m.block_count):
        b = w.blocks.contents.data[i].contents
        a = rms(x, b.attn_norm_weight)
        q, k, v = ((a @ get(wt).T).reshape(n, H, hd) for wt in (b.WQ, b.WK, b.WV))
        q, k = (rotate(t, np.arange(n), m.rope_freq_base, False) for t in (q, k))
        s = np.einsum("shd,thd->hst", q, k) / np.sqrt(hd)
        p = np.exp(np.where(later, -np.inf, s - s.max(-1, keepdims=True)))
        o = np.einsum("hst,thd->shd", p / p.sum(-1, keepdims=True), v).reshape(n, D)
        x = x + o @ get(b.WO).T
        a = rms(x, b.ffn_norm_weight)
        gate = a @ get(b.WG).T
        x = x + ((a @ get(b.WU).T) * gate / (1 + np.exp(-gate))) @ get(b.WD).T
    return rms(x, w.output_norm_weight) @ get(w.output_weight).T


def test_batched_loop_matches_the_token_loop(ctx, vk, tiny):
    r = np.random.default_rng(0)
    # (row, first step, tokens): rows are used again after a sequence's end, and lengths pass several pages
    plan = [(0, 0, 60), (1, 3, 20), (2, 5, 33), (1, 30, 25), (3, 11, 2), (3, 20, 17), (0, 62, 3)]
    seqs = [dict(row=row, start=start, toks=r.integers(0, 32000, n).astype(np.uint32), got=[]) for row, start, n in plan]
    srv = Server(ctx, vk, tiny)
    try:
        for step in range(66):
            print(f"[paged loop] step {step}", flush=True) if step % 10 == 0 else None
            lengths, counts, tokens = (np.zeros(ROWS, np.uint32) for _ in range(3))
            alive = [s for s in seqs if s["start"] <= step < s["start"] + len(s["toks"])]
            for s in alive:
                i = step - s["start"]
                lengths[s["row"]], counts[s["row"]], tokens[s["row"]] = i + 1, 1, s["toks"][i]
            # SLOT_MAP packs new tokens in row order: the batch's rows are those of the live sequences, in order
            order = [b for b in range(ROWS) if counts[b]]
            if order != list(range(len(order))):  # a row without a sequence takes a token all the same, to keep rows in step
                counts[:] = 1
            raw, _ = srv.step(lengths, counts, tokens)
            table = ctx.download(srv.table)[0, 0]
            assert np.array_equal(table[:, 0], lengths)
            for s in alive:
                s["got"].append(raw[s["row"]].astype(np.float32))
    finally:
        srv.close()
    for s in seqs:
        print(f"[paged loop] sequence of row {s['row']} from step {s['start']}", flush=True)
        # some 8 roundings of 2^-11 a layer, independent: sqrt(8 * 6) * 2^-11 / sqrt(3) = 2e-3 of a logit's deviation, 0.34
        # (sqrt(288) * 0.02); five deviations over a million logits are 3.4e-3, and half a step of a logit below 4 is 1e-3
        err = np.abs(np.stack(s["got"]) - forward(ctx, tiny, s["toks"])).max(1)
        print(f"[paged loop] max|dlogit| {err.max():.3g} against the forward pass", flush=True)
        assert err.max() <= 2e-2, (s["row"], int(err.argmax()), err.max())  # the bar of the token loop's own tests
        for i, tok in enumerate(s["toks"][:tiny.meta.embedding_length // tiny.meta.head_count - 1]):
            tiny.step(np.array([tok], np.uint32), i)
            want = tiny.last_logits(1)[0].astype(np.float32)
            err = float(np.abs(s["got"][i] - want).max())
            assert err <= 2e-2, (s["row"], i, err)


def test_a_captured_step_replays(ctx, vk, tiny):
    """The paged operators of one step recorded into a hipGraph and replayed, with eager work on the same context between the
    replays: each replay's table, cache rows, attention and logits are those of an eager run."""
    H, L = _hip_runtime(), vk.lib()
    stream, graph, exe = (ctypes.c_void_p() for _ in range(3))
    vk.check("stream", L.vkllm_hip_context_stream(ctx.vp, ctypes.byref(stream)))
    r = np.random.default_rng(8)
    B, P, R, KV, G, hd, V = 3, 40, 16, 2, 4, 64, 5000
    pages = B * P
    f16 = lambda *s: r.standard_normal(s).astype(np.float16)  # noqa: E731
    with Bag(ctx) as bag:
        lengths, counts = bag.put(rows4(np.ones((1, B)))), bag.put(rows4(np.ones((1, B))))
        zero = np.zeros((B, 1 + P), np.uint32)
        k, v, q, x = bag.put(f16(1, B, KV, hd)), bag.put(f16(1, B, KV, hd)), bag.put(f16(1, B, KV * G, hd)), bag.put(f16(1, 1, B, V))
        history = bag.put(rows4(r.integers(0, V, (B, 9))))
        rules = np.zeros((B, 4), np.uint32)
        rules[:, :3] = np.array([1.5, 0.25, 0.5], np.float32).view(np.uint32)
        rules = bag.put(rows4(rules))
        first = f16(pages, 2 * KV, R, hd)
        ops = []

        def op(name, code, shape, dtype, srcs, params=None, start=None):
            t = ctx.tensor(list(shape), dtype, op=code, srcs=srcs, params=params)
            bag.made.append(t)
            if start is not None:
                ctx.upload(t, start)
            ops.append((name, t))
            return t

        table = op("page_table", vk.OP_PAGE_TABLE, (1, 1, B, 1 + P), vk.U32, [lengths], vk.PageTableParams(R, pages), zero)
        at = op("slot_map", vk.OP_SLOT_MAP, (1, 1, B, 2), vk.U32, [table, lengths, counts], vk.SlotMapParams(R))
        cache = op("update_pages", vk.OP_UPDATE_PAGES, first.shape, vk.F16, [k, v, at], vk.UpdatePagesParams(1e4, True), first)
        op("paged_attn", vk.OP_PAGED_ATTN, (1, B, KV * G, hd), vk.F16, [q, cache, table], vk.PagedAttnParams(0.125, 1e4, True))
        op("adjust_logits", vk.OP_ADJUST_LOGITS, (1, 1, B, V), vk.F16, [x, history, rules])
        steps = [[600, 1, 0], [601, 17, 5], [0, 640, 5], [33, 0, 639]]

        def all_runs():
            for name, t in ops:
                vk.check(name, getattr(L, f"vkllm_op_{name}_run")(ctx.vp, ctx.cmds, t))

        def reset():
            ctx.upload(table, zero)
            ctx.upload(cache, first)

        def results():
            return [ctx.download_raw(t).copy() for _, t in ops]

        want = []
        reset()
        for s in steps:
            ctx.upload(lengths, np.array(s, np.uint32))
            all_runs()
            want.append(results())
        reset()
        try:
            assert H.hipStreamBeginCapture(stream, 0) == 0
            rcs = [getattr(L, f"vkllm_op_{name}_run")(ctx.vp, ctx.cmds, t) for name, t in ops]
            end = H.hipStreamEndCapture(stream, ctypes.byref(graph))
            assert rcs == [vk.ERR_OK] * 5 and end == 0
            assert H.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
            a, b = ctx.tensor_from(f16(1, 1, 300, 512)), ctx.tensor_from(f16(1, 1, 256, 512))
            bag.made += [a, b]
            for i, s in enumerate(steps):
                print(f"[paged capture] replay {i}", flush=True)
                ctx.upload(lengths, np.array(s, np.uint32))
                assert H.hipGraphLaunch(exe, stream) == 0
                assert H.hipStreamSynchronize(stream) == 0
                for (name, _), g, w in zip(ops, results(), want[i]):
                    assert np.array_equal(g, w), (name, i)
                bag.op("matmul", (1, 1, 300, 256), vk.F16, vk.OP_MATMUL, [a, b], vk.MatmulParams(1.0, 0))  # shares the workspace
        finally:
            if exe.value:
                H.hipGraphExecDestroy(exe)
            if graph.value:
                H.hipGraphDestroy(graph)


def test_a_first_call_under_capture_is_refused(ctx, vk):
    """An operator whose result has no memory yet cannot make it while the stream is captured: it says so, the capture goes on,
    and the same call works afterwards."""
    H, L = _hip_runtime(), vk.lib()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    vk.check("stream", L.vkllm_hip_context_stream(ctx.vp, ctypes.byref(stream)))
    r = np.random.default_rng(1)
    q, cache = (r.standard_normal(s).astype(np.float16) for s in ((1, 2, 4, 64), (5, 4, 16, 64)))
    table = np.array([[20, 0, 1], [3, 4, 0xFFFFFFFF]], np.uint32)
    with Bag(ctx) as bag:
        t = ctx.tensor([1, 2, 4, 64], vk.F16, op=vk.OP_PAGED_ATTN, srcs=[bag.put(q), bag.put(cache), bag.put(rows4(table))],
                       params=vk.PagedAttnParams(0.125, 0.0, False))
        x = bag.put(r.standard_normal((1, 1, 2, 100)).astype(np.float16))
        y = ctx.tensor([1, 1, 2, 100], vk.F16, op=vk.OP_ADJUST_LOGITS, srcs=[x])
        bag.made += [t, y]
        assert H.hipStreamBeginCapture(stream, 0) == 0
        rcs = [L.vkllm_op_paged_attn_run(ctx.vp, ctx.cmds, t), L.vkllm_op_adjust_logits_run(ctx.vp, ctx.cmds, y)]
        assert H.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        if graph.value:
            H.hipGraphDestroy(graph)
        assert rcs == [vk.ERR_ARGS, vk.ERR_ARGS]
        vk.check("paged_attn", ctx.run_op("paged_attn", t))
        vk.check("adjust_logits", ctx.run_op("adjust_logits", y))
        want, off = attention(q[0], cache, table, 0.125, 0.0, False)
        assert (np.abs(ctx.download(t)[0] - want) <= np.abs(want) * 2.0 ** -11 * 1.001 + off + 2.0 ** -25).all()
        assert np.array_equal(ctx.download(y), ctx.download(x))


def test_a_source_that_never_ran_is_refused_under_capture(ctx, vk):
    """Nor can an operator make the memory of a source: a table that no call has written yet."""
    H, L = _hip_runtime(), vk.lib()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    vk.check("stream", L.vkllm_hip_context_stream(ctx.vp, ctypes.byref(stream)))
    with Bag(ctx) as bag:
        lengths, counts = bag.put(rows4(np.array([[5, 20]], np.uint32))), bag.put(rows4(np.array([[1, 2]], np.uint32)))
        table = ctx.tensor([1, 1, 2, 4], vk.U32, op=vk.OP_PAGE_TABLE, srcs=[lengths], params=vk.PageTableParams(16, 4))
        slots = ctx.tensor([1, 1, 3, 2], vk.U32, op=vk.OP_SLOT_MAP, srcs=[table, lengths, counts],
                           params=vk.SlotMapParams(16))
        bag.made += [table, slots]
        ctx.upload(slots, np.zeros((1, 1, 3, 2), np.uint32))
        assert H.hipStreamBeginCapture(stream, 0) == 0
        rc = L.vkllm_op_slot_map_run(ctx.vp, ctx.cmds, slots)
        assert H.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        if graph.value:
            H.hipGraphDestroy(graph)
        assert rc == vk.ERR_ARGS
        ctx.upload(table, np.array([[[[0, 0, 0, 0], [0, 0, 0, 0]]]], np.uint32))
        vk.check("page_table", ctx.run_op("page_table", table))
        vk.check("slot_map", ctx.run_op("slot_map", slots))
        assert ctx.download(slots)[0, 0].tolist() == [[4, 4], [34, 18], [35, 19]]


def test_two_captured_calls_share_the_workspace(ctx, vk):
    """Two attention calls, one of long rows that are joined over two levels and one of many short rows, each in a graph of its
    own on the context's stream, replayed in turn with lengths that change between the replays and without a wait between
    the two: every result is that of an eager call, and so are those of the eager calls behind the replays."""
    H, L = _hip_runtime(), vk.lib()
    stream = ctypes.c_void_p()
    vk.check("stream", L.vkllm_hip_context_stream(ctx.vp, ctypes.byref(stream)))
    r = np.random.default_rng(21)
    shapes = [(2, 16, 1, 128, 1200, 16), (70, 4, 2, 64, 12, 16)]  # rows, heads, key heads, head_dim, columns, page rows
    graphs, execs = [], []
    with Bag(ctx) as bag:
        tables, outs = [], []
        for B, heads, KV, hd, P, R in shapes:
            pages = 300
            q = bag.put(r.standard_normal((1, B, heads, hd)).astype(np.float16))
            cache = bag.put(r.standard_normal((pages, 2 * KV, R, hd)).astype(np.float16))
            ids = r.integers(0, pages, (B, 1 + P)).astype(np.uint32)  # pages that rows share
            tables.append((bag.put(rows4(ids)), ids))
            outs.append(ctx.tensor([1, B, heads, hd], vk.F16, op=vk.OP_PAGED_ATTN, srcs=[q, cache, tables[-1][0]],
                                   params=vk.PagedAttnParams(hd ** -0.5, 1e4, True)))
            bag.made.append(outs[-1])

        def set_lengths(i):
            for (t, ids), (B, _, _, _, P, R) in zip(tables, shapes):
                lengths = np.random.default_rng(100 + i).integers(0, P * R + 1, B)
                lengths[-1] = P * R if i % 2 else 0
                ids[:, 0] = lengths
                ctx.upload(t, rows4(ids))

        def eager():
            for t in outs:
                vk.check("paged_attn", L.vkllm_op_paged_attn_run(ctx.vp, ctx.cmds, t))
            return [ctx.download_raw(t).copy() for t in outs]

        want = []
        for i in range(5):
            set_lengths(i)
            want.append(eager())
        try:
            for t in outs:
                graphs.append(ctypes.c_void_p())
                execs.append(ctypes.c_void_p())
                assert H.hipStreamBeginCapture(stream, 0) == 0
                rc = L.vkllm_op_paged_attn_run(ctx.vp, ctx.cmds, t)
                end = H.hipStreamEndCapture(stream, ctypes.byref(graphs[-1]))
                assert rc == vk.ERR_OK and end == 0
                assert H.hipGraphInstantiate(ctypes.byref(execs[-1]), graphs[-1], None, None, 0) == 0
            for i in range(5):
                print(f"[paged graphs] replay {i}", flush=True)
                set_lengths(i)
                for k in range(6):  # each three times, in turn
                    assert H.hipGraphLaunch(execs[k % 2], stream) == 0
                assert H.hipStreamSynchronize(stream) == 0
                for t, w in zip(outs, want[i]):
                    assert np.array_equal(ctx.download_raw(t), w), i
                for got, w in zip(eager(), want[i]):
                    assert np.array_equal(got, w), i
        finally:
            for e in execs:
                if e.value:
                    H.hipGraphExecDestroy(e)
            for g in graphs:
                if g.value:
                    H.hipGraphDestroy(g)
