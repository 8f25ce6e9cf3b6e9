"""Prompts taken in at once beside a batch in progress: a prompt's tokens attend to their own keys with ROPE, MATMUL and SOFTMAX,
as the model graph's do, while UPDATE_PAGES stores the same keys and values; the sequence then goes on in the batch, a token a
step. Logits after every prompt token and every step are those of the model's forward pass in numpy."""
import ctypes

import numpy as np
import pytest

from test_paged_gpu import Bag, rows4
from test_paged_loop_gpu import PAGE, ROWS, Server, forward, tiny  # noqa: F401

pytestmark = pytest.mark.gpu


class Prompts(Bag):
    """Prompts of one server's model into its pages."""

    def __init__(self, ctx, vk, model, srv):
        super().__init__(ctx)
        self.vk, self.model, self.srv = vk, model, srv

    def do(self, name, shape, op, srcs, params=None, dtype=None):
        return self.op(name, shape, dtype or self.vk.F16, op, srcs, params)

    def seen(self, t, shape, axes=None):
        """t's memory as `shape`, its axes in the order `axes`."""
        r = self.vk.TensorP()
        L = self.vk.lib()
        self.vk.check("copy_ref", L.vkllm_tensor_copy_ref(self.ctx.vp, t, ctypes.byref(r)))
        self.vk.check("reshape", L.vkllm_tensor_reshape(self.ctx.vp, r, (ctypes.c_uint32 * 4)(*shape)))
        if axes:
            self.vk.check("permute", L.vkllm_tensor_permute(self.ctx.vp, r, (ctypes.c_uint32 * 4)(*axes)))
        self.made.append(r)
        return r

    def run(self, lengths, row, toks):
        """Logits [T, V] of the row's T tokens; `lengths` are the batch's with the prompt, whose row is the only one with new
        tokens."""
        vk, srv, m, w = self.vk, self.srv, self.model.meta, self.model.m.weights
        D, H, V, T = m.embedding_length, m.head_count, m.vocab_size, len(toks)
        hd = D // H
        rms, plain = vk.RmsnormParams(2.0, m.layer_norm_rms_epsilon), vk.MatmulParams(1.0, 0)
        counts = np.zeros(ROWS)
        counts[row] = T
        wanted, counts = self.put(rows4(np.asarray(lengths)[None])), self.put(rows4(counts[None]))
        self.ctx.upload(srv.lengths, np.asarray(lengths, np.uint32))
        vk.check("page_table", self.ctx.run_op("page_table", srv.table))
        at = self.do("slot_map", (1, 1, T, 2), vk.OP_SLOT_MAP, [srv.table, wanted, counts], vk.SlotMapParams(PAGE), vk.U32)
        tokens = self.put(np.asarray(toks, np.uint32).reshape(1, 1, 1, T))
        x = self.do("embedding", (1, 1, T, D), vk.OP_EMBEDDING, [tokens, w.tok_embed_weights], ctypes.c_uint32(0))
        for i, cache in enumerate(srv.caches):
            b = w.blocks.contents.data[i].contents
            n = self.do("rmsnorm", (1, 1, T, D), vk.OP_RMSNORM, [x, b.attn_norm_weight], rms)
            q, k, v = (self.do("matmul", (1, 1, T, D), vk.OP_MATMUL, [n, wt], plain) for wt in (b.WQ, b.WK, b.WV))
            # the cache's node takes this prompt's rows, then the batch's again
            c, mine = cache.contents, [self.seen(k, (1, T, H, hd)), self.seen(v, (1, T, H, hd)), at]
            steps = [vk.TensorP.from_buffer_copy(c.srcs[j]) for j in range(3)]  # c.srcs[j] itself follows the node
            for j in range(3):
                c.srcs[j] = mine[j]
            vk.check("update_pages", self.ctx.run_op("update_pages", cache))
            for j in range(3):
                c.srcs[j] = steps[j]
            turn = vk.RopeParams(0, m.rope_freq_base, False)
            q, k = (self.do("rope", (1, H, T, hd), vk.OP_ROPE, [self.seen(t, (1, T, H, hd), (0, 2, 1, 3))], turn) for t in (q, k))
            s = self.do("matmul", (1, H, T, T), vk.OP_MATMUL, [q, k], vk.MatmulParams(hd ** -0.5, 0))
            p = self.do("softmax", (1, H, T, T), vk.OP_SOFTMAX, [s], vk.SoftmaxParams(1, 0))
            # values as [1, H, hd, T]: read as rows of one dim whatever T is
            o = self.do("matmul", (1, H, T, hd), vk.OP_MATMUL, [p, self.seen(v, (1, T, H, hd), (0, 2, 3, 1))], plain)
            o = self.do("copy", (1, T, H, hd), vk.OP_COPY, [self.seen(o, (1, H, T, hd), (0, 2, 1, 3))])
            o = self.do("matmul", (1, 1, T, D), vk.OP_MATMUL, [self.seen(o, (1, 1, T, D)), b.WO], plain)
            x = self.do("bin", (1, 1, T, D), vk.OP_BIN, [x, o], ctypes.c_int32(0))
            n = self.do("rmsnorm", (1, 1, T, D), vk.OP_RMSNORM, [x, b.ffn_norm_weight], rms)
            u = self.do("ffn_up_and_gate", (1, 1, T, b.WU.contents.shapes[2]), vk.OP_FFN_UP_AND_GATE, [n, b.WU, b.WG])
            x = self.do("bin", (1, 1, T, D), vk.OP_BIN, [x, self.do("matmul", (1, 1, T, D), vk.OP_MATMUL, [u, b.WD], plain)],
                        ctypes.c_int32(0))
        n = self.do("rmsnorm", (1, 1, T, D), vk.OP_RMSNORM, [x, w.output_norm_weight], rms)
        return self.ctx.download(self.do("matmul", (1, 1, T, V), vk.OP_MATMUL, [n, w.output_weight], plain))[0, 0]


def test_prompts_beside_a_batch(ctx, vk, tiny):  # noqa: F811
    r = np.random.default_rng(5)
    hd = tiny.meta.embedding_length // tiny.meta.head_count
    # row: what its prompt waits for (steps done), its prompt's length and how many steps follow it
    plan = {0: (0, hd, 14), 2: (0, 60, 9), 1: (4, 5, 20), 3: (6, 1, 3)}
    seqs = {row: dict(start=start, prompt=n, end=start + steps, toks=r.integers(0, 32000, n + steps).astype(np.uint32), got=[])
            for row, (start, n, steps) in plan.items()}
    srv = Server(ctx, vk, tiny)
    try:
        lengths = np.zeros(ROWS, np.uint32)
        for step in range(max(s["end"] for s in seqs.values())):
            for row, s in seqs.items():
                if s["end"] == step:
                    lengths[row] = 0
            for row, s in seqs.items():
                if s["start"] == step:
                    print(f"[paged prompt] row {row}: {s['prompt']} tokens before step {step}", flush=True)
                    lengths[row] = s["prompt"]
                    with Prompts(ctx, vk, tiny, srv) as prompts:
                        s["got"] += list(prompts.run(lengths, row, s["toks"][:s["prompt"]]).astype(np.float32))
                    assert np.array_equal(ctx.download(srv.table)[0, 0][:, 0], lengths)
            live = [row for row, s in seqs.items() if s["start"] <= step < s["end"]]
            tokens = np.zeros(ROWS, np.uint32)
            for row in live:
                s = seqs[row]
                tokens[row] = s["toks"][s["prompt"] + step - s["start"]]
                lengths[row] += 1
            # a token in every row: those without a sequence have no position, and the map no slot for them
            raw, _ = srv.step(lengths, np.ones(ROWS), tokens)
            assert np.array_equal(ctx.download(srv.table)[0, 0][:, 0], lengths)
            for row in live:
                seqs[row]["got"].append(raw[row].astype(np.float32))
    finally:
        srv.close()
    for row, s in seqs.items():
        assert len(s["got"]) == len(s["toks"])
        err = np.abs(np.stack(s["got"]) - forward(ctx, tiny, s["toks"])).max(1)
        print(f"[paged prompt] row {row}: max|dlogit| {err[:s['prompt']].max():.3g} of the prompt, {err[s['prompt']:].max():.3g} behind",
              flush=True)
        assert err.max() <= 2e-2, (row, int(err.argmax()), err.max())  # the bar of the token loop's own tests
