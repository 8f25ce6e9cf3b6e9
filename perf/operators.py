"""The operators of batched generation over a paged key-value cache, timed case by case.

A cache is one tensor of pages [pages, 2 KV, page, hd]: KV heads of keys, then KV heads of values, `page` rows each. A
batch of sequences has a page table [rows, 1 + columns] of 32-bit words: a sequence's length, then its pages in order,
then NONE. Four kinds of case:

  tables   PAGE_TABLE: the table for the lengths that the host wants next (sequences grow, shrink, end and begin; pages
           come from those that no row keeps, the lowest first); SLOT_MAP: (cache row, position) of each new token
  rows     UPDATE_PAGES: new tokens' keys, rotated to their positions, and values into the rows that the map names
  attend   PAGED_ATTN: one new token of each sequence, its query rotated to the last position, over that sequence's pages
  logits   ADJUST_LOGITS: repetition, frequency and presence penalties, token biases and a grammar's mask

With `own` false, run() computes them in elementary torch operations in 32 bits (angles in 64); with it true it calls
the VKLLM_OP_* operators on a context's stream, which is torch's current stream from the first prepare() on: what a caller
does with the results in torch comes after them.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

THETA = 10000.0
NONE = -1  # 0xFFFFFFFF as torch's int32 holds it


def listed():
    return [
        # one user's next token, a context of 4096 positions in pages of 16: nothing but latency
        {"name": "tables_1", "kind": "tables", "rows": 1, "page": 16, "columns": 256, "pages": 256, "tokens": 1},
        # a server's step: 256 sequences of up to 8192 positions, some that end, some that begin with a prompt
        {"name": "tables_256", "kind": "tables", "rows": 256, "page": 16, "columns": 512, "pages": 65536, "tokens": 2048},
        # the row of one generated token at the 7B heads
        {"name": "rows_7b_1", "kind": "rows", "tokens": 1, "kv": 32, "hd": 128, "page": 16, "pages": 256, "neox": False,
         "dtype": "f16"},
        # a step of 61 sequences at the 13B heads, in 32 bits
        {"name": "rows_13b_61_f32", "kind": "rows", "tokens": 61, "kv": 40, "hd": 128, "page": 16, "pages": 512,
         "neox": False, "dtype": "f32"},
        # the prompts that a server took in at once
        {"name": "rows_prompt", "kind": "rows", "tokens": 4001, "kv": 32, "hd": 128, "page": 64, "pages": 128, "neox": True,
         "dtype": "f16"},
        # the smallest model's token: the smallest call
        {"name": "attend_tiny", "kind": "attend", "rows": 1, "heads": 6, "kv": 6, "hd": 48, "longest": 200, "page": 16,
         "neox": False, "dtype": "f16"},
        # one user deep into a conversation at the 7B heads
        {"name": "attend_7b_1", "kind": "attend", "rows": 1, "heads": 32, "kv": 32, "hd": 128, "longest": 4001, "page": 16,
         "neox": False, "dtype": "f16"},
        # a small batch at the 13B heads, in 32 bits
        {"name": "attend_13b_f32", "kind": "attend", "rows": 5, "heads": 40, "kv": 40, "hd": 128, "longest": 2000,
         "page": 32, "neox": False, "dtype": "f32"},
        # a server's batch of ragged lengths, four query heads to a key head
        {"name": "attend_ragged", "kind": "attend", "rows": 64, "heads": 32, "kv": 8, "hd": 128, "longest": 8192,
         "page": 16, "neox": True, "dtype": "f16"},
        # two long documents, eight query heads to a key head
        {"name": "attend_long", "kind": "attend", "rows": 2, "heads": 32, "kv": 4, "hd": 128, "longest": 131072, "page": 64,
         "neox": True, "dtype": "f16"},
        # one user's next token
        {"name": "logits_1", "kind": "logits", "rows": 1, "vocab": 32000, "history": 131, "biases": 4, "dtype": "f16"},
        # a server's batch with a large vocabulary and long histories
        {"name": "logits_256", "kind": "logits", "rows": 256, "vocab": 131072, "history": 4096, "biases": 300,
         "dtype": "f16"},
    ]


def log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tables", "rows", "attend", "attend", "logits"])
    page, dtype = 16 * rng.choice([1, 1, 2, 3, 4, 8]), rng.choice(["f16", "f16", "f32"])
    if kind == "tables":
        rows, columns = log_int(rng, 1, 1000), log_int(rng, 4, 700)
        return {"kind": kind, "rows": rows, "page": page, "columns": columns,
                "pages": max(4, int(rows * columns * rng.uniform(0.3, 0.6))), "tokens": log_int(rng, rows, 8 * rows + 8)}
    if kind == "logits":
        return {"kind": kind, "rows": log_int(rng, 1, 200), "vocab": log_int(rng, 1000, 130000),
                "history": log_int(rng, 1, 4096), "biases": log_int(rng, 1, 300), "dtype": dtype}
    hd = rng.choice([48, 64, 80, 96, 128, 128, 128, 256])
    neox = rng.random() < 0.5
    if kind == "rows":
        tokens, kv = log_int(rng, 1, 2500), rng.choice([1, 2, 6, 8, 32])
        return {"kind": kind, "tokens": tokens, "kv": kv, "hd": hd, "page": page, "pages": -(-tokens // page) * 2 + 3,
                "neox": neox, "dtype": dtype}
    kv = rng.choice([1, 2, 4, 8, 8, 32])
    heads = kv * rng.choice([1, 1, 2, 4, 5, 8] if kv > 8 else [1, 2, 4, 7, 8, 16])
    rows = log_int(rng, 1, 128)
    most = 1.0e8 / (rows * kv * hd)  # a cache of half a GB at most in 16 bits
    return {"kind": kind, "rows": rows, "heads": heads, "kv": kv, "hd": hd,
            "longest": min(log_int(rng, 1, 100000), int(most)), "page": page, "neox": neox, "dtype": dtype}


# ---- inputs, made from the seed alone ------------------------------------------------------------------------------
TORCH = {"f16": torch.float16, "f32": torch.float32}


class Inputs:
    """Tensors of one seed, in the order in which they are asked for; `r` draws what the host knows (lengths, ids)."""

    def __init__(self, seed):
        self.r = np.random.RandomState((int(seed) * 7919 + 17) % (1 << 32))
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) * 7919 + 17)

    def normal(self, *shape, dtype, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32).mul_(std).to(TORCH[dtype])

    def words(self, a):
        return torch.from_numpy(np.ascontiguousarray(a).astype(np.uint32).view(np.int32)).cuda()


def table_of(r, lengths, page, columns, pages):
    """A table of `lengths`, its pages in an order that a long-running server leaves them in."""
    need = -(-lengths // page)
    order, at = r.permutation(pages), np.concatenate([[0], np.cumsum(need)])
    table = np.full((lengths.size, 1 + columns), 0xFFFFFFFF, np.uint32)
    table[:, 0] = lengths
    for b in range(lengths.size):
        table[b, 1:1 + need[b]] = order[at[b]:at[b + 1]]
    return table


def ragged(r, rows, longest):
    """Lengths of a batch: one at the longest, the others spread below it, one in sixteen without a token."""
    lengths = np.exp(r.uniform(0, math.log(longest + 1), rows)).astype(np.int64).clip(1, longest)
    lengths = np.where(r.rand(rows) < 0.5, r.randint(1, longest + 1, rows), lengths)
    lengths[r.rand(rows) < 1 / 16] = 0
    lengths[r.randint(rows)] = longest
    return lengths


def table_inputs(case, seed):
    x = Inputs(seed)
    r, rows, page, columns, pages = x.r, case["rows"], case["page"], case["columns"], case["pages"]
    longest = columns * page - 1
    old = ragged(r, rows, max(1, longest - 1))
    while (-(-old // page)).sum() > 0.8 * pages:
        old = (old * 0.9).astype(np.int64)
    new, counts, room = old + 1, np.ones(rows, np.int64), case["tokens"] - rows
    ends = (r.rand(rows) < 0.06) & (np.arange(rows) > 0)
    new[ends], counts[ends] = 0, 0
    for b in np.flatnonzero(old == 0):  # rows without a sequence take a prompt while there is room
        n = min(1 + int(r.randint(1 + max(0, room))), longest)
        new[b], counts[b], room = n, n, room - (n - 1)
    return {"old": x.words(table_of(r, old, page, columns, pages)), "lengths": x.words(new), "counts": x.words(counts)}


def rows_inputs(case, seed):
    x = Inputs(seed)
    T, KV, hd, page, pages, dt = (case[n] for n in ("tokens", "kv", "hd", "page", "pages", "dtype"))
    slots, positions = x.r.permutation(pages * page)[:T], x.r.randint(0, 100000, T)
    if T > 3:
        slots[x.r.randint(T)] = 0xFFFFFFFF  # a padded batch: a token without a row
    return {"cache": x.normal(pages, 2 * KV, page, hd, dtype=dt), "k": x.normal(1, T, KV, hd, dtype=dt),
            "v": x.normal(1, T, KV, hd, dtype=dt), "map": x.words(np.stack([slots, positions], 1))}


def attend_inputs(case, seed):
    x = Inputs(seed)
    B, H, KV, hd, page, dt = (case[n] for n in ("rows", "heads", "kv", "hd", "page", "dtype"))
    lengths = ragged(x.r, B, case["longest"])
    need, columns = -(-lengths // page), -(-case["longest"] // page)
    pages = B * columns  # of which a ragged batch leaves some free
    if B > 4:
        pages = max(int(need.sum()), (2 * B * columns) // 3)
    table = table_of(x.r, lengths, page, columns, pages)
    return {"q": x.normal(1, B, H, hd, dtype=dt, std=1.3), "cache": x.normal(pages, 2 * KV, page, hd, dtype=dt, std=1.3),
            "table": x.words(table)}


def logits_inputs(case, seed):
    x = Inputs(seed)
    B, V, T, n = case["rows"], case["vocab"], case["history"], case["biases"]
    r = x.r
    history = np.zeros((B, 1 + T), np.uint32)
    history[:, 1:] = np.minimum(r.zipf(1.3, (B, T)) * 7919 % V, V - 1)  # a text's words: a few often, many once
    history[:, 0] = np.maximum(1, r.randint(T // 2, T + 1, B))
    rules = np.zeros((B, 4 + 2 * n), np.uint32)
    rules[:, 0:3] = np.stack([r.uniform(1.0, 1.3, B), r.uniform(0, 0.8, B), r.uniform(0, 0.8, B)], 1).astype(
        np.float32).view(np.uint32)
    rules[:, 3] = r.randint(0, n + 1, B)
    rules[:, 4::2] = r.randint(0, V, (B, n))
    rules[:, 5::2] = r.choice([-100.0, -2.5, 1.25, 5.0], (B, n)).astype(np.float32).view(np.uint32)
    words = -(-V // 32)
    mask = r.randint(0, 1 << 32, (B, words), dtype=np.uint32) | r.randint(0, 1 << 32, (B, words), dtype=np.uint32)
    mask[r.rand(B) < 0.5] = 0xFFFFFFFF  # half of the requests have no grammar
    return {"logits": x.normal(1, 1, B, V, dtype=case["dtype"], std=3.0), "history": x.words(history),
            "rules": x.words(rules), "mask": x.words(mask)}


INPUTS = {"tables": table_inputs, "rows": rows_inputs, "attend": attend_inputs, "logits": logits_inputs}


# ---- the framework's calls -----------------------------------------------------------------------------------------
def framework():
    sys.path.insert(1, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vkllm.c_amd"))
    import pyvkllm

    return pyvkllm


class DeviceArray:
    """A device address for torch.as_tensor; the tensor made of it keeps its owner."""

    def __init__(self, ptr, shape, typestr, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False), "version": 2,
                                         "strides": None}


def on_device(V, t, owner):
    """The memory of a packed framework tensor of the program `owner` as a torch tensor."""
    c = t.contents
    kind = {V.F32: "<f4", V.F16: "<f2", V.U32: "<i4"}[c.dtype]
    return torch.as_tensor(DeviceArray(c.data.dev, tuple(c.shapes), kind, owner), device="cuda")


class Program:
    """What a program that generates in batches holds for one case: its tensors and the operators over them."""

    context = None  # one for the process, as such a program has it

    def __init__(self, case, x):
        V = self.V = framework()
        if Program.context is None:
            Program.context = V.Ctx(0)
            stream = ctypes.c_void_p()
            V.check("stream", V.lib().vkllm_hip_context_stream(Program.context.vp, ctypes.byref(stream)))
            torch.cuda.synchronize()  # what torch has done so far was on another stream
            torch.cuda.set_stream(torch.cuda.ExternalStream(stream.value))
        self.ctx, self.L, self.tensors, self.todo, self.seen = Program.context, V.lib(), [], [], None
        F = {"f16": V.F16, "f32": V.F32}.get(case.get("dtype"))
        page, kind = case.get("page"), case["kind"]
        self.out = {}
        if kind == "tables":
            rows, wide = x["old"].shape
            old, lengths, counts = (self.input(x[n], V.U32) for n in ("old", "lengths", "counts"))
            table = self.op("table", "page_table", (1, 1, rows, wide), V.U32, V.OP_PAGE_TABLE, [lengths, old],
                            V.PageTableParams(page, case["pages"]))
            self.op("map", "slot_map", (1, 1, case["tokens"], 2), V.U32, V.OP_SLOT_MAP, [table, lengths, counts],
                    V.SlotMapParams(page))
        elif kind == "rows":
            k, v, at = self.input(x["k"], F), self.input(x["v"], F), self.input(x["map"], V.U32)
            cache = self.op("cache", "update_pages", x["cache"].shape, F, V.OP_UPDATE_PAGES, [k, v, at],
                            V.UpdatePagesParams(THETA, case["neox"]))
            on_device(V, cache, self).copy_(x["cache"])
        elif kind == "attend":
            q, cache, table = self.input(x["q"], F), self.input(x["cache"], F), self.input(x["table"], V.U32)
            self.op("heads", "paged_attn", x["q"].shape, F, V.OP_PAGED_ATTN, [q, cache, table],
                    V.PagedAttnParams(1.0 / math.sqrt(case["hd"]), THETA, case["neox"]))
        else:
            srcs = [self.input(x["logits"], F)] + [self.input(x[n], V.U32) for n in ("history", "rules", "mask")]
            self.op("logits", "adjust_logits", x["logits"].shape, F, V.OP_ADJUST_LOGITS, srcs)
        torch.cuda.synchronize()

    def input(self, x, dtype):
        shape = (1,) * (4 - x.dim()) + tuple(x.shape)
        t = self.ctx.tensor(list(shape), dtype)
        self.tensors.append(t)
        on_device(self.V, t, self).copy_(x.view(shape))
        return t

    def op(self, name, call, shape, dtype, op, srcs, params=None):
        t = self.ctx.tensor(list(shape), dtype, op=op, srcs=srcs, params=params)
        self.tensors.append(t)
        self.out[name] = t
        V, L = self.V, self.L
        V.check(call, getattr(L, f"vkllm_op_{call}_init")(self.ctx.vp, self.ctx.cmds, t))
        self.todo.append((call, getattr(L, f"vkllm_op_{call}_run"), t))
        return t

    def run(self):
        for call, run_op, t in self.todo:
            self.V.check(call, run_op(self.ctx.vp, self.ctx.cmds, t))
        if self.seen is None:  # the outputs' memory exists from the first pass on
            self.seen = {n: on_device(self.V, t, self) for n, t in self.out.items()}
        return self.seen

    def __del__(self):
        if getattr(self, "ctx", None) is not None:
            self.ctx.sync()
            for t in self.tensors:
                self.ctx.free(t)


# ---- the operators in plain form -----------------------------------------------------------------------------------
def rotated(x, position, neox, dtype):
    """RoPE of the last axis of x [..., T, H, hd], token t at position[t], in `dtype`, angles in 64 bits."""
    hd = x.shape[-1]
    freq = THETA ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = (position.double()[:, None] * freq)[:, None]
    c, s, x = angle.cos().to(dtype), angle.sin().to(dtype), x.to(dtype)
    a, b = (x[..., :hd // 2], x[..., hd // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
    u, w = c * a - s * b, s * a + c * b
    return torch.cat((u, w), -1) if neox else torch.stack((u, w), -1).flatten(-2)


def plain_tables(case, x):
    page, pages, T = case["page"], case["pages"], case["tokens"]
    old, want = x["old"].long(), x["lengths"].long()
    columns = old.shape[1] - 1
    had, held = old[:, 0], old[:, 1:]
    want = torch.where(want > columns * page, had, want)
    keep = (torch.minimum(had, want) + page - 1) // page
    need = (want + page - 1) // page - keep
    column = torch.arange(columns, device="cuda")
    kept = column < keep[:, None]
    used = torch.zeros(pages + 1, dtype=torch.int64, device="cuda")
    used = used.scatter(0, torch.where(kept, held, pages).flatten(), 1)[:pages]
    rank = torch.cumsum(1 - used, 0)
    free = torch.zeros(pages + 1, dtype=torch.int64, device="cuda").scatter(
        0, torch.where(used == 0, rank - 1, pages), torch.arange(pages, device="cuda"))
    start = torch.cumsum(need, 0) - need
    fits = (need == 0) | (start + need <= rank[-1])
    fresh = (column >= keep[:, None]) & (column < (keep + need)[:, None]) & fits[:, None]
    given = free[torch.where(fresh, start[:, None] + column - keep[:, None], 0)]
    length = torch.where(fits, want, had)
    table = torch.cat((length[:, None], torch.where(kept, held, torch.where(fresh, given, NONE))), 1)

    counts, asked = x["counts"].long(), x["lengths"].long()
    end = torch.cumsum(counts, 0)
    token = torch.arange(T, device="cuda")
    row = torch.searchsorted(end, token, right=True)
    live, row = row < counts.numel(), row.clamp(max=counts.numel() - 1)
    position = asked[row] - end[row] + token
    live &= (position >= 0) & (position < length[row])
    position = torch.where(live, position, 0)
    slot = table[row, 1 + position // page] * page + position % page
    pairs = torch.stack((torch.where(live, slot, NONE), torch.where(live, position, 0)), 1)
    return {"table": table.int()[None, None], "map": pairs.int()[None, None]}


def plain_rows(case, x):
    page, KV, cache = case["page"], case["kv"], x["cache"]
    slot, position = x["map"][:, 0].long(), x["map"][:, 1].long()
    rows = torch.cat((rotated(x["k"][0], position, case["neox"], torch.float32), x["v"][0].float()), 1).to(cache.dtype)
    live = slot >= 0
    # a token without a row repeats what the first that has one does
    token = torch.where(live, torch.arange(slot.numel(), device="cuda"), live.int().argmax())
    slot = slot[token]
    cache.transpose(1, 2).index_put_((slot // page, slot % page), rows[token])
    return {"cache": cache}


def plain_attend(case, x):
    B, H, KV, hd, page = (case[n] for n in ("rows", "heads", "kv", "hd", "page"))
    table = x["table"].long()
    length, at = table[:, 0], table[:, 1:].clamp(min=0)
    kv = x["cache"][at].float().permute(0, 2, 1, 3, 4).reshape(B, 2 * KV, -1, hd)
    k, v = kv[:, :KV], kv[:, KV:]
    q = rotated(x["q"][0], (length - 1).clamp(min=0), case["neox"], torch.float32).view(B, KV, H // KV, hd)
    masked = (torch.arange(k.shape[2], device="cuda") >= length[:, None])[:, None, None]
    scores = (torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)).masked_fill(masked, -math.inf)
    top = scores.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
    e = torch.exp(scores - top)
    heads = torch.matmul(e, v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return {"heads": heads.view(1, B, H, hd).to(x["q"].dtype)}


def adjusted(x, V, dtype):
    """The rules on logits [B, V] in `dtype`."""
    logits, history, rules = x["logits"][0, 0].to(dtype), x["history"].long(), x["rules"]
    B, T, n = history.shape[0], history.shape[1] - 1, (rules.shape[1] - 4) // 2
    seen = torch.arange(T, device="cuda") < history[:, :1]
    count = torch.zeros(B, V + 1, dtype=dtype, device="cuda").scatter_add(
        1, torch.where(seen, history[:, 1:], V), torch.ones(B, T, dtype=dtype, device="cuda"))[:, :V]
    rep, freq, pres = rules[:, :3].contiguous().view(torch.float32).to(dtype)[:, :, None].unbind(1)
    y = torch.where(logits > 0, logits / rep, logits * rep) - (freq * count + pres)
    y = torch.where(count > 0, y, logits)
    entry, token = torch.arange(n, device="cuda"), rules[:, 4::2].long()
    token = torch.where(entry < rules[:, 3:4], token, V)
    last = torch.zeros(B, V + 1, dtype=torch.int64, device="cuda").scatter_reduce(
        1, token, (entry + 1).expand(B, n), "amax")[:, :V]
    value = torch.cat((torch.zeros(B, 1, device="cuda", dtype=dtype),
                       rules[:, 5::2].contiguous().view(torch.float32).to(dtype)), 1)
    y = y + value.gather(1, last)
    bits = (x["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    return y.masked_fill(bits.flatten(1)[:, :V] == 0, -math.inf)


def plain_logits(case, x):
    return {"logits": adjusted(x, case["vocab"], torch.float32).to(x["logits"].dtype)[None, None]}


PLAIN = {"tables": plain_tables, "rows": plain_rows, "attend": plain_attend, "logits": plain_logits}


# ---- what a program has in hand, and a pass ------------------------------------------------------------------------
def prepare(case, seed):
    x = INPUTS[case["kind"]](case, seed)
    if own:
        return Program(case, x)
    torch.cuda.synchronize()
    return {"case": case, "inputs": x}


def run(state):
    if own:
        return state.run()
    return PLAIN[state["case"]["kind"]](state["case"], state["inputs"])


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    size = {"f16": 2, "f32": 4}.get(case.get("dtype"))
    if case["kind"] == "tables":
        table = case["rows"] * (1 + case["columns"])
        return {"bytes": 4 * (2 * table + 2 * case["rows"] + 2 * case["tokens"]), "flops": 0}
    if case["kind"] == "rows":
        values = case["tokens"] * case["kv"] * case["hd"]
        return {"bytes": 4 * values * size + 8 * case["tokens"], "flops": 3 * values}
    if case["kind"] == "attend":
        B, H, KV, hd, page = (case[n] for n in ("rows", "heads", "kv", "hd", "page"))
        total = int(np.mean([ragged(np.random.RandomState(s), B, case["longest"]).sum() for s in range(16)]))
        return {"bytes": 2 * total * KV * hd * size + 2 * B * H * hd * size + 4 * (B + total // page),
                "flops": 4 * total * H * hd}
    B, V = case["rows"], case["vocab"]
    return {"bytes": B * (2 * V * size + 4 * (-(-V // 32) + 1 + case["history"] + 4 + 2 * case["biases"])), "flops": 2 * B * V}


# ---- the same in 64 bits, from the definitions ---------------------------------------------------------------------
def turn(x, position, neox):
    """x [H, hd] at one position, in complex numbers."""
    hd = x.shape[-1]
    w = position * THETA ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)
    x = x.double()
    z = torch.complex(x[:, :hd // 2], x[:, hd // 2:]) if neox else torch.view_as_complex(x.reshape(x.shape[0], -1, 2))
    z = z * torch.polar(torch.ones_like(w), w)
    return torch.cat((z.real, z.imag), -1) if neox else torch.view_as_real(z).reshape(x.shape)


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None  # whole numbers: no rounding to compare
    x = INPUTS[kind](case, seed)
    if kind == "rows":
        cache, KV, page = x["cache"].double(), case["kv"], case["page"]
        for t, (slot, position) in enumerate(x["map"].tolist()):
            if slot >= 0:
                cache[slot // page, :KV, slot % page] = turn(x["k"][0, t], position, case["neox"])
                cache[slot // page, KV:, slot % page] = x["v"][0, t].double()
        return {"cache": cache}
    if kind == "attend":
        B, H, KV, hd, page = (case[n] for n in ("rows", "heads", "kv", "hd", "page"))
        heads = torch.zeros(1, B, H, hd, device="cuda", dtype=torch.float64)
        for b, row in enumerate(x["table"].tolist()):
            if row[0] == 0:
                continue
            at = torch.tensor(row[1:1 + -(-row[0] // page)], device="cuda")
            kv = x["cache"][at].transpose(0, 1).reshape(2 * KV, -1, hd)[:, :row[0]].double()
            q = turn(x["q"][0, b], row[0] - 1, case["neox"])
            for h in range(KV):
                mine = slice(h * (H // KV), (h + 1) * (H // KV))
                heads[0, b, mine] = torch.softmax(q[mine] @ kv[h].T / math.sqrt(hd), -1) @ kv[KV + h]
        return {"heads": heads}
    V, rows = case["vocab"], []
    for b in range(case["rows"]):
        y, h, rule = x["logits"][0, 0, b].double(), x["history"][b], x["rules"][b]
        rep, freq, pres = rule[:3].view(torch.float32).double()
        count = torch.bincount(h[1:1 + int(h[0])].long(), minlength=V).double()
        y = torch.where(count > 0, torch.where(y > 0, y / rep, y * rep) - freq * count - pres, y)
        pairs = rule[4:4 + 2 * int(rule[3])].cpu()
        bias = dict(zip(pairs[0::2].tolist(), pairs[1::2].contiguous().view(torch.float32).tolist()))
        if bias:
            y[torch.tensor(list(bias), device="cuda")] += torch.tensor(list(bias.values()), device="cuda").double()
        word = torch.arange(V, device="cuda")
        rows.append(torch.where((x["mask"][b][word // 32] >> (word % 32)) & 1 == 1, y, -math.inf))
    return {"logits": torch.stack(rows)[None, None]}
