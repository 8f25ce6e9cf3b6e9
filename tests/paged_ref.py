"""The operators over a paged cache in numpy, from their definitions, in 64 bits."""
import numpy as np

NONE = 0xFFFFFFFF


def page_table(old, want, page_rows, pages):
    """The table after VKLLM_OP_PAGE_TABLE, row by row."""
    B, P = old.shape[0], old.shape[1] - 1
    new = np.full_like(old, NONE)
    had = np.minimum(old[:, 0].astype(np.int64), P * page_rows)
    target = np.where(want.astype(np.int64) > P * page_rows, had, want.astype(np.int64))
    keep = -(-np.minimum(had, target) // page_rows)
    used = set()
    for b in range(B):
        used |= {int(i) for i in old[b, 1:1 + keep[b]] if i < pages}
    free = [i for i in range(pages) if i not in used]
    asked = 0
    for b in range(B):
        need = -(-int(target[b]) // page_rows) - int(keep[b])
        new[b, 1:1 + keep[b]] = old[b, 1:1 + keep[b]]
        fits = need == 0 or asked + need <= len(free)
        if fits:
            new[b, 1 + keep[b]:1 + keep[b] + need] = free[asked:asked + need]
        new[b, 0] = target[b] if fits else had[b]
        asked += need
    return new


def slot_map(table, lengths, counts, T, page_rows):
    out = np.zeros((T, 2), np.uint32)
    out[:, 0] = NONE
    t = 0
    for b in range(table.shape[0]):
        held = min(int(table[b, 0]), (table.shape[1] - 1) * page_rows)
        for i in range(int(counts[b])):
            if t >= T:
                return out
            pos = int(lengths[b]) - int(counts[b]) + i
            if 0 <= pos < held and int(table[b, 1 + pos // page_rows]) * page_rows + pos % page_rows < NONE:
                out[t] = int(table[b, 1 + pos // page_rows]) * page_rows + pos % page_rows, pos
            t += 1
    return out


def rotate(x, position, base, neox):
    """RoPE of x [..., T, H, hd], token t at position[t]."""
    x = x.astype(np.float64)
    if base == 0:
        return x
    hd = x.shape[-1]
    angle = (np.asarray(position, np.float64)[:, None] * float(base) ** (-np.arange(0, hd, 2) / hd))[:, None]
    z = x[..., :hd // 2] + 1j * x[..., hd // 2:] if neox else x[..., 0::2] + 1j * x[..., 1::2]
    z = z * np.exp(1j * angle)
    if neox:
        return np.concatenate((z.real, z.imag), -1)
    return np.stack((z.real, z.imag), -1).reshape(x.shape)


def attention(q, cache, table, scale, base, neox, eps_q=0.0):
    """(out [B, H, hd], a bound on what fp32 sums and exponentials may be off). Positions on absent pages are left out."""
    B, H, hd = q.shape
    pages, KV2, R, _ = cache.shape
    KV, P = KV2 // 2, table.shape[1] - 1
    out, off = np.zeros((B, H, hd)), np.zeros((B, H, hd))
    for b in range(B):
        n = min(int(table[b, 0]), P * R)
        pos = np.arange(n)
        page = table[b, 1 + pos // R].astype(np.int64)
        there = page < pages
        page, row = page[there], (pos % R)[there]
        if page.size == 0:
            continue
        rows = cache[page, :, row].astype(np.float64)  # [n, 2 KV, hd]
        qr = rotate(q[b][None], [n - 1], base, neox)[0]
        for h in range(H):
            k, v = rows[:, h // (H // KV)], rows[:, KV + h // (H // KV)]
            s = scale * (k @ qr[h])
            # scores: fp32 sums of hd products (16 roundoffs of their magnitudes, as dot_atol counts), the rotation's
            # three roundings and, in the exponent, the product with log2(e)
            eps = (16 + 8 * (base != 0)) * 2.0 ** -24 * abs(scale) * (np.abs(k) @ np.abs(qr[h])).max() \
                + 2.0 ** -22 * np.abs(s).max() + eps_q
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, h] = p @ v
            # a score off by eps moves a probability by 2 eps of itself; the exponential, sums and quotient add a few
            # roundoffs; fp16 probabilities in two parts keep 22 bits, and those under 2^-33 of the sum may vanish
            off[b, h] = (2.2 * eps + 32 * 2.0 ** -24) * (p @ np.abs(v)) + page.size * 2.0 ** -33 * np.abs(v).max(0)
    return out, off


def adjust(x, history, rules, mask):
    """Rows of logits [B, V] in 64 bits."""
    y = x.astype(np.float64).copy()
    B, V = y.shape
    for b in range(B):
        if history is not None:
            rep, freq, pres = rules[b, :3].view(np.float32).astype(np.float64)
            used = history[b, 1:1 + min(int(history[b, 0]), history.shape[1] - 1)]
            for v, n in zip(*np.unique(used[used < V], return_counts=True)):
                y[b, v] = (y[b, v] / rep if y[b, v] > 0 else y[b, v] * rep) - (freq * n + pres)
        if rules is not None:
            n = min(int(rules[b, 3]), (rules.shape[1] - 4) // 2)
            bias = {}
            for i in range(n):
                bias[int(rules[b, 4 + 2 * i])] = float(rules[b, 5 + 2 * i:6 + 2 * i].view(np.float32)[0])
            for v, value in bias.items():
                if v < V:
                    y[b, v] += value
        if mask is not None:
            v = np.arange(V)
            y[b][(mask[b, v // 32] >> (v % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return y
