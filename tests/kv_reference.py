"""The paged cache's operators from their definitions, in numpy / torch on the
host, and the error bounds that their roundings add up to."""
import math

import numpy as np
import torch

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U32 = 2.0 ** -24  # half a step of float32, relative


def half_step(name):
    return torch.finfo(TORCH[name]).eps / 2


def tables(cached, added, page, free, head, table, table_w, max_tokens):
    """(table, slots, start, lengths, head, status) of a step."""
    table = np.array(table, copy=True)
    slots = np.full(max_tokens, -1, np.int64)
    start, lengths, status, t, at = [0], [], 0, 0, head
    if head < 0 or head > len(free):
        status |= 8
        at = min(max(head, 0), len(free))
    for b, (c, a) in enumerate(zip(cached, added)):
        c, a = int(c), int(a)
        if c < 0 or a < 0 or c + a > 2 ** 31 - 1:
            status |= 8
            c = a = 0
        have, need = -(-c // page), -(-(c + a) // page)
        if need > table_w:
            status |= 2
        got = []
        for j in range(have, need):
            got.append(int(free[at]) if at < len(free) else -1)
            if at >= len(free):
                status |= 1
            at += 1
            if j < table_w:
                table[b, j] = got[-1]
        for i in range(a):
            j = (c + i) // page
            if t < max_tokens:
                pid = -1 if j >= table_w else (int(table[b, j]) if j < have else got[j - have])
                slots[t] = -1 if pid < 0 else pid * page + (c + i) % page
            t += 1
        start.append(t)
        lengths.append(c + a)
    if t > max_tokens:
        status |= 4
    return table, slots, np.minimum(start, max_tokens).astype(np.int32), np.array(lengths, np.int32), min(at, len(free)), status


def rows_of(pool, table, n, page):
    """[n, heads, dim] float64 of a table's first n keys, and which of them are there."""
    table = torch.as_tensor(np.asarray(table), dtype=torch.int64)
    key = torch.arange(n)
    j = key // page
    there = j < len(table)
    pid = torch.full((n,), -1, dtype=torch.int64)
    pid[there] = table[j[there]]
    there = (pid >= 0) & (pid < pool.shape[0])
    return pool[pid.clamp(0, pool.shape[0] - 1), :, key % page].double(), there


def attention(q, k_pool, v_pool, scale, prefix_table, prefix_len, table, lengths, start, qtype):
    """(out, bound) in float64: q [T, heads, dim], pools [pages, kv heads,
    page, dim], everything on the host.

    The bound of an output is, with w its weights over their sum and A = sum w
    |V|: half a step of the output's type; half a step a weight where q is 16
    bits wide (weights rounded for the product with V); and in 32 bits the
    score's error ds (dim products and sums, the scaling), which moves a weight
    by e^ds - 1 and the total as much, the exponentials' (four roundings and
    units each of: the argument, up to |s - m| + |m| large, and the function,
    for the weight, the rescalings of its block and part), and sums over n keys
    and the joins (n + 64 roundings each, numerator and denominator)."""
    T, heads, dim = q.shape
    page, kvh = k_pool.shape[2], k_pool.shape[1]
    G = heads // kvh
    out = torch.zeros(T, heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    pk, pthere = rows_of(k_pool, prefix_table, prefix_len, page)
    pv, _ = rows_of(v_pool, prefix_table, prefix_len, page)
    B = len(lengths)
    for t in range(T):
        b = next((x for x in range(B) if start[x] <= t < start[x + 1]), None)
        k, v, there = pk, pv, pthere
        if b is not None:
            seen = int(lengths[b]) - (int(start[b + 1]) - int(start[b])) + (t - int(start[b])) + 1
            seen = max(seen, 0)
            ok, othere = rows_of(k_pool, table[b], seen, page)
            ov, _ = rows_of(v_pool, table[b], seen, page)
            k, v, there = torch.cat([pk, ok]), torch.cat([pv, ov]), torch.cat([pthere, othere])
        k, v = k[there], v[there]
        n = len(k)
        if n == 0:
            continue
        for h in range(heads):
            x = q[t, h].double()
            s = (k[:, h // G] @ x) * scale
            m = s.max()
            if m == -math.inf:
                continue
            w = torch.exp(s - m)
            w = w / w.sum()
            vv = v[:, h // G]
            out[t, h] = w @ vv
            A = w @ vv.abs()
            fin = s[torch.isfinite(s)]
            big = float(fin.abs().max()) if len(fin) else 0.0
            sumabs = (k[:, h // G].abs() @ x.abs()) * abs(scale)
            ds = float(sumabs[torch.isfinite(sumabs)].max()) * (dim + 3) * U32 if len(fin) else 0.0
            rel = (half_step(qtype) if qtype != "f32" else 0.0) + 2 * ds + 4 * (2 * big * 1.5 + 4) * U32 + 2 * (n + 64) * U32
            bound[t, h] = half_step(qtype) * out[t, h].abs() * (1 + rel) + rel * A * (1 + rel) + 1e-30
            if qtype == "f16":
                bound[t, h] += 2.0 ** -25 * (1 + vv.abs().max())  # results, and weights, below float16's normal range
    return out, bound
