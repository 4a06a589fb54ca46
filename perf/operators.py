"""Timed cases of the paged key/value cache and of the attention that reads it.

A serving program keeps the keys and values of many requests in one pool of
pages.  Each step it gives every request the pages that its new tokens need
and maps those tokens to slots (``tables``), writes their keys and values
there (``write``), and attends: each token to a prefix that all requests share
and that the pool holds once, and to its own request's tokens up to itself
(``attention``).

Layout: the pools are [pages, kv heads, page size, head dim] ("head") or
[pages, page size, kv heads, head dim] ("token"); slot s is place s % page
size of page s // page size.  The shapes are those of the Llama-2-7B-shaped
decode layers of the benchmark (32 heads of 128), of grouped heads, and ragged
ones between them.
"""
import functools
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# ---- cases -----------------------------------------------------------------


def listed():
    return [
        # One decode step's tables: 64 requests, one new token each; latency.
        {"name": "tables_step_b64", "kind": "tables", "B": 64, "page": 16, "cached": 1024, "added_lo": 1, "added": 1},
        # A burst of fresh prompts, 0 to 512 tokens each, as an offline batch starts.
        {"name": "tables_prompts_b2048", "kind": "tables", "B": 2048, "page": 16, "cached": 0, "added_lo": 0,
         "added": 512},
        # One decode step's keys and values, float32 out of the products, into a
        # bf16 cache of 32 heads.
        {"name": "write_step_t64", "kind": "write", "T": 64, "heads": 32, "dim": 128, "page": 16, "layout": "head",
         "src": "f32", "cache": "bf16"},
        # A chunk of prompts with odd sizes, token-major pages of 24.
        {"name": "write_odd_t1001", "kind": "write", "T": 1001, "heads": 5, "dim": 80, "page": 24, "layout": "token",
         "src": "f16", "cache": "f16"},
        # A large chunk of prompts.
        {"name": "write_prompts_t16384", "kind": "write", "T": 16384, "heads": 32, "dim": 128, "page": 16,
         "layout": "head", "src": "bf16", "cache": "bf16"},
        # The smallest step: four chats behind a short system prompt; latency.
        {"name": "attn_step_small", "kind": "attn", "B": 4, "heads": 32, "kv_heads": 32, "dim": 128, "page": 16,
         "layout": "head", "q": "bf16", "cache": "bf16", "prefix": 512, "cached": 63, "added_lo": 1, "added": 1},
        # A batch of eight with float32 activations, as the products of the
        # decode stack give them, on a bf16 cache.
        {"name": "attn_step_f32q_b8", "kind": "attn", "B": 8, "heads": 32, "kv_heads": 32, "dim": 128, "page": 16,
         "layout": "head", "q": "f32", "cache": "bf16", "prefix": 2048, "cached": 511, "added_lo": 1, "added": 1},
        # The same in float32 throughout, a longer prefix, token-major pages.
        {"name": "attn_step_f32_b8", "kind": "attn", "B": 8, "heads": 32, "kv_heads": 32, "dim": 128, "page": 32,
         "layout": "token", "q": "f32", "cache": "f32", "prefix": 4096, "cached": 1023, "added_lo": 1, "added": 1},
        # Many requests of one application behind its long instructions, every
        # query head with keys of its own.
        {"name": "attn_step_mha_b64", "kind": "attn", "B": 64, "heads": 32, "kv_heads": 32, "dim": 128, "page": 16,
         "layout": "head", "q": "bf16", "cache": "bf16", "prefix": 8192, "cached": 1023, "added_lo": 1, "added": 1},
        # The same with eight query heads to a key head and a whole document as
        # the prefix.
        {"name": "attn_step_gqa_b128", "kind": "attn", "B": 128, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "layout": "head", "q": "f16", "cache": "f16", "prefix": 16384, "cached": 2047, "added_lo": 1, "added": 1},
        # Ragged pieces of prompts (some requests have none), odd heads, pages
        # and lengths.
        {"name": "attn_prompts_odd", "kind": "attn", "B": 9, "heads": 15, "kv_heads": 5, "dim": 80, "page": 24,
         "layout": "token", "q": "bf16", "cache": "bf16", "prefix": 1111, "cached": 150, "added_lo": 0, "added": 70},
        # The first pass over the requests' own prompts behind the prefix.
        {"name": "attn_prompts_gqa", "kind": "attn", "B": 16, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "layout": "head", "q": "bf16", "cache": "bf16", "prefix": 4096, "cached": 0, "added_lo": 1, "added": 512},
    ]


def draw(rng):
    """One more case of the listed kinds, sizes over their whole ranges."""
    top = {}  # the largest listed work of each kind
    for c in listed():
        w, t = work(c), top.setdefault(c["kind"], {"bytes": 0, "flops": 0})
        top[c["kind"]] = {k: max(t[k], w[k]) for k in t}

    def size(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        if n >= 64 and rng.random() < 0.5:  # half of the sizes round, half ragged
            n = n // 64 * 64
        return min(max(n, lo), hi)

    kind = rng.choice(["tables", "write", "attn", "attn", "attn"])
    while True:
        c = {"kind": kind, "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 100])}
        if kind == "tables":
            c |= {"B": size(1, 2048), "cached": rng.choice([0, size(1, 4096)])}
            c |= rng.choice([{"added_lo": 1, "added": 1}, {"added_lo": 0, "added": size(2, 2048)}])
        else:
            c |= {"dim": rng.choice([64, 80, 96, 128, 128]), "layout": rng.choice(["head", "token"])}
            c["page"] = max(c["page"], 8)
        if kind == "write":
            c |= {"T": size(1, 16384), "heads": rng.choice([1, 4, 5, 8, 32]),
                  "cache": rng.choice(["f32", "f16", "bf16", "bf16"])}
            c["src"] = rng.choice(["f32", c["cache"]])
        if kind == "attn":
            kv = rng.choice([1, 5, 8, 12, 32])
            c |= {"B": size(1, 128), "kv_heads": kv, "heads": kv * (1 if kv > 8 else rng.choice([1, 3, 4, 8])),
                  "cache": rng.choice(["f32", "f16", "bf16", "bf16"]), "prefix": rng.choice([0, size(1, 16384), size(1, 16384)]),
                  "cached": rng.choice([0, size(1, 2047)])}
            c["q"] = rng.choice(["f32", c["cache"], c["cache"]])
            c |= rng.choice([{"added_lo": 1, "added": 1}, {"added_lo": 1, "added": 1},
                             {"added_lo": 0, "added": size(2, 512)}])
            if _plain_bytes(c) > 12e9:  # the plain form's padded arrays
                continue
        w = work(c)
        if all(w[k] <= top[kind][k] for k in w):
            return c


def _spread(lo, hi, n):
    """n lengths from lo to hi, evenly apart; hi alone where n is 1."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case):
    """(cached, added) of each request, before prepare() shuffles the requests."""
    B = case["B"]
    cached = _spread(0, case["cached"], B)
    added = _spread(case["added_lo"], case["added"], B)
    # many cached tokens do not mean many new ones
    return cached, [added[i * _step(B) % B] for i in range(B)]


def _step(n):
    """A step that visits all of 0 .. n - 1, about 0.62 n."""
    return next(s for s in range(max(1, int(0.618 * n)), n + 1) if math.gcd(s, n) == 1)


def _esize(t):
    return 4 if t == "f32" else 2


def _plain_bytes(c):
    cached, added = _lengths(c)
    rows, W = c["heads"] * max(1, sum(added)), max(a + b for a, b in zip(cached, added)) + c["page"]
    padded = c["B"] * W * (c["kv_heads"] * c["dim"] * 4 + c["heads"] * max(added) * 4)
    return 3 * (rows * c["prefix"] * 4 + padded)


def work(case):
    k = case["kind"]
    if k == "tables":
        cached, added = _lengths(case)
        p = case["page"]
        new = sum(-(-(a + b) // p) - -(-a // p) for a, b in zip(cached, added))
        last = sum(1 for a, b in zip(cached, added) if b and a % p)  # pages that go on being filled
        return {"bytes": 8 * case["B"] + 8 * new + 4 * last + 8 * sum(added) + 8 * case["B"] + 16, "flops": 0}
    if k == "write":
        n = 2 * case["T"] * case["heads"] * case["dim"]
        return {"bytes": n * (_esize(case["src"]) + _esize(case["cache"])) + 8 * case["T"], "flops": 0}
    cached, added = _lengths(case)
    T = sum(added)
    seen = sum(b * case["prefix"] + b * a + b * (b + 1) // 2 for a, b in zip(cached, added))
    keys = case["prefix"] + sum(a + b for a, b in zip(cached, added) if b)
    return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * _esize(case["cache"])
            + 2 * T * case["heads"] * case["dim"] * _esize(case["q"]) + 4 * -(-keys // case["page"]) + 8 * case["B"],
            "flops": 4 * case["dim"] * case["heads"] * seen}


# ---- inputs ----------------------------------------------------------------


def _generator(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    return g


def _normal(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float32).to(dtype)


def _i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _pools(case, pages, heads, gen):
    """Key and value pools, as [pages, heads, page size, dim] views of either layout."""
    shape = (pages, heads, case["page"], case["dim"])
    if case["layout"] == "token":
        shape = (pages, case["page"], heads, case["dim"])
    pools = [_normal(shape, TYPES[case["cache"]], gen) for _ in range(2)]
    return [p.transpose(1, 2) if case["layout"] == "token" else p for p in pools]


def _requests(case, seed):
    """cached, added and their sums on the host, in the seed's order."""
    cached, added = _lengths(case)
    order = torch.randperm(case["B"], generator=_generator(seed, "cpu")).tolist()
    return [cached[i] for i in order], [added[i] for i in order]


def _tables(case, counts, width, first_page, pages, seed, device):
    """Block table of `counts` pages a request, ids shuffled among first_page .. pages - 1, and the ids left over."""
    ids = torch.randperm(pages - first_page, generator=_generator(seed + 1, "cpu")) + first_page
    counts = torch.tensor(counts)
    col = torch.arange(width)[None, :]
    used = col < counts[:, None]
    table = torch.full((len(counts), width), -1, dtype=torch.int64)
    table[used] = ids[:int(counts.sum())]
    return table.to(torch.int32).to(device), ids[int(counts.sum()):].to(torch.int32).to(device)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = _generator(seed, device)
    k, page = case["kind"], case["page"]
    s = {"kind": k, "case": case}
    if k == "write":
        T, heads, dim = case["T"], case["heads"], case["dim"]
        pages = -(-T // page) * 2 + 3
        s["k_pool"], s["v_pool"] = _pools(case, pages, heads, gen)
        s["k"], s["v"] = (_normal((T, heads, dim), TYPES[case["src"]], gen) for _ in range(2))
        # tokens of several requests: runs of slots within pages in any order,
        # every 50th token is padding
        place = torch.randperm(pages, generator=_generator(seed, "cpu"))[:-(-T // page)]
        slots = (place[:, None] * page + torch.arange(page)[None, :]).reshape(-1)[:T]
        slots[49::50] = -1
        s["slots"] = slots.to(device)
        if own:
            s["cache"] = _cache(case, s)
        return s
    cached, added = _requests(case, seed)
    B, T = case["B"], sum(added)
    have = [-(-a // page) for a in cached]
    need = [-(-(a + b) // page) for a, b in zip(cached, added)]
    if k == "tables":
        pages = sum(need) + 64
        s["table"], s["free"] = _tables(case, have, max(max(need), 1), 0, pages, seed, device)
        s["cached"], s["added"] = _i32(cached, device), _i32(added, device)
        s["head"] = _i32([7], device)
        s["tokens"] = T + 5  # a little room, as a program with fixed buffers has
        s["out"] = (torch.empty(s["tokens"], dtype=torch.int64, device=device),
                    torch.empty(B + 1, dtype=torch.int32, device=device),
                    torch.empty(B, dtype=torch.int32, device=device), torch.empty(1, dtype=torch.int32, device=device),
                    torch.empty(1, dtype=torch.int32, device=device))
        return s
    prefix_pages = -(-case["prefix"] // page)
    pages = prefix_pages + sum(need) + 1
    s["k_pool"], s["v_pool"] = _pools(case, pages, case["kv_heads"], gen)
    s["q"] = _normal((T, case["heads"], case["dim"]), TYPES[case["q"]], gen)
    s["out"] = torch.empty_like(s["q"])
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    s["prefix_table"] = torch.randperm(max(prefix_pages, 1), generator=_generator(seed + 2, "cpu")).to(torch.int32).to(device)
    s["table"], _ = _tables(case, need, max(max(need), 1), prefix_pages, pages, seed, device)
    s["lengths"] = _i32([a + b for a, b in zip(cached, added)], device)
    s["start"] = _i32([0] + torch.tensor(added).cumsum(0).tolist(), device)
    # what the program's scheduler knows on the host
    s["max_added"], s["max_length"] = max(added), max(a + b for a, b in zip(cached, added))
    if own:
        s["cache"] = _cache(case, s)
    return s


# ---- plain forms -----------------------------------------------------------


def _plain_tables(s):
    page, cached, added = s["case"]["page"], s["cached"].long(), s["added"].long()
    table, device = s["table"].clone(), s["table"].device
    have, need = (cached + page - 1) // page, (cached + added + page - 1) // page
    before = torch.cumsum(need - have, 0) - (need - have)
    col = torch.arange(table.shape[1], device=device)[None, :]
    new = (col >= have[:, None]) & (col < need[:, None])
    entry = (s["head"].long() + before[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    table = torch.where(new, s["free"][entry], table)
    ends = torch.cumsum(added, 0)
    t = torch.arange(s["tokens"], device=device)
    b = torch.searchsorted(ends, t, right=True).clamp(max=len(added) - 1)
    pos = cached[b] + t - (ends - added)[b]
    block = (pos // page).clamp(max=table.shape[1] - 1)
    slots = torch.where(t < ends[-1], table[b, block].long() * page + pos % page, torch.full_like(t, -1))
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    start = torch.cat([zero, ends.int()])
    head = s["head"] + (need - have).sum().int()
    return {"table": table, "slots": slots, "start": start, "lengths": (cached + added).int(), "head": head,
            "status": zero}


def _plain_write(s):
    page, slots = s["case"]["page"], s["slots"]
    kept = slots >= 0
    at, kp, vp = slots[kept], s["k_pool"], s["v_pool"]
    kp[at // page, :, at % page] = s["k"][kept].float().to(kp.dtype)
    vp[at // page, :, at % page] = s["v"][kept].float().to(vp.dtype)
    return {"k": kp, "v": vp}


def _gather(pool, table):
    """[..., kv heads, keys, dim] in float32 of the pages in table [..., W]."""
    x = pool[table.long().clamp(min=0)]  # [..., W, heads, page, dim]
    x = x.movedim(-3, -4)
    return x.reshape(*x.shape[:-3], x.shape[-3] * x.shape[-2], x.shape[-1]).float()


def _plain_attention(s):
    c = s["case"]
    H, D, P, B = c["kv_heads"], c["dim"], c["prefix"], c["B"]
    G, T, N = c["heads"] // c["kv_heads"], s["q"].shape[0], s["max_added"]
    device = s["q"].device
    q = s["q"].float().view(T, H, G, D) * s["scale"]
    start, lengths = s["start"].long(), s["lengths"].long()
    t = torch.arange(T, device=device)
    b = torch.searchsorted(start, t, right=True) - 1  # the token's request
    i = t - start[b]
    # the prefix, for every token
    kp, vp = (_gather(s[n], s["prefix_table"])[:, :P] for n in ("k_pool", "v_pool"))
    qp = q.permute(1, 0, 2, 3).reshape(H, T * G, D)
    sp = torch.matmul(qp, kp.transpose(1, 2))
    # each request's own keys, padded to the longest
    ks, vs = (_gather(s[n], s["table"]) for n in ("k_pool", "v_pool"))
    L = ks.shape[2]
    at = (start[:-1, None] + torch.arange(N, device=device)[None, :]).clamp(max=T - 1)
    qs = q[at].permute(0, 2, 1, 3, 4).reshape(B, H, N * G, D)
    ss = torch.matmul(qs, ks.transpose(2, 3)).view(B, H, N, G, L)
    ss = ss.permute(0, 2, 1, 3, 4)[b, i]  # [T, H, G, L]
    key = torch.arange(L, device=device)
    pos = lengths[b] - (start[1:] - start[:-1])[b] + i
    ss = ss.masked_fill((key[None, :] > pos[:, None])[:, None, None, :], -math.inf)
    ss = ss.permute(1, 0, 2, 3).reshape(H, T * G, L)
    m = ss.amax(2, keepdim=True)
    if P:
        m = torch.maximum(m, sp.amax(2, keepdim=True))
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    ep, es = torch.exp(sp - m), torch.exp(ss - m)
    total = ep.sum(2, keepdim=True) + es.sum(2, keepdim=True)
    op = torch.matmul(ep, vp)
    # back to the padded form for the products with each request's values
    pad = torch.zeros(B, N, H, G, L, device=device)
    pad[b, i] = es.view(H, T, G, L).permute(1, 0, 2, 3)
    vs = vs.masked_fill((key[None, :] >= lengths[:, None])[:, None, :, None], 0.0)
    os = torch.matmul(pad.permute(0, 2, 1, 3, 4).reshape(B, H, N * G, L), vs)
    os = os.view(B, H, N, G, D).permute(0, 2, 1, 3, 4)[b, i]
    o = op.view(H, T, G, D).permute(1, 0, 2, 3) + os
    total = total.view(H, T, G, 1).permute(1, 0, 2, 3)
    o = torch.where(total == 0, torch.zeros_like(o), o / total)
    return o.reshape(T, H * G, D).to(s["q"].dtype)


# ---- the framework's operators -----------------------------------------------


@functools.lru_cache(maxsize=1)
def _ctx():
    from pyflamert_amd import rocm

    return rocm.Context(torch.cuda.current_device())


def _cache(case, s):
    """The handle of the pools that a program binds once."""
    kp, vp = s["k_pool"], s["v_pool"]
    pages, heads, page, dim = kp.shape
    return _ctx().kv_bind(kp.data_ptr(), vp.data_ptr(), case["cache"], pages, page, heads, dim,
                          page_stride=kp.stride(0), head_stride=kp.stride(1), token_stride=kp.stride(2))


def _own(s):
    ctx, c = _ctx(), s["case"]
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    if s["kind"] == "tables":
        slots, start, lengths, head, status = s["out"]
        ctx.kv_tables_dev(s["cached"].data_ptr(), s["added"].data_ptr(), c["B"], c["page"], s["free"].data_ptr(),
                          s["free"].numel(), s["head"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1],
                          slots.data_ptr(), s["tokens"], start.data_ptr(), lengths.data_ptr(), head.data_ptr(),
                          status.data_ptr())
        return {"table": s["table"], "slots": slots, "start": start, "lengths": lengths, "head": head,
                "status": status}
    if s["kind"] == "write":
        s["cache"].write_dev(s["k"].data_ptr(), s["v"].data_ptr(), c["T"], s["slots"].data_ptr(), c["src"])
        return {"k": s["k_pool"], "v": s["v_pool"]}
    s["cache"].attention_dev(s["q"].data_ptr(), s["q"].shape[0], c["heads"], s["out"].data_ptr(), c["q"], s["scale"],
                             prefix_table_ptr=s["prefix_table"].data_ptr(), prefix_len=c["prefix"],
                             table_ptr=s["table"].data_ptr(), table_w=s["table"].shape[1], B=c["B"],
                             lengths_ptr=s["lengths"].data_ptr(), start_ptr=s["start"].data_ptr(),
                             max_added=s["max_added"], max_length=s["max_length"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"tables": _plain_tables, "write": _plain_write, "attn": _plain_attention}[state["kind"]](state)


# ---- from the definitions, in 64 bits ----------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return None  # whole numbers
    if case["kind"] == "write":
        out = {}
        slots = s["slots"].tolist()
        rows = torch.tensor([t for t, x in enumerate(slots) if x >= 0], device="cuda")
        flat = torch.tensor([x for x in slots if x >= 0], device="cuda")
        for name in ("k", "v"):
            pool = s[name + "_pool"]
            pages, heads, page, dim = pool.shape
            by_slot = pool.double().transpose(1, 2).reshape(pages * page, heads, dim)
            by_slot.index_copy_(0, flat, s[name].double()[rows])
            out[name] = by_slot.view(pages, page, heads, dim).transpose(1, 2)
        return out
    H, G, page = case["kv_heads"], case["heads"] // case["kv_heads"], case["page"]

    def keys(pool, pages, n):
        x = pool[pages.long()].double().transpose(1, 2)  # [W, page, H, D]
        return x.reshape(-1, H, case["dim"])[:n].transpose(0, 1).contiguous()  # [H, n, D]

    start, lengths = s["start"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    shared = [keys(s[n], s["prefix_table"], case["prefix"]) for n in ("k_pool", "v_pool")]
    for r in range(case["B"]):
        n, length = start[r + 1] - start[r], lengths[r]
        if n == 0:
            continue
        pages = s["table"][r, :-(-length // page)]
        mine = [keys(s[name], pages, length) for name in ("k_pool", "v_pool")]
        q = s["q"][start[r]:start[r + 1]].double().view(n, H, G, -1).permute(1, 2, 0, 3).reshape(H, G * n, -1)
        score = torch.cat([q @ x.transpose(1, 2) for x in (shared[0], mine[0])], 2) * s["scale"]
        last = torch.arange(length - n, length, device="cuda").repeat(G)  # the last key of each row
        place = torch.cat([torch.full((case["prefix"],), -1, device="cuda"), torch.arange(length, device="cuda")])
        score.masked_fill_(place[None, None, :] > last[None, :, None], -math.inf)
        p = torch.softmax(score, 2)
        o = p[:, :, :case["prefix"]] @ shared[1] + p[:, :, case["prefix"]:] @ mine[1]
        out[start[r]:start[r + 1]] = o.view(H, G, n, -1).permute(2, 0, 1, 3).reshape(n, H * G, -1)
    return out
