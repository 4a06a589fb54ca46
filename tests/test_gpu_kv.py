"""The paged key/value cache on the GPU: tables, writes and attention against
their definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx():
    from pyflamert_amd import rocm

    c = rocm.Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    torch.cuda.synchronize()
    c.close()


def i32(x):
    return torch.tensor(np.asarray(x, np.int64), dtype=torch.int64).to(torch.int32).to(DEV)


# ---- block tables and slot maps ---------------------------------------------


def run_tables(ctx, cached, added, page, free, head, table_w, max_tokens, pad=3, no_head=False):
    B = len(cached)
    rng = np.random.default_rng(B + page)
    table = rng.integers(0, 1000, (B, table_w + pad)).astype(np.int32)
    td = torch.from_numpy(table.copy()).to(DEV)
    slots = torch.full((max_tokens + 2,), 77, dtype=torch.int64, device=DEV)
    start, lengths = torch.full((B + 3,), 77, dtype=torch.int32, device=DEV), torch.full((B + 2,), 77, dtype=torch.int32, device=DEV)
    tail = torch.full((4,), 77, dtype=torch.int32, device=DEV)
    c, a, f, h = i32(cached), i32(added), i32(free), i32([head])
    for _ in range(2):  # the same inputs give the same outputs again
        ctx.kv_tables_dev(c.data_ptr(), a.data_ptr(), B, page, f.data_ptr(), len(free), None if no_head else h.data_ptr(),
                          td.data_ptr(), table_w, slots.data_ptr(), max_tokens, start.data_ptr(), lengths.data_ptr(),
                          tail[0:1].data_ptr(), tail[2:3].data_ptr(), table_ld=table_w + pad)
    torch.cuda.synchronize()
    want = R.tables(cached, added, page, free, 0 if no_head else head, table[:, :table_w], table_w, max_tokens)
    got = td.cpu().numpy()
    assert np.array_equal(got[:, :table_w], want[0])
    assert np.array_equal(got[:, table_w:], table[:, table_w:])
    assert np.array_equal(slots[:max_tokens].cpu().numpy(), want[1]) and slots[max_tokens:].tolist() == [77, 77]
    assert np.array_equal(start[:B + 1].cpu().numpy(), want[2]) and start[B + 1:].tolist() == [77, 77]
    assert np.array_equal(lengths[:B].cpu().numpy(), want[3]) and lengths[B:].tolist() == [77, 77]
    assert tail.tolist() == [want[4], 77, want[5], 77]
    return want


@pytest.mark.parametrize("B,page,cached,added", [
    (1, 16, 0, 1), (1, 16, 16, 1), (1, 1, 5, 7), (3, 24, 100, 0), (64, 16, 1024, 1), (255, 16, 40, 5), (256, 100, 300, 9),
    (257, 7, 30, 40), (700, 16, 0, 20), (5, 64, 3, 5000), (2, 1 << 20, 9, 3),
])
def test_tables(ctx, B, page, cached, added):
    rng = np.random.default_rng(7 * B + page)
    c = rng.integers(0, cached + 1, B)
    a = rng.integers(0, added + 1, B)
    a[-1] = added
    need = [-(-(x + y) // page) for x, y in zip(c, a)]
    free = rng.permutation(sum(need) + 30)
    st = run_tables(ctx, c, a, page, free, 11, max(max(need), 1), int(a.sum()) + 9)
    assert st[5] == 0


def test_tables_no_requests(ctx):
    run_tables(ctx, [], [], 16, [3, 4], 1, 2, 5)


@pytest.mark.parametrize("case,bits", [("pages", 1), ("width", 2), ("slots", 4), ("count", 8), ("overflow", 8), ("head", 8),
                                       ("low head", 8), ("all", 15)])
def test_tables_what_does_not_fit(ctx, case, bits):
    """What is asked for too much shows in the status; the rest is as it should be."""
    rng = np.random.default_rng(3)
    B, page = 300, 16
    c, a = rng.integers(0, 60, B), rng.integers(0, 60, B)
    if case in ("count", "all"):
        c[7], a[270] = -5, -1
    if case == "overflow":
        c[299], a[299] = 2 ** 31 - 1, 5
    need = sum(-(-max(x + y, 0) // page) for x, y in zip(c[:299], a[:299])) + 10
    free = rng.permutation(need)
    width = 4 if case in ("width", "all") else 9
    if case in ("pages", "all"):
        free = free[:200]
    tokens = 3000 if case in ("slots", "all") else int(a.clip(0).sum()) + 5
    head = {"head": len(free) + 4, "low head": -3}.get(case, 0)
    st = run_tables(ctx, c, a, page, free, head, width, tokens)
    assert st[5] & bits == bits


def test_tables_default_head_and_empty_list(ctx):
    run_tables(ctx, [5, 0], [3, 2], 4, [9, 8, 7, 6], 0, 4, 8, no_head=True)
    st = run_tables(ctx, [5, 0], [3, 2], 8, [], 0, 4, 8)
    assert st[5] == 1


# ---- writes -------------------------------------------------------------------


def pools(shape, layout, dtype, gen, pad=0):
    """Two pools as [pages, heads, page, dim] views of a layout."""
    pages, heads, page, dim = shape
    out = []
    for _ in range(2):
        if layout == "token":
            p = torch.randn(pages, page, heads, dim, generator=gen).to(R.TORCH[dtype]).to(DEV).transpose(1, 2)
        else:
            p = torch.randn(pages, heads, page, dim + pad, generator=gen).to(R.TORCH[dtype]).to(DEV)[..., :dim]
        out.append(p)
    return out


def bind(ctx, kp, vp, dtype):
    pages, heads, page, dim = kp.shape
    assert kp.stride() == vp.stride() and kp.stride(3) == 1
    return ctx.kv_bind(kp.data_ptr(), vp.data_ptr(), dtype, pages, page, heads, dim, page_stride=kp.stride(0),
                       head_stride=kp.stride(1), token_stride=kp.stride(2))


def bits(x):
    return x.contiguous().view(torch.int32 if x.element_size() == 4 else torch.int16)


@pytest.mark.parametrize("src,dtype", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("T,heads,dim,page,layout", [
    (1, 1, 8, 1, "head"), (1, 32, 128, 16, "head"), (7, 3, 80, 24, "token"), (65, 5, 256, 16, "head"), (333, 2, 72, 7, "token"),
])
def test_write(ctx, src, dtype, T, heads, dim, page, layout):
    gen = torch.Generator().manual_seed(T * dim)
    pages = T // page + 5
    kp, vp = pools((pages, heads, page, dim), layout, dtype, gen, pad=8)
    want_k, want_v = kp.cpu(), vp.cpu()
    slots = torch.randperm(pages * page, generator=gen)[:T]
    if T > 5:
        slots[2], slots[3], slots[4] = -1, pages * page, -2 ** 62
    # keys and values inside one fused row, at an offset that is not 16-byte aligned
    row = heads * dim
    fused = (torch.randn(T, 2 * row + 5, generator=gen) * 3).to(R.TORCH[src])
    fused[0, 1], fused[0, row + 2], fused[0, 3] = math.inf, math.nan, 1e30 if src == "f32" else 1.0
    k = fused[:, 1:1 + row].reshape(T, heads, dim)
    v = fused[:, 2 + row:2 + 2 * row].reshape(T, heads, dim)
    for t in range(T):
        s = int(slots[t])
        if 0 <= s < pages * page:
            want_k[s // page, :, s % page] = k[t].to(R.TORCH[dtype])
            want_v[s // page, :, s % page] = v[t].to(R.TORCH[dtype])
    d = fused.to(DEV)
    cache = bind(ctx, kp, vp, dtype)
    sd = slots.to(DEV)
    es = d.element_size()
    cache.write_dev(d.data_ptr() + es, d.data_ptr() + (2 + row) * es, T, sd.data_ptr(), src, ldk=2 * row + 5, ldv=2 * row + 5)
    torch.cuda.synchronize()
    for got, want in ((kp.cpu(), want_k), (vp.cpu(), want_v)):
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(bits(got.masked_fill(nan, 0)), bits(want.masked_fill(nan, 0)))
    cache.free()


# ---- attention ------------------------------------------------------------------


class Case:
    """Pools, tables and queries of a batch; attributes may be changed before run()."""

    def __init__(self, heads, kv_heads, dim, page, layout, q, cache, prefix, lengths, added, seed=0, spare=0.0):
        gen = torch.Generator().manual_seed(seed + 1000 * heads + dim)
        self.qtype, self.ctype, self.prefix, self.page, self.heads = q, cache, prefix, page, heads
        B = len(lengths)
        pp = -(-prefix // page)
        per = [-(-n // page) for n in lengths]
        pages = pp + sum(per) + 2
        kp, vp = pools((pages, kv_heads, page, dim), layout, cache, gen)
        self.kp, self.vp = kp, vp
        ids = torch.randperm(pages, generator=gen).tolist()
        self.prefix_table = np.array(ids[:pp] or [0], np.int32)
        w = max(per + [1]) + 1
        self.table = np.full((B, w), -1, np.int32)
        at = pp
        for b, n in enumerate(per):
            self.table[b, :n] = ids[at:at + n]
            at += n
        # whatever no key occupies holds NaN or infinities
        used = torch.zeros(pages, page, dtype=torch.bool)
        for tab, n in [(self.prefix_table, prefix)] + list(zip(self.table, lengths)):
            for key in range(n):
                used[tab[key // page], key % page] = True
        hole = ~used[:, None, :, None].expand(pages, kv_heads, page, dim)
        self.kp.masked_fill_(hole.to(DEV), math.nan)
        self.vp.masked_fill_(hole.to(DEV), math.inf)
        self.lengths = np.array(lengths, np.int32)
        self.start = np.concatenate([[0], np.cumsum(added)]).astype(np.int32)
        self.T = int(self.start[-1])
        self.q = torch.randn(self.T, heads, dim, generator=gen).to(R.TORCH[q]).to(DEV)
        self.scale = dim ** -0.5
        self.max_added, self.max_length = max(list(added) + [0]), max(list(lengths) + [0])

    def slot_of(self, b, key):
        return int(self.table[b, key // self.page]), key % self.page

    def run(self, ctx, fused=True):
        T, heads, dim = self.q.shape
        B = len(self.lengths)
        # queries and outputs within wider rows
        qrow = torch.full((T, heads * dim + 3), math.nan, dtype=self.q.dtype, device=DEV)
        qrow[:, 3:] = self.q.reshape(T, -1)
        out = torch.full((T, heads * dim + 5), 7.0, dtype=self.q.dtype, device=DEV)
        cache = bind(ctx, self.kp, self.vp, self.ctype)
        pt, tab, ln, st = i32(self.prefix_table), i32(self.table), i32(self.lengths), i32(self.start)
        es = self.q.element_size()
        cache.attention_dev(qrow.data_ptr() + 3 * es, T, heads, out.data_ptr() + 2 * es, self.qtype, self.scale,
                            prefix_table_ptr=pt.data_ptr(), prefix_len=self.prefix, table_ptr=tab.data_ptr(),
                            table_w=self.table.shape[1], B=B, lengths_ptr=ln.data_ptr(), start_ptr=st.data_ptr(),
                            max_added=self.max_added, max_length=self.max_length, ldq=heads * dim + 3, ldo=heads * dim + 5)
        torch.cuda.synchronize()
        cache.free()
        o = out.cpu()
        assert bool((o[:, :2] == 7).all()) and bool((o[:, 2 + heads * dim:] == 7).all())
        return o[:, 2:2 + heads * dim].reshape(T, heads, dim)

    def want(self):
        return R.attention(self.q.cpu(), self.kp.cpu(), self.vp.cpu(), self.scale, self.prefix_table, self.prefix,
                           self.table, self.lengths, self.start, self.qtype)

    def check(self, ctx):
        got = self.run(ctx)
        want, bound = self.want()
        same(got, want, bound)
        return got


def same(got, want, bound):
    g = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(g[inf], want[inf])
    over = (g[fin] - want[fin]).abs() - bound[fin]
    assert bool((over <= 0).all()), "off by up to %.3g times its bound" % float(
        ((g[fin] - want[fin]).abs() / bound[fin].clamp(min=1e-30)).max())


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")]
SHAPES = {
    # heads, kv heads, dim, page, layout, prefix, lengths, added
    "one token, one key": (1, 1, 64, 16, "head", 0, [1], [1]),
    "prefix alone": (2, 1, 128, 16, "head", 33, [1], [1]),
    "step": (4, 4, 128, 16, "head", 200, [1, 17, 64, 300], [1, 1, 1, 1]),
    "step, grouped heads": (24, 3, 64, 32, "token", 129, [5, 90, 31], [1, 1, 1]),
    "step, many rows a tile": (8, 2, 128, 16, "head", 100, [3, 8, 2, 33, 12, 40, 7, 9, 1, 6], [1] * 10),
    "odd pages": (6, 2, 80, 24, "token", 111, [20, 70, 49], [3, 0, 7]),
    "page of one": (2, 2, 72, 1, "head", 5, [9, 2], [2, 2]),
    "page of seven": (2, 1, 96, 7, "head", 65, [40, 13], [1, 5]),
    "prompts": (4, 2, 128, 16, "head", 70, [50, 130, 19], [50, 33, 2]),
    "prompts, no prefix": (4, 1, 64, 16, "head", 0, [65, 1, 40], [65, 1, 37]),
    "small heads": (3, 3, 8, 16, "head", 40, [33, 9], [1, 4]),
    "wide heads": (4, 2, 256, 16, "head", 70, [20, 45], [1, 9]),
    "wide odd heads": (2, 2, 200, 16, "token", 33, [20, 35], [1, 2]),
    "long": (2, 1, 128, 16, "head", 3000, [1500, 700], [1, 1]),
    "rows of one tile and a bit": (20, 1, 128, 16, "head", 90, [40, 7], [1, 1]),
    "prefix of many rows": (8, 2, 128, 16, "head", 700, [9, 1, 40, 33] * 6, [1] * 24),
    "many requests": (8, 1, 64, 16, "head", 300, [1 + 7 * i % 90 for i in range(100)], [1] * 100),
    "many requests, no prefix": (2, 2, 128, 16, "token", 0, [1 + 7 * i % 90 for i in range(70)], [1] * 70),
    "prefix of many rows, odd dim": (6, 1, 72, 7, "token", 333, [9, 1, 40, 33] * 3, [1] * 12),
    "prefix and own keys of many rows": (8, 1, 64, 16, "token", 1100, [40, 330, 25], [9, 6, 30]),
    "many rows a request": (8, 1, 64, 16, "head", 130, [230, 95], [200, 90]),
    "many rows a request, odd dim": (4, 2, 80, 24, "token", 70, [250, 180], [250, 170]),
    "many rows a request, no prefix": (8, 1, 128, 16, "head", 0, [130, 200], [130, 100]),
    "many rows a request, longer than a window": (16, 1, 96, 1, "head", 2500, [90, 1300], [30, 20]),
    "one long request": (4, 1, 128, 16, "head", 200, [900, 5, 3], [300, 4, 1]),
}


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("name", SHAPES)
def test_attention(ctx, name, q, cache):
    heads, kvh, dim, page, layout, prefix, lengths, added = SHAPES[name]
    Case(heads, kvh, dim, page, layout, q, cache, prefix, lengths, added).check(ctx)


@pytest.mark.parametrize("q,cache", TYPES[:4])
@pytest.mark.parametrize("how", ["step", "prompt"])
def test_attention_rows_without_keys(ctx, q, cache, how):
    """Requests of length zero, tokens before the first key, and scores that are
    all -inf give zeros; tokens past start[B] see the prefix only."""
    added = [1, 1, 1] if how == "step" else [20, 4, 1]
    c = Case(4, 2, 128, 16, "head", q, cache, 0, [0, 3, 9], added)
    got = c.check(ctx)
    assert bool((got[:added[0]] == 0).all())
    c = Case(4, 2, 128, 16, "head", q, cache, 0, [4, 3, 9], added)
    c.q[...] = c.q.abs() + 0.5
    for key in range(4):
        p, off = c.slot_of(0, key)
        c.kp[p, :, off] = -math.inf
    got = c.check(ctx)
    assert bool((got[:added[0]] == 0).all())
    c = Case(4, 2, 128, 16, "head", q, cache, 21, [4, 3, 9], added)
    c.start = c.start[:3].copy()
    c.lengths, c.table = c.lengths[:2], c.table[:2]
    c.check(ctx)
    c.start, c.lengths, c.table = np.zeros(1, np.int32), np.zeros(0, np.int32), np.zeros((0, 1), np.int32)
    c.check(ctx)


@pytest.mark.parametrize("q,cache", TYPES[:2])
def test_attention_of_many_rows_where_keys_are_missing(ctx, q, cache):
    """Rows without keys, tokens of no request and pages outside the pool, where a
    request has many rows."""
    c = Case(8, 1, 64, 16, "head", q, cache, 0, [0, 60, 90], [40, 100, 30])
    got = c.check(ctx)
    assert bool((got[:40] == 0).all()) and bool((got[40:80] == 0).all())  # 60 keys of 100 tokens: 40 before the first
    for prefix in (0, 150):
        c = Case(8, 1, 128, 16, "token", q, cache, prefix, [130, 90, 33], [100, 60, 20])
        c.table[0, 1] = -1
        c.table[1, :] = 2 ** 31 - 1
        if prefix:
            c.prefix_table[2] = c.kp.shape[0]
        c.check(ctx)
        # the last request's tokens are of none; then the first 100 as well
        c.lengths, c.table, c.start = c.lengths[:2], c.table[:2], c.start[:3].copy()
        c.check(ctx)
        c.lengths, c.table, c.start = c.lengths[1:], c.table[1:], c.start[1:].copy()
        c.check(ctx)


@pytest.mark.parametrize("q,cache", TYPES[:2])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_attention_of_many_rows_later_keys(ctx, q, cache, value):
    """An infinity or a NaN in a late value reaches the tokens that see it, in its
    column, and no others, across tiles of rows and of keys."""
    def case():
        return Case(8, 1, 128, 16, "head", q, cache, 40, [290, 9], [260, 3])

    clean = case().run(ctx)
    for key in (31, 64, 200, 289):  # token key - 30 of request 0 is the first that sees it
        c = case()
        p, off = c.slot_of(0, key)
        c.vp[p, :, off, 77] = value
        got = c.run(ctx)
        first = key - 30
        assert torch.equal(bits(got[:first]), bits(clean[:first])) and torch.equal(bits(got[260:]), bits(clean[260:]))
        assert bool((~torch.isfinite(got[first:260, :, 77])).all())
        rest = torch.arange(128) != 77
        assert torch.equal(bits(got[first:260][..., rest]), bits(clean[first:260][..., rest]))


@pytest.mark.parametrize("q,cache", TYPES[:4])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_attention_later_keys_do_not_reach_earlier_tokens(ctx, q, cache, value):
    """An infinity or a NaN in a key or a value reaches the tokens that see it, and no others."""
    for which in ("k", "v"):
        c = Case(4, 2, 128, 16, "head", q, cache, 40, [70, 9], [35, 3])
        for b, key in ((0, 36), (0, 50), (0, 69), (1, 8)):
            p, off = c.slot_of(b, key)
            (c.kp if which == "k" else c.vp)[p, :, off, 3] = value
        got = c.run(ctx)
        clean = Case(4, 2, 128, 16, "head", q, cache, 40, [70, 9], [35, 3]).run(ctx)
        # token 0 of request 0 sees keys 0 .. 35, request 1's tokens 0 and 1 see up to 7
        for t in (0, 35, 36):
            assert torch.equal(bits(got[t]), bits(clean[t])), (which, t)
        hit = got[[1, 20, 34, 37]]
        if which == "v":
            assert bool((~torch.isfinite(hit[..., 3])).all())
            others = torch.cat([hit[..., :3], hit[..., 4:]], -1)
            assert bool(torch.isfinite(others).all())
        elif math.isnan(value):
            assert bool(torch.isnan(hit).all())
        else:  # a score of +inf (no other weight counts, and inf - inf) or -inf
            pos = (c.q[[1, 20, 34, 37], :, 3] > 0).cpu()
            assert bool(torch.isnan(hit[pos]).all())


@pytest.mark.parametrize("q,cache", TYPES[:4])
def test_attention_missing_pages(ctx, q, cache):
    """Keys on pages outside the pool, or past the table, count as absent."""
    c = Case(4, 2, 64, 16, "head", q, cache, 100, [60, 90, 33], [1, 6, 1])
    pages = c.kp.shape[0]
    c.prefix_table[2] = -1
    c.prefix_table[5] = pages
    c.table[0, 1] = -1
    c.table[1, 3] = 2 ** 31 - 1
    c.table[2, :] = -2 ** 31
    c.check(ctx)
    c = Case(4, 2, 64, 16, "head", q, cache, 20, [60, 90], [1, 6])
    c.table = c.table[:, :2].copy()  # 32 keys
    c.check(ctx)


@pytest.mark.parametrize("max_added,max_length", [(0, 0), (1, 1), (1, 700), (64, 16)])
def test_attention_bounds_only_shape_the_launch(ctx, max_added, max_length):
    c = Case(4, 2, 128, 16, "head", "bf16", "bf16", 90, [200, 333, 64], [40, 9, 64])
    c.max_added, c.max_length = max_added, max_length
    c.check(ctx)


def test_attention_scale(ctx):
    for scale in (0.0, -0.3, 2.5):
        c = Case(4, 4, 64, 16, "head", "f32", "f32", 50, [20, 30], [1, 1])
        c.scale = scale
        c.check(ctx)


def test_attention_offsets_past_32_bits(ctx):
    """Keys in pages that lie more than 2^32 elements into the pool."""
    page, heads, dim, pages = 16, 2, 128, 40
    stride = (1 << 32) // 36 // 8 * 8  # the last pages start past 2^32 elements
    pool = torch.empty(stride * (pages - 1) + heads * page * dim, dtype=torch.bfloat16, device=DEV)
    kp = pool.as_strided((pages, heads, page, dim), (stride, page * dim, dim, 1))
    gen = torch.Generator().manual_seed(5)
    kp.copy_(torch.randn(pages, heads, page, dim, generator=gen).to(torch.bfloat16))
    assert (pages - 1) * stride > 1 << 32
    cache = ctx.kv_bind(pool.data_ptr(), pool.data_ptr(), "bf16", pages, page, heads, dim, page_stride=stride)
    q = torch.randn(1, heads, dim, generator=gen).to(torch.bfloat16)
    qd, out = q.to(DEV), torch.empty(1, heads, dim, dtype=torch.bfloat16, device=DEV)
    ptab, tab, n, st = np.array([38, 0]), np.array([[39, 37]]), [20], [0, 1]
    a, b, c, d = i32(ptab), i32(tab), i32(n), i32(st)
    # the last page's first slot, written through the cache
    k1 = torch.randn(1, heads, dim, generator=gen).to(torch.bfloat16)
    kd, slot = k1.to(DEV), torch.tensor([39 * page], device=DEV)
    cache.write_dev(kd.data_ptr(), kd.data_ptr(), 1, slot.data_ptr(), "bf16")
    cache.attention_dev(qd.data_ptr(), 1, heads, out.data_ptr(), "bf16", prefix_table_ptr=a.data_ptr(), prefix_len=30,
                        table_ptr=b.data_ptr(), table_w=2, B=1, lengths_ptr=c.data_ptr(), start_ptr=d.data_ptr())
    torch.cuda.synchronize()
    small = kp.cpu()
    assert torch.equal(bits(small[39, :, 0]), bits(k1[0]))
    same(out.cpu(), *R.attention(q, small, small, dim ** -0.5, ptab, 30, tab, n, st, "bf16"))


def test_step_on_another_stream_and_in_a_graph(ctx):
    """Tables, write and attention of a step on a stream of their own, eager and
    as a graph that is replayed with new inputs between eager work."""
    heads, kvh, dim, page, prefix = 8, 4, 64, 16, 75
    lengths = [30, 47, 16, 0]
    c = Case(heads, kvh, dim, page, "head", "bf16", "bf16", prefix, lengths, [1] * 4)
    B, pages = 4, c.kp.shape[0]
    left = [p for p in range(pages) if p not in set(c.table.ravel()) | set(c.prefix_table)]
    # room: as many pages again
    kp = torch.cat([c.kp, torch.zeros_like(c.kp)]).contiguous()
    vp = torch.cat([c.vp, torch.zeros_like(c.vp)]).contiguous()
    cache = bind(ctx, kp, vp, "bf16")
    free = i32(left + list(range(pages, 2 * pages)))
    table = i32(np.concatenate([c.table, np.full((B, 1), -1)], 1))
    w = table.shape[1]
    cached, added, head = i32(lengths), i32([1] * B), i32([0])
    slots = torch.empty(B, dtype=torch.int64, device=DEV)
    start, ln, head2, status = (torch.empty(n, dtype=torch.int32, device=DEV) for n in (B + 1, B, 1, 1))
    pt = i32(c.prefix_table)
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(B, (heads + 2 * kvh) * dim, generator=gen).to(torch.bfloat16).to(DEV)
    out = torch.empty(B, heads * dim, dtype=torch.bfloat16, device=DEV)
    row, es = qkv.shape[1], 2

    def step():
        ctx.kv_tables_dev(cached.data_ptr(), added.data_ptr(), B, page, free.data_ptr(), free.numel(), head.data_ptr(),
                          table.data_ptr(), w, slots.data_ptr(), B, start.data_ptr(), ln.data_ptr(), head2.data_ptr(),
                          status.data_ptr())
        k = qkv.data_ptr() + heads * dim * es
        cache.write_dev(k, k + kvh * dim * es, B, slots.data_ptr(), "bf16", ldk=row, ldv=row)
        cache.attention_dev(qkv.data_ptr(), B, heads, out.data_ptr(), "bf16", prefix_table_ptr=pt.data_ptr(),
                            prefix_len=prefix, table_ptr=table.data_ptr(), table_w=w, B=B, lengths_ptr=ln.data_ptr(),
                            start_ptr=start.data_ptr(), max_added=1, ldq=row)

    old = ctx.stream
    s = torch.cuda.Stream()
    try:
        s.wait_stream(torch.cuda.current_stream())
        ctx.set_stream(s.cuda_stream)
        step()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
            step()
        for it in range(4):
            new = torch.randn(qkv.shape, generator=gen).to(torch.bfloat16)
            qkv.copy_(new)
            torch.cuda.synchronize()
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            ctx.set_stream(s.cuda_stream)
            out.zero_()
            torch.cuda.synchronize()
            step()
            s.synchronize()
            assert torch.equal(bits(got), bits(out))
            assert status.tolist() == [0] and ln.tolist() == [x + 1 for x in lengths]
            q = new[:, :heads * dim].reshape(B, heads, dim)
            want, bound = R.attention(q, kp.cpu(), vp.cpu(), dim ** -0.5, c.prefix_table, prefix, table.cpu().numpy(),
                                      ln.cpu().numpy(), start.cpu().numpy(), "bf16")
            same(got.cpu().reshape(B, heads, dim), want, bound)
            # the next step's tables: one token more each
            lengths = [x + 1 for x in lengths]
            cached.copy_(ln)
            head.copy_(head2)
    finally:
        ctx.set_stream(old)


@pytest.mark.parametrize("q,cache", TYPES)
@pytest.mark.parametrize("name", ["steps", "steps behind a prefix", "steps of longer requests", "pieces of prompts"])
def test_attention_of_many_short_requests(ctx, q, cache, name):
    """More requests than the chip takes workgroups, most of a few keys each; passes
    give the same bits."""
    heads, kvh, dim, prefix, lengths, added = {
        "steps": (8, 8, 128, 0, [1 + i % 30 for i in range(150)], [1] * 150),
        "steps behind a prefix": (8, 8, 64, 70, [1 + i % 20 for i in range(140)], [1] * 140),
        "steps of longer requests": (32, 32, 64, 0, [1 + i * 37 % 500 for i in range(130)], [1] * 130),
        "pieces of prompts": (8, 8, 80, 0, [i % 21 + i % 9 for i in range(70)], [i % 21 for i in range(70)]),
    }[name]
    c = Case(heads, kvh, dim, 8, "head", q, cache, prefix, lengths, added)
    first = c.check(ctx)
    for _ in range(5):
        assert torch.equal(bits(first), bits(c.run(ctx)))


@pytest.mark.parametrize("q,cache", TYPES[:2])
def test_attention_of_prompts_repeats_bit_for_bit(ctx, q, cache):
    """Prompts whose tiles are cut between workgroups give the same bits from call to
    call, other calls in between."""
    c = Case(8, 1, 128, 16, "head", q, cache, 700, [290, 600, 31], [260, 333, 31])
    other = Case(4, 2, 64, 16, "head", q, cache, 90, [50, 9], [1, 1])
    first, first_other = c.check(ctx), other.check(ctx)
    for _ in range(10):
        assert torch.equal(bits(first), bits(c.run(ctx)))
        assert torch.equal(bits(first_other), bits(other.run(ctx)))


def test_attention_repeats_bit_for_bit(ctx):
    c = Case(16, 2, 128, 16, "head", "f16", "f16", 2000, [300, 900, 40, 700] * 4, [1] * 16)
    first = c.run(ctx)
    for _ in range(3):
        assert torch.equal(bits(first), bits(c.run(ctx)))
