"""What the paged cache's entry points refuse, and the index arithmetic of their
kernels on broken tables, without a device."""
import ctypes as C
import os
import subprocess

import pytest

from pyflamert_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20  # an address that nothing here reads


def bind(k=A, v=2 * A, dtype=_lib.PFR_BF16, pages=10, page=16, heads=2, dim=64, ps=2048, hs=1024, ts=64):
    h = C.c_void_p()
    rc = _lib.load().pfr_kv_bind(k, v, dtype, pages, page, heads, dim, ps, hs, ts, C.byref(h))
    return rc, h


@pytest.mark.parametrize("code,text,kw", [
    (1, "null pool", {"k": None}),
    (1, "null pool", {"v": None}),
    (1, "float32, float16 or bfloat16", {"dtype": _lib.PFR_I8}),
    (1, "empty extent", {"pages": 0}),
    (1, "empty extent", {"heads": 0}),
    (1, "empty extent", {"dim": 0}),
    (1, "page size", {"page": 0}),
    (1, "page size", {"page": (1 << 20) + 1}),
    (1, "too large", {"pages": 1 << 31}),
    (3, "multiple of 8", {"dim": 60}),
    (3, "multiple of 8", {"dim": 264, "ts": 264, "hs": 264 * 16, "ps": 264 * 32}),
    (1, "negative stride", {"ps": -2048}),
    (1, "below the head dim", {"ts": 56}),
    (1, "below the head dim", {"hs": 0}),
    (1, "16 bytes", {"ts": 68}),
    (1, "16 bytes", {"k": A + 8}),
    (1, "16 bytes", {"v": A + 2}),
])
def test_bind_refuses(code, text, kw):
    rc, h = bind(**kw)
    assert rc == code and not h.value
    assert text in _lib.load().pfr_last_error().decode()


def test_bind_describes():
    rc, h = bind()
    assert rc == 0 and h.value
    L = _lib.load()
    dt, n = C.c_int(), [C.c_int64() for _ in range(4)]
    assert L.pfr_kv_info(h, C.byref(dt), *(C.byref(x) for x in n)) == 0
    assert dt.value == _lib.PFR_BF16 and [x.value for x in n] == [10, 16, 2, 64]
    assert L.pfr_kv_free(h) == 0
    assert L.pfr_kv_free(None) == 0
    assert L.pfr_kv_info(None, None, None, None, None, None) == 1


TABLES = dict(cached=A, added=2 * A, B=4, page=16, free=3 * A, n_free=9, head=4 * A, table=5 * A, table_w=8, table_ld=8,
              slots=6 * A, max_tokens=32, start=7 * A, lengths=8 * A, head_out=9 * A, status=10 * A)


@pytest.mark.parametrize("text,kw", [
    ("negative", {"B": -1}),
    ("negative", {"max_tokens": -1}),
    ("2^20 requests", {"B": (1 << 20) + 1}),
    ("page size", {"page": 0}),
    ("2^31", {"n_free": 1 << 31}),
    ("row stride", {"table_ld": 7}),
    ("null start", {"start": None}),
    ("null start", {"head_out": None}),
    ("null start", {"status": None}),
    ("null cached", {"cached": None}),
    ("null cached", {"lengths": None}),
    ("null table", {"table": None}),
    ("null slots", {"slots": None}),
    ("null free list", {"free": None}),
    ("overlaps", {"lengths": A + 12}),
    ("overlaps", {"start": 2 * A - 4}),
    ("overlaps", {"head_out": 4 * A}),
    ("null context", {}),
    ("null context", {"B": 0, "cached": None, "added": None, "lengths": None, "table": None}),
    ("null context", {"head": None, "n_free": 0, "free": None}),
])
def test_tables_refuse(text, kw):
    a = {**TABLES, **kw}
    L = _lib.load()
    assert L.pfr_kv_tables_dev(None, *a.values()) == 1
    assert text in L.pfr_last_error().decode()


@pytest.mark.parametrize("code,text,kw", [
    (1, "null kv", {"kv": None}),
    (1, "negative", {"T": -1}),
    (1, "float32, float16", {"dtype": _lib.PFR_I32}),
    (3, "own type", {"dtype": _lib.PFR_F16}),
    (1, "token stride", {"ldk": 127}),
    (1, "token stride", {"ldv": 0}),
    (1, "null k/v", {"k": None}),
    (1, "null k/v", {"slots": None}),
    (1, "too many", {"T": 1 << 40}),
    (1, "null context", {}),
    (1, "null context", {"T": 0, "k": None, "v": None, "slots": None}),
])
def test_write_refuses(code, text, kw):
    _, h = bind()
    a = {**dict(kv=h, k=A, v=2 * A, dtype=_lib.PFR_F32, T=3, ldk=128, ldv=128, slots=3 * A), **kw}
    L = _lib.load()
    assert L.pfr_kv_write_dev(None, *a.values()) == code
    assert text in L.pfr_last_error().decode()
    L.pfr_kv_free(h)


@pytest.mark.parametrize("code,text,kw", [
    (1, "null kv", {"kv": None}),
    (1, "negative", {"T": -1}),
    (1, "negative", {"prefix_len": -1}),
    (1, "multiple of the cache's heads", {"heads": 3}),
    (1, "multiple of the cache's heads", {"heads": 0}),
    (3, "float32 or of the cache's type", {"dtype": _lib.PFR_F16}),
    (1, "token stride", {"ldq": 255}),
    (1, "token stride", {"ldo": 255}),
    (1, "scale", {"scale": float("nan")}),
    (1, "scale", {"scale": float("inf")}),
    (1, "null q", {"q": None}),
    (1, "null q", {"out": None}),
    (1, "null prefix", {"prefix_table": None}),
    (1, "null lengths", {"lengths": None}),
    (1, "null lengths", {"start": None}),
    (1, "null table", {"table": None}),
    (1, "row stride", {"table_ld": 7}),
    (1, "negative bound", {"max_added": -1}),
    (1, "negative bound", {"max_length": -1}),
    (1, "too large", {"T": 1 << 25}),
    (1, "too large", {"prefix_len": (1 << 30) + 1}),
    (1, "too large", {"table_w": 1 << 27, "table_ld": 1 << 27}),
    (1, "overlaps q", {"out": A + 512}),
    (1, "null context", {}),
    (1, "null context", {"T": 0, "q": None, "out": None}),
    (1, "null context", {"B": 0, "table": None, "lengths": None, "start": None}),
    (1, "null context", {"prefix_len": 0, "prefix_table": None}),
])
def test_attention_refuses(code, text, kw):
    _, h = bind()
    a = {**dict(kv=h, q=A, dtype=_lib.PFR_BF16, T=3, heads=4, ldq=256, scale=0.125, prefix_table=3 * A, prefix_len=100,
                table=4 * A, table_w=8, table_ld=8, B=2, lengths=5 * A, start=6 * A, max_added=0, max_length=0,
                out=2 * A, ldo=256), **kw}
    L = _lib.load()
    assert L.pfr_kv_attention_dev(None, *a.values()) == code
    assert text in L.pfr_last_error().decode()
    L.pfr_kv_free(h)


INDEX_CPP = r"""
#include "kv_index.hpp"
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
using namespace pfr;
#define CHECK(c) do { if (!(c)) { printf("line %d\n", __LINE__); return 1; } } while (0)
int main() {
    std::mt19937 r(7);
    for (uint32_t d : {1u, 2u, 3u, 7u, 8u, 16u, 24u, 100u, 1000003u, 1u << 20, 0x7fffffffu, 0x80000000u, 0xffffffffu}) {
        FastDiv f(d);
        for (uint64_t q : {0ull, 1ull, 2ull, 0xffffffffull / d})
            for (int e = -1; e < 2; ++e) {
                const int64_t x = (int64_t)(q * d) + e;
                if (x >= 0 && x <= 0xffffffffll) CHECK(f.div((uint32_t)x) == (uint32_t)x / d);
            }
        for (int i = 0; i < 20000; ++i) { const uint32_t x = r(); CHECK(f.div(x) == x / d); }
    }
    // offsets of any key through any table lie in the pool or are -1; the table is never read past its end
    for (int it = 0; it < 300; ++it) {
        PageMap m;
        const int page = 1 + r() % 40, w = r() % 6;
        m.page = FastDiv(page);
        m.pages = 1 + r() % 9;
        m.token_stride = 8 * (1 + r() % 4);
        m.page_stride = m.token_stride * page + 8 * (r() % 3);
        int32_t* t = (int32_t*)malloc(4 * (w ? w : 1));  // of its size, so that a read past it shows under a sanitizer
        for (int i = 0; i < w; ++i) t[i] = (int32_t)(r() % 4 ? r() % 12 : r()) - (r() % 5 == 0 ? 20 : 0);
        const int hi = w ? 1 + r() % (w * page) : 0;
        for (int key = 0; hi && key < (w + 2) * page; ++key) {
            const KeyPlace p = key_place(m, key, hi);
            const int64_t o = key_offset(m, p, t[p.entry], key, hi);
            const bool in = key < hi && t[key / page] >= 0 && t[key / page] < (int)m.pages;
            CHECK((o >= 0) == in);
            if (in) CHECK(o == (int64_t)t[key / page] * m.page_stride + (key % page) * m.token_stride);
        }
        free(t);
    }
    // a pool past 2^32 elements
    PageMap big;
    big.page = FastDiv(16);
    big.pages = 3000000;
    big.token_stride = 128;
    big.page_stride = 65536;
    const int32_t far = 2999999;
    CHECK(key_offset(big, key_place(big, 15, 16), far, 15, 16) == 2999999ll * 65536 + 15 * 128);
    // token ranges stay within T for any start
    for (int it = 0; it < 20000; ++it) {
        const int T = r() % 50;
        const int32_t s[2] = {(int32_t)(r() % 3 ? r() % 60 : r()), (int32_t)(r() % 3 ? r() % 60 : r())};
        int a, b;
        request_tokens(s, 0, T, &a, &b);
        CHECK(a >= 0 && a <= b && b <= T);
        if (s[0] >= 0 && s[0] <= s[1] && s[1] <= T) CHECK(a == s[0] && b == s[1]);
    }
    // splits cover [0, end) once, in order, whatever length they were planned for
    for (int it = 0; it < 20000; ++it) {
        const int n = 1 + r() % 7, chunk = 128 * (1 + r() % 3), end = r() % 3000;
        int at = 0;
        for (int s = 0; s < n; ++s) {
            int lo, hi;
            split_span(s, n, chunk, end, &lo, &hi);
            CHECK(lo == at && hi >= lo && hi <= end);
            at = hi;
        }
        CHECK(at == end);
    }
    for (int len : {INT32_MIN, -1, 0, 1, 5, kMaxKeys, INT32_MAX})
        for (int n : {1, 2, 1 << 25}) {
            const int l0 = first_limit(len, n);
            for (int i : {0, n - 1})
                for (int64_t room : {(int64_t)0, (int64_t)7, (int64_t)kMaxKeys}) {
                    const int e = keys_end(l0, i, room);
                    CHECK(e >= 0 && e <= room);
                    if (len >= 0 && len <= kMaxKeys) CHECK(e == std::max<int64_t>(0, std::min<int64_t>(room, (int64_t)len - n + 1 + i)));
                }
        }
    puts("ok");
}
"""


def test_index_arithmetic(tmp_path):
    src = tmp_path / "index.cpp"
    src.write_text("#include <algorithm>\n" + INDEX_CPP)
    exe = str(tmp_path / "index")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                    "-I" + os.path.join(ROOT, "pyflamert_amd", "csrc", "rocm"), str(src), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr[-2000:]
