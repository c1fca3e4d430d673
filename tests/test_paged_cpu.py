"""CPU checks of the operators on paged caches and of token scores: refused arguments, and the index
arithmetic that keeps any content of the device arrays inside the buffers."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import dfx
from conftest import REPO
from paged_ref import TABLE, e4m3, scale_of

L = dfx.lib
PTR = 0x10000            # an aligned address that is never followed: every call here is refused or empty


def cache(**kw):
    d = dict(type=dfx.TYPE_F8, page_size=64, n_head_kv=4, head_dim=128, n_pages=8, k=PTR, v=PTR, scale=PTR)
    d.update(kw)
    return dfx.PagedCache(**d)


def batch(**kw):
    d = dict(n_seqs=2, n_rows=5, rows=PTR, n_keys=PTR, pages=PTR, ld_pages=4, max_keys=100)
    d.update(kw)
    return dfx.PagedBatch(**d)


BAD = [(dict(type=dfx.TYPE_Q8_0), {}, -2), (dict(head_dim=96), {}, -2), (dict(page_size=48), {}, -2),
       (dict(page_size=8), {}, -2), (dict(page_size=512), {}, -2), (dict(page_size=0), {}, -2),
       (dict(n_head_kv=0), {}, -1), (dict(n_head_kv=3), {}, -1), (dict(n_pages=0), {}, -1),
       (dict(n_pages=1 << 40), {}, -1), (dict(k=None), {}, -1), (dict(v=None), {}, -1), (dict(scale=None), {}, -1),
       (dict(k=PTR + 8), {}, -1), (dict(v=PTR + 1), {}, -1), (dict(scale=PTR + 4), {}, -1),
       ({}, dict(n_seqs=-1), -1), ({}, dict(n_rows=-1), -1), ({}, dict(max_keys=-1), -1),
       ({}, dict(n_rows=1 << 30), -1), ({}, dict(n_rows=(1 << 20) + 1), -1), ({}, dict(rows=None), -1), ({}, dict(n_keys=None), -1),
       ({}, dict(pages=None), -1), ({}, dict(ld_pages=0), -1)]


@pytest.mark.parametrize("ckw,bkw,code", BAD)
def test_unsound_caches_and_batches_are_refused(ckw, bkw, code):
    c, b = cache(**ckw), batch(**bkw)
    assert L().dfx_paged_append(C.byref(c), C.byref(b), PTR, 8, PTR, 100, dfx.TYPE_F16, PTR, None) == code
    assert b"dfx_paged_append" in L().dfx_last_error()
    assert L().dfx_paged_attention(C.byref(c), C.byref(b), PTR, dfx.TYPE_F16, 8, 1, 0, PTR, None, None) == code
    assert b"dfx_paged_attention" in L().dfx_last_error()
    assert L().dfx_paged_attention_ws_bytes(C.byref(c), C.byref(b), 8, dfx.TYPE_F16) == 0


def test_unsound_calls_are_refused():
    c, b = cache(), batch()
    ap = L().dfx_paged_append
    at = L().dfx_paged_attention
    assert ap(None, C.byref(b), PTR, 8, PTR, 100, 1, PTR, None) == -1
    assert ap(C.byref(c), None, PTR, 8, PTR, 100, 1, PTR, None) == -1
    assert ap(C.byref(c), C.byref(b), PTR, 8, PTR, 100, dfx.TYPE_Q8_0, PTR, None) == -2
    for args in ((None, 8, PTR, 100, 1, PTR), (PTR, 8, None, 100, 1, PTR), (PTR, 8, PTR, 100, 1, None),
                 (PTR, 8, PTR, 0, 1, PTR), (PTR + 4, 8, PTR, 100, 1, PTR), (PTR, 8, PTR + 8, 100, 1, PTR),
                 (PTR, 8, PTR, 100, 1, PTR + 2), (PTR, 0, PTR, 100, 1, PTR), (PTR, 6, PTR, 100, 1, PTR)):
        assert ap(C.byref(c), C.byref(b), *args, None) == -1
    assert at(C.byref(c), C.byref(b), PTR, dfx.TYPE_Q8_0, 8, 1, 0, PTR, None, None) == -2
    for args in ((None, 1, 8, 1, 0, PTR, None), (PTR, 1, 8, 1, 0, None, None), (PTR, 1, 8, 1, -1, PTR, None),
                 (PTR, 1, 8, 0, 5, PTR, None), (PTR + 2, 1, 8, 1, 0, PTR, None), (PTR, 1, 8, 1, 0, PTR + 2, None),
                 (PTR, 1, 8, 1, 0, PTR, PTR + 4), (PTR, 1, 5, 1, 0, PTR, None)):
        assert at(C.byref(c), C.byref(b), *args, None) == -1
    # nothing to do is no error
    for kw in (dict(n_rows=0), dict(n_seqs=0), dict(n_rows=0, rows=None, pages=None, n_keys=None)):
        e = batch(**kw)
        assert ap(C.byref(c), C.byref(e), PTR, 8, PTR, 100, 1, PTR, None) == 0
        assert at(C.byref(c), C.byref(e), PTR, 1, 8, 1, 0, PTR, None, None) == 0


def test_unsound_scores_are_refused():
    lp = L().dfx_token_logprobs

    def call(logits=PTR, ld=100, n_logits=4, rows=None, n_rows=4, V=100, tokens=PTR, n_tok=1, lpo=PTR, ent=PTR, n_top=5,
             tid=PTR, tlp=PTR, ws=PTR):
        return lp(logits, ld, n_logits, rows, n_rows, V, tokens, n_tok, lpo, ent, n_top, tid, tlp, ws, None)

    for kw in (dict(logits=None), dict(ld=99), dict(V=0), dict(V=1 << 31), dict(n_rows=-1), dict(n_rows=(1 << 22) + 1),
               dict(n_logits=-1), dict(n_tok=-1), dict(n_top=-1), dict(n_top=65), dict(tokens=None), dict(lpo=None),
               dict(tid=None), dict(tlp=None), dict(ws=None), dict(ws=PTR + 8)):
        assert call(**kw) == -1, kw
        assert b"dfx_token_logprobs" in L().dfx_last_error()
    assert call(n_rows=0) == 0
    assert L().dfx_token_logprobs_ws_bytes(4, 100, 65) == 0
    assert L().dfx_token_logprobs_ws_bytes(4, 100, 5) > 0


INDEX_PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <climits>
#include <vector>
#include "dfx_pages.h"
#define REQUIRE(x) do { if (!(x)) { printf("line %d: %s (case %d)\n", __LINE__, #x, it); return 1; } } while (0)
static int wild() {     // anything an int32 array can hold
    switch (rand() % 6) {
        case 0: return INT_MIN; case 1: return INT_MAX; case 2: return -(rand() % 100); case 3: return rand() % 40;
        case 4: return rand() - RAND_MAX / 2; default: return rand() % 500;
    }
}
int main() {
    for (int it = 0; it < 20000; it++) {
        paged_t p = {};
        const int S = 1 + rand() % 6, shift = 4 + rand() % 5, ld = 1 + rand() % 7;
        std::vector<int32_t> rows(S + 1), keys(S), pages(S * ld);
        for (auto & x : rows) x = wild();
        for (auto & x : keys) x = wild();
        for (auto & x : pages) x = wild();
        p.rows = rows.data(); p.n_keys = keys.data(); p.pages = pages.data(); p.ld_pages = ld;
        p.page_shift = shift; p.cap = ld << shift; p.n_pages = 1 + rand() % 20; p.Hkv = 1 + rand() % 8;
        p.n_seqs = S; p.n_rows = rand() % 300;
        const int64_t blocks = (int64_t)p.n_pages * p.Hkv << (shift - 4);
        for (int s = 0; s < S; s++) {
            const seq_t q = pg_seq(p, s);
            REQUIRE(q.r0 >= 0 && q.n >= 0 && q.r0 + q.n <= p.n_rows && q.keys >= 0 && q.keys <= p.cap);
            for (int k = 0; k < 60; k++) {
                const int pos = k < 20 ? wild() : rand() % (p.cap + 20) - 10, h = rand() % p.Hkv;
                const int64_t b = pg_block(p, s, h, pos);
                REQUIRE(b >= -1 && b < blocks);
                if (pos < 0 || pos >= p.cap) REQUIRE(b == -1);
                else {
                    const int page = pages[s * ld + (pos >> shift)];
                    if (page < 0 || page >= p.n_pages) REQUIRE(b == -1);
                    else REQUIRE(b == ((int64_t)page * p.Hkv + h) * (1 << (shift - 4)) + (pos % (1 << shift)) / 16);
                }
            }
            // the tiles of a query tile hold every key that one of its rows sees, inside the sequence
            const int G = 1 + rand() % 8, causal = rand() % 2, window = causal && rand() % 2 ? 1 + rand() % 90 : 0;
            if (!q.n) continue;
            const int T = 16 << rand() % 4, tile = rand() % ((q.n * G + T - 1) / T);
            const int f0 = tile * T, f1 = f0 + T < q.n * G ? f0 + T - 1 : q.n * G - 1;
            const tiles_t t = pg_tiles(q, f0, f1, G, causal, window);
            REQUIRE(t.t0 >= 0 && t.t0 <= t.t1 && t.t1 <= (q.keys + 63) / 64);
            for (int f = f0; f <= f1; f++) {
                const int pos = q.keys - q.n + f / G;
                const seen_t e = pg_seen(pos, q.keys, causal, window);
                if (e.hi < e.lo) { REQUIRE(pos < 0 || q.keys == 0); continue; }
                REQUIRE(e.lo >= 0 && e.hi < q.keys && e.lo / 64 >= t.t0 && e.hi / 64 < t.t1);
                if (causal) REQUIRE(e.hi == pos && (window ? e.lo == (pos + 1 > window ? pos + 1 - window : 0) : e.lo == 0));
                else REQUIRE(e.lo == 0 && e.hi == q.keys - 1);
            }
            // parts cover the tiles once, in order, whatever bound the split was chosen for
            const int chunk = 1 + rand() % 9, most = 1 + rand() % 9;
            int at = t.t0;
            const int parts = part_of(t, 0, chunk, most).parts;
            REQUIRE(parts >= 1 && parts <= most);
            for (int i = 0; i < parts; i++) {
                const part_at a = part_of(t, i, chunk, most);
                REQUIRE(a.parts == parts && (t.t0 == t.t1 ? a.t0 == a.t1 : a.t0 == at && a.t1 > a.t0));
                at = a.t1;
            }
            REQUIRE(t.t0 == t.t1 || at == t.t1);
            const part_at none = part_of(t, parts, chunk, most);
            REQUIRE(none.t0 == none.t1);
        }
    }
    puts("ok");
    return 0;
}
"""


def test_indices_stay_inside_for_any_device_content(tmp_path):
    """Row offsets, key counts and page ids of any value: rows, keys, blocks and key tiles stay inside, bad
    pages are none, and the split of a key range covers it exactly."""
    src, exe = tmp_path / "index.cpp", tmp_path / "index"
    src.write_text(INDEX_PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-D__host__=",
                           "-D__device__=", "-I", os.path.join(REPO, "include"), "-I",
                           os.path.join(REPO, "diffuse-cpp_amd", "csrc"), str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout[-500:] + r.stderr[-500:]


def test_the_tests_e4m3_is_torchs():
    """The numpy E4M3 of the tests against torch's conversion: every code, ties, the ends."""
    torch = pytest.importorskip("torch")
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(codes, TABLE.astype(np.float32), equal_nan=True)
    rng = np.random.default_rng(0)
    fin = TABLE[np.isfinite(TABLE)]
    x = np.concatenate([fin, (fin[:-1] + fin[1:]) / 2, rng.standard_normal(20000) * 50, rng.standard_normal(20000) * 0.01,
                        [448.0, -448.0, 0.0, -0.0, 2.0 ** -10, 2.0 ** -11]]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(e4m3(x), want)
    assert scale_of(0.0) == 2.0 ** -15 and scale_of(448.0) == 1 and scale_of(448.1) == 2 and scale_of(1e9) == 128
