"""Append to and attention over paged caches on the GPU, against plain forms (tests/paged_ref.py): the
append bit for bit in its float32 steps, the attention in float64 within the bound of its arithmetic."""
import ctypes as C

import numpy as np
import pytest

import dfx
from paged_ref import BLOCK, TABLE, Batch, Cache, check_attention, e4m3, ref, ref_append, rope_table, rotate, same_cells
from paged_ref import scale_of

pytestmark = pytest.mark.gpu
L = dfx.lib
F16, F32, F8 = dfx.TYPE_F16, dfx.TYPE_F32, dfx.TYPE_F8
NP = {F16: np.float16, F32: np.float32}


def run_append(c, b, qkv, H, tab, qt, q_fill=None, stream=None):
    q = np.full((b.M, H, c.hd), 7.0, NP[qt]) if q_fill is None else q_fill
    dq, dx, dt = dfx.Buf.of(q), dfx.Buf.of(qkv), dfx.Buf.of(tab)
    cd, bd = c.desc(), b.desc()
    dfx.check(L().dfx_paged_append(ref(cd), ref(bd), dx.ptr, H, dt.ptr, len(tab), qt, dq.ptr, stream), "append")
    dfx.sync(stream)
    return dq.download(NP[qt], shape=q.shape)


def run_attention(c, b, q, H, causal, window, ws=True, stream=None):
    f32 = q.dtype == np.float32
    typ = F32 if f32 else F16
    cd, bd = c.desc(), b.desc()
    n = L().dfx_paged_attention_ws_bytes(ref(cd), ref(bd), H, typ)
    w = dfx.Buf.of(np.full(n, 0xFF, np.uint8)) if ws and n else None        # NaN if read before written
    dq, do = dfx.Buf.of(q), dfx.Buf.of(np.full(q.shape, 7.0, q.dtype))
    dfx.check(L().dfx_paged_attention(ref(cd), ref(bd), dq.ptr, typ, H, int(causal), window, do.ptr,
                                      w.ptr if w else None, stream), "attention")
    dfx.sync(stream)
    return do.download(q.dtype, shape=q.shape)


def fill_keys(c, b, rng):
    """Ordinary keys and values at every key of the batch; the rest of the pages keeps what it holds."""
    for s, keys in enumerate(b.keys):
        for blk in range(-(-min(keys, b.pages.shape[1] * b.page) // BLOCK)):
            page = b.page_of(s, blk * BLOCK, c.n_pages)
            if page < 0:
                continue
            nb, t = blk * BLOCK % c.page // BLOCK, min(BLOCK, keys - blk * BLOCK)
            for h in range(c.Hkv):
                k, v = rng.standard_normal((t, c.hd)), rng.standard_normal((t, c.hd))
                for side, x, cells in ((0, k, c.k[page, h, nb * BLOCK:nb * BLOCK + t]), (1, v, c.v[page, h, nb].T[:t])):
                    if c.f8:
                        sc = scale_of(np.abs(x).max())
                        c.scale[page, h, nb, side] = sc
                        cells[:] = e4m3(x / sc)
                    else:
                        cells[:] = x
    c.upload()


def qkv_of(rng, M, heads, hd):
    return (rng.standard_normal((M, heads, hd)) * rng.uniform(0.2, 4.0, (1, heads, 1))).astype(np.float32)


# ---------------------------------------------------------------- append
APPENDS = [
    # rows, keys after the call, page, Hkv, G, hd
    ([1], [1], 16, 1, 1, 64),
    ([1], [192], 64, 4, 7, 128),
    ([1] * 5, [1, 16, 17, 32, 200], 16, 2, 4, 64),
    ([3, 0, 40, 1, 17], [3, 9, 61, 130, 33], 32, 2, 1, 128),
    ([16, 15, 33], [32, 31, 100], 128, 3, 2, 64),
    ([70], [75], 256, 2, 2, 128),
    ([0, 0, 1, 0, 2, 0], [5, 0, 18, 0, 2, 40], 16, 1, 2, 128),
]


@pytest.mark.parametrize("typ", [F8, F16])
@pytest.mark.parametrize("qt", [F16, F32])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_bits(gpu, typ, qt, case):
    n, keys, page, Hkv, G, hd = APPENDS[case]
    rng = np.random.default_rng(100 + case)
    H = Hkv * G
    c = Cache(typ, page, Hkv, hd, sum(-(-k // page) for k in keys) + 3, seed=case)
    b = Batch(n, keys, page, c.n_pages, seed=case, pad_rows=case % 3, ld_extra=case % 2)
    tab = rope_table(max(keys) + 1, hd)
    qkv = qkv_of(rng, b.M, H + 2 * Hkv, hd)
    want = np.full((b.M, H, hd), 7.0, NP[qt])
    ref_append(c, b, qkv, H, tab, want)          # c's arrays now hold what the device should
    got = run_append(c, b, qkv, H, tab, qt)
    assert np.array_equal(got, want)             # rows of no sequence included
    k, v, sc = c.download()
    assert same_cells(c, k, c.k) and same_cells(c, v, c.v)
    if c.f8:
        assert np.array_equal(sc, c.scale)


@pytest.mark.parametrize("typ", [F8, F16])
def test_append_against_64_bits(gpu, typ):
    """Rotated values in float64: an f32 result is off by three roundings of its terms (3 * 2^-24 of
    |x0 c| + |x1 s|); a cell by half a step of E4M3 (2^-4 of the value, 2^-10 of the scale at the low
    end) or of f16 (2^-11, 2^-25), of a value that is itself off by that."""
    rng = np.random.default_rng(3)
    n, keys, page, Hkv, G, hd = [50, 7], [66, 23], 32, 2, 2, 128
    H = Hkv * G
    c = Cache(typ, page, Hkv, hd, 8)
    b = Batch(n, keys, page, c.n_pages)
    tab = rope_table(100, hd)
    qkv = qkv_of(rng, b.M, H + 2 * Hkv, hd)
    q = run_append(c, b, qkv, H, tab, F32)
    c.k, c.v, c.scale = c.download()
    for s in range(2):
        for i in range(n[s]):
            r, pos = int(b.rows[s]) + i, keys[s] - n[s] + i
            x = qkv[r].astype(np.float64)
            y = rotate(x[None, :H + Hkv], tab, np.array([pos]))[0]
            t = rotate(np.abs(x[None, :H + Hkv]), np.abs(tab), np.array([pos]))[0]
            size = np.maximum(np.abs(t), np.abs(np.concatenate([t[..., hd // 2:], t[..., :hd // 2]], -1)))
            assert (np.abs(q[r] - y[:H]) <= 3 * 2.0 ** -24 * 2 * size[:H]).all()
            for h in range(Hkv):
                page_id = b.page_of(s, pos, c.n_pages)
                k, v = c.values(page_id, h, pos)
                blk = pos % page // BLOCK
                for got, w, e, sd in ((k, y[H + h], 6 * 2.0 ** -24 * size[H + h], 0), (v, x[H + Hkv + h], 0.0, 1)):
                    if c.f8:
                        tol = 2.0 ** -4 * (np.abs(w) + e) + 2.0 ** -10 * float(c.scale[page_id, h, blk, sd]) + e
                    else:
                        tol = 2.0 ** -11 * (np.abs(w) + e) + 2.0 ** -25 + e
                    assert (np.abs(got - w) <= tol).all()


def test_append_in_pieces_is_append_at_once(gpu):
    """A prompt appended at once, in ragged chunks and token by token: the same cells, as no value is so
    small that a grown scale takes it below E4M3's normal range twice (values within 2^-5 of a block's
    largest lose no bit to a power of two)."""
    rng = np.random.default_rng(5)
    Hkv, G, hd, page, N = 2, 2, 64, 32, 75
    H = Hkv * G
    tab = rope_table(N, hd)
    qkv = (rng.choice([-1.0, 1.0], (N, H + 2 * Hkv, hd)) * rng.uniform(0.25, 4.0, (N, H + 2 * Hkv, hd))).astype(np.float32)
    tab[..., 0], tab[..., 1] = 1.0, 0.0          # no rotation: the magnitudes stay in their range
    results = []
    for cuts in ([0, N], [0, 5, 21, 22, 37, 64, N], list(range(N + 1))):
        c = Cache(F8, page, Hkv, hd, 3, seed=9)
        c.scale[:] = 1.0
        c.upload()
        pages = np.array([[2, 0, 1]])
        for a, z in zip(cuts, cuts[1:]):
            b = Batch([z - a], [z], page, 3, pages=pages)
            run_append(c, b, qkv[a:z], H, tab, F16)
        results.append(c.download())
    for k, v, sc in results[1:]:
        live = np.zeros((3, Hkv, page), bool)
        for p in range(N):
            live[pages[0, p // page], :, p % page] = True
        assert np.array_equal(k[live], results[0][0][live])
        vv, v0 = (x.transpose(0, 1, 2, 4, 3).reshape(3, Hkv, page, hd) for x in (v, results[0][1]))
        assert np.array_equal(vv[live], v0[live])
        blocks = live.reshape(3, Hkv, page // BLOCK, BLOCK).any(-1)
        assert np.array_equal(sc[blocks], results[0][2][blocks])


@pytest.mark.parametrize("typ", [F8, F16])
def test_append_of_a_recomputed_block(gpu, typ):
    """A step that writes the same last positions again, with other values: the tokens before them stay, the
    rest is as if written first."""
    rng = np.random.default_rng(6)
    Hkv, G, hd, page = 2, 2, 128, 16
    H = Hkv * G
    c = Cache(typ, page, Hkv, hd, 6)
    tab = rope_table(80, hd)
    b0, b1 = Batch([21], [21], page, 6), Batch([40], [61], page, 6)
    b1.pages[:, :2] = b0.pages
    b1.pages[:, 2:] = [p for p in range(6) if p not in b0.pages[0]][:2]
    b1.d[2].upload(b1.pages)
    for b, times in ((b0, 1), (b1, 3)):
        for i in range(times):
            qkv = qkv_of(rng, b.M, H + 2 * Hkv, hd) * np.float32(2.0 ** (i * 3))
            want = np.full((b.M, H, hd), 7.0, np.float16)
            with np.errstate(over="ignore"):
                ref_append(c, b, qkv, H, tab, want)
            assert np.array_equal(run_append(c, b, qkv, H, tab, F16), want)
            k, v, sc = c.download()
            assert same_cells(c, k, c.k) and same_cells(c, v, c.v)
            assert not c.f8 or np.array_equal(sc, c.scale)


@pytest.mark.parametrize("typ", [F8, F16])
def test_append_of_extreme_values(gpu, typ):
    """Zeros, values beyond the largest scale, below the smallest, infinities and NaN, f16 overflow."""
    rng = np.random.default_rng(8)
    Hkv, hd, page = 2, 64, 16
    c = Cache(typ, page, Hkv, hd, 8)
    b = Batch([16, 20, 5, 9], [16, 30, 5, 9], page, 8)
    qkv = qkv_of(rng, b.M, 3 * Hkv, hd)
    qkv[0:16] = 0.0
    qkv[16:36] *= np.float32(1e5)
    qkv[36:41] *= np.float32(1e-7)
    qkv[41:50][rng.random((9, 3 * Hkv, hd)) < 0.2] = np.inf
    qkv[41:50][rng.random((9, 3 * Hkv, hd)) < 0.1] = np.nan
    qkv[45, 2, 3] = -np.inf
    tab = rope_table(32, hd)
    want = np.full((b.M, Hkv, hd), 7.0, np.float32)
    with np.errstate(invalid="ignore"):
        ref_append(c, b, qkv, Hkv, tab, want)
    got = run_append(c, b, qkv, Hkv, tab, F32)
    assert np.array_equal(got, want, equal_nan=True)
    k, v, sc = c.download()
    assert same_cells(c, k, c.k) and same_cells(c, v, c.v)
    assert not c.f8 or np.array_equal(sc, c.scale)


@pytest.mark.parametrize("typ", [F8, F16])
@pytest.mark.parametrize("rows_each", [1, 20])
def test_append_skips_what_has_no_place(gpu, typ, rows_each):
    """Positions behind the rotation table or the page ids, before the first, page ids of no page: skipped,
    and nothing else changes."""
    rng = np.random.default_rng(10 + rows_each)
    Hkv, G, hd, page = 2, 2, 64, 16
    H = Hkv * G
    c = Cache(typ, page, Hkv, hd, 12)
    n = [rows_each] * 6
    keys = [rows_each - 1, 40, 48, 33, 500, 30]
    pages = np.array([[0, 1, 2], [3, -1, 4], [5, 6, 12], [7, 1 << 30, 8], [9, 10, 11], [-(1 << 31), -5, 99]])
    b = Batch(n, keys, page, 12, pages=pages)
    tab = rope_table(45, hd)
    qkv = qkv_of(rng, b.M, H + 2 * Hkv, hd)
    want = np.full((b.M, H, hd), 7.0, np.float32)
    ref_append(c, b, qkv, H, tab, want)
    assert np.array_equal(run_append(c, b, qkv, H, tab, F32), want)
    k, v, sc = c.download()
    assert same_cells(c, k, c.k) and same_cells(c, v, c.v)
    assert not c.f8 or np.array_equal(sc, c.scale)


@pytest.mark.parametrize("S,empty", [(64, 0), (65, 3), (200, 2), (4200, 5)])
def test_append_of_many_sequences(gpu, S, empty):
    """One token each, empty sequences between them, more sequences than one probe of the wave covers."""
    rng = np.random.default_rng(S)
    Hkv, hd, page = 1, 64, 16
    n = [0 if empty and rng.integers(0, empty) else 1 for _ in range(S)]
    keys = [int(rng.integers(1, 33)) for _ in range(S)]
    c = Cache(F8, page, Hkv, hd, sum(-(-k // page) for k in keys))
    b = Batch(n, keys, page, c.n_pages, pad_rows=5)
    tab = rope_table(33, hd)
    qkv = qkv_of(rng, b.M, 3 * Hkv, hd)
    want = np.full((b.M, Hkv, hd), 7.0, np.float16)
    ref_append(c, b, qkv, Hkv, tab, want)
    assert np.array_equal(run_append(c, b, qkv, Hkv, tab, F16), want)
    k, v, sc = c.download()
    assert same_cells(c, k, c.k) and same_cells(c, v, c.v) and np.array_equal(sc, c.scale)


# ---------------------------------------------------------------- attention
ATTENDS = [
    # rows, keys, page, Hkv, G, hd
    ([1], [1], 16, 1, 1, 64),
    ([1], [64], 64, 4, 7, 128),
    ([1], [65], 16, 1, 1, 128),
    ([1] * 6, [1, 15, 16, 17, 63, 300], 16, 2, 4, 64),
    ([5, 0, 33, 1], [5, 12, 90, 130], 32, 2, 3, 128),
    ([17, 2], [40, 2], 128, 1, 1, 64),
    ([0, 130, 0], [0, 150, 7], 64, 2, 2, 64),
    ([3], [700], 256, 1, 7, 128),
    ([160], [200], 16, 1, 1, 128),
    ([300], [340], 64, 1, 4, 128),
    ([40, 3, 0, 21], [90, 70, 64, 21], 16, 3, 2, 64),
    ([35, 90], [35, 260], 32, 5, 1, 128),
]


@pytest.mark.parametrize("causal,window", [(False, 0), (True, 0), (True, 1), (True, 37)])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("typ", [F8, F16])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(gpu, case, typ, f32, causal, window):
    n, keys, page, Hkv, G, hd = ATTENDS[case]
    rng = np.random.default_rng(200 + case)
    H = Hkv * G
    c = Cache(typ, page, Hkv, hd, sum(-(-k // page) for k in keys) + 2, seed=case)
    b = Batch(n, keys, page, c.n_pages, seed=case, pad_rows=case % 2)
    fill_keys(c, b, rng)
    q = (rng.standard_normal((b.M, H, hd)) * 1.5).astype(np.float32 if f32 else np.float16)
    got = run_attention(c, b, q, H, causal, window)
    check_attention(got, c, b, q, causal, window, f32)
    assert (got[int(b.rows[-1]):] == 7.0).all()          # rows of no sequence are left


# Rows times heads beyond 8192 take 32 queries a workgroup, beyond 32768 128: the same masks, types and ragged
# batches on those kernels
WIDE = [([130], [150], 64, 64), ([135, 0, 1], [135, 9, 300], 16, 128), ([70, 33, 40], [340, 33, 64], 32, 64)]


@pytest.mark.parametrize("causal,window", [(False, 0), (True, 0), (True, 1), (True, 37)])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("typ", [F8, F16])
@pytest.mark.parametrize("G", [1, 4])
@pytest.mark.parametrize("case", range(len(WIDE)))
def test_attention_of_many_heads(gpu, case, G, typ, f32, causal, window):
    n, keys, page, hd = WIDE[case]
    rng = np.random.default_rng(300 + case)
    Hkv = 64
    H = Hkv * G
    assert sum(n) * H > (32768 if G == 4 else 8192)
    c = Cache(typ, page, Hkv, hd, sum(-(-k // page) for k in keys) + 2, seed=case)
    b = Batch(n, keys, page, c.n_pages, seed=case, pad_rows=case % 2)
    fill_keys(c, b, rng)
    q = (rng.standard_normal((b.M, H, hd)) * 1.5).astype(np.float32 if f32 else np.float16)
    got = run_attention(c, b, q, H, causal, window)
    check_attention(got, c, b, q, causal, window, f32)
    assert (got[int(b.rows[-1]):] == 7.0).all()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("Hkv,G,n,keys", [(3, 4, 800, 1400), (8, 5, 900, 1300), (1, 4, 800, 1400)])
def test_attention_of_long_chunks(gpu, Hkv, G, n, keys, f32):
    """Many rows over ranges of more than 16 key tiles, with a workspace and without; one KV head's are split over
    workgroups, where there are enough of them they stay whole and need no workspace."""
    rng = np.random.default_rng(71)
    hd, page, H = 64, 64, Hkv * G
    c = Cache(F8, page, Hkv, hd, -(-keys // page))
    b = Batch([n], [keys], page, c.n_pages)
    fill_keys(c, b, rng)
    q = (rng.standard_normal((n, H, hd)) * 1.5).astype(np.float32 if f32 else np.float16)
    cd, bd = c.desc(), b.desc()
    assert L().dfx_paged_attention_ws_bytes(ref(cd), ref(bd), H, F32 if f32 else F16) > 0 or Hkv > 1
    for causal, window in ((True, 0), (False, 0), (True, 1100)):
        got = run_attention(c, b, q, H, causal, window)
        check_attention(got, c, b, q, causal, window, f32)
        check_attention(run_attention(c, b, q, H, causal, window, ws=False), c, b, q, causal, window, f32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("n,keys", [([1], [5000]), ([1, 1, 2], [3000, 10, 1500]), ([40], [2100])])
def test_attention_of_long_caches_is_split(gpu, n, keys, f32):
    """The split over workgroups and its join, against the same call without a workspace and float64; twice
    the same bits."""
    rng = np.random.default_rng(7)
    Hkv, G, hd, page = 1, 2, 64, 64
    H = Hkv * G
    c = Cache(F8, page, Hkv, hd, sum(-(-k // page) for k in keys))
    b = Batch(n, keys, page, c.n_pages)
    fill_keys(c, b, rng)
    q = (rng.standard_normal((b.M, H, hd)) * 1.5).astype(np.float32 if f32 else np.float16)
    cd, bd = c.desc(), b.desc()
    assert L().dfx_paged_attention_ws_bytes(ref(cd), ref(bd), H, F32 if f32 else F16) > 0
    for causal, window in ((True, 0), (True, 900), (False, 0)):
        got = run_attention(c, b, q, H, causal, window)
        check_attention(got, c, b, q, causal, window, f32)
        assert np.array_equal(got, run_attention(c, b, q, H, causal, window))
        check_attention(run_attention(c, b, q, H, causal, window, ws=False), c, b, q, causal, window, f32)
    # a bound below the real count: the last part takes the rest
    b.max_keys = 600
    check_attention(run_attention(c, b, q, H, True, 0), c, b, q, True, 0, f32)


@pytest.mark.parametrize("causal,window", [(False, 0), (True, 0), (True, 20)])
@pytest.mark.parametrize("S,most,Hkv", [(63, 2, 1), (64, 30, 1), (65, 3, 1), (150, 40, 1), (70, 150, 1), (64, 40, 8),
                                        (70, 40, 8), (64, 60, 16), (75, 60, 16), (5, 90, 40)])
def test_attention_of_many_sequences(gpu, S, most, Hkv, causal, window):
    """Ragged batches of up to and beyond 64 sequences, empty ones among them, at rows that take each kernel:
    every tile of every sequence is computed once."""
    rng = np.random.default_rng(S + most)
    G, hd, page = 1, 64, 16
    n = [0 if rng.random() < 0.1 else int(rng.integers(most // 2 + 1, most + 1)) for _ in range(S)]
    keys = [m + int(rng.integers(0, 80)) for m in n]
    c = Cache(F8, page, Hkv, hd, sum(-(-k // page) for k in keys))
    b = Batch(n, keys, page, c.n_pages, pad_rows=3)
    fill_keys(c, b, rng)
    q = (rng.standard_normal((b.M, Hkv, hd)) * 1.5).astype(np.float16)
    got = run_attention(c, b, q, Hkv, causal, window)
    check_attention(got, c, b, q, causal, window, False)
    assert (got[int(b.rows[-1]):] == 7.0).all()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("S,Hkv,window", [(40, 16, 0), (40, 16, 1100), (70, 8, 0)])
def test_attention_of_uneven_sequences_is_split(gpu, S, Hkv, window, f32):
    """Few long sequences among many short ones: long ranges in parts beside whole ones, some without keys."""
    rng = np.random.default_rng(90 + S)
    G, hd, page = 2, 64, 64
    n = [int(rng.integers(0, 3)) for _ in range(S)]
    keys = [int(rng.integers(0, 70)) for _ in range(S)]
    for s, k in ((0, 2300), (S // 2, 1500), (S - 1, 1030)):
        n[s], keys[s] = 1 + s % 2, k
    c = Cache(F8, page, Hkv, hd, sum(-(-k // page) for k in keys) + 1)
    b = Batch(n, keys, page, c.n_pages, seed=S, pad_rows=2)
    fill_keys(c, b, rng)
    H = Hkv * G
    q = (rng.standard_normal((b.M, H, hd)) * 1.5).astype(np.float32 if f32 else np.float16)
    cd, bd = c.desc(), b.desc()
    assert L().dfx_paged_attention_ws_bytes(ref(cd), ref(bd), H, F32 if f32 else F16) > 0
    got = run_attention(c, b, q, H, True, window)
    check_attention(got, c, b, q, True, window, f32)
    assert (got[int(b.rows[-1]):] == 7.0).all()


@pytest.mark.parametrize("typ", [F8, F16])
@pytest.mark.parametrize("rows,Hkv", [(1, 1), (30, 1), (100, 1), (200, 1), (90, 64), (200, 90)])
def test_attention_never_sees_hidden_keys(gpu, typ, rows, Hkv):
    """NaN and infinities in keys and values that some rows see and others do not (later positions, left of
    the window), in the same tile: they reach exactly the rows that see them."""
    rng = np.random.default_rng(40 + rows)
    G, hd, page, keys = 2, 64, 32, 230
    H, last = Hkv * G, Hkv - 1
    c = Cache(typ, page, Hkv, hd, 9)
    b = Batch([rows], [keys], page, 9)
    fill_keys(c, b, rng)
    bad = np.uint8(0x7f) if c.f8 else np.float16(np.nan)
    for pos, dim, side in ((keys - 3, 5, 1), (keys - 20, 9, 1), (keys - 25, 3, 0), (keys - 60, 1, 1), (100, 60, 1)):
        page_id, t = b.page_of(0, pos, 9), pos % page
        if side:
            c.v[page_id, last, t // BLOCK, dim, t % BLOCK] = bad
            if not c.f8:
                c.v[page_id, last, t // BLOCK, dim + 1, t % BLOCK] = np.inf
                c.v[page_id, last, t // BLOCK, dim + 2, t % BLOCK] = -np.inf
        else:
            c.k[page_id, last, t, dim] = bad
    c.upload()
    for f32 in (False, True):
        q = (rng.standard_normal((b.M, H, hd)) * 0.3).astype(np.float32 if f32 else np.float16)
        for causal, window in ((True, 0), (True, 24), (False, 0)):
            check_attention(run_attention(c, b, q, H, causal, window), c, b, q, causal, window, f32)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,Hkv", [(1, 1), (90, 64), (200, 90)])
def test_attention_ignores_scales_of_unwritten_blocks(gpu, rows, Hkv, hd):
    """Scales behind the last key hold anything, as memory that no append has written does."""
    rng = np.random.default_rng(60 + rows)
    G, page, keys = 2, 64, 230
    c = Cache(F8, page, Hkv, hd, 6)
    b = Batch([rows], [keys], page, 6)
    fill_keys(c, b, rng)
    left = np.array([np.nan, np.inf, -np.inf, 0.0, 1e-40, -3e38, 3.4e38], np.float32)
    page_id = b.page_of(0, keys, 6)
    c.scale[page_id, :, 3] = rng.choice(left, c.scale[page_id, :, 3].shape)
    for other in set(range(6)) - {b.page_of(0, p, 6) for p in range(0, keys, page)}:
        c.scale[other] = rng.choice(left, c.scale[other].shape)
    c.upload()
    for f32 in (False, True):
        q = rng.standard_normal((b.M, Hkv * G, hd)).astype(np.float32 if f32 else np.float16)
        for causal in (True, False):
            check_attention(run_attention(c, b, q, Hkv * G, causal, 0), c, b, q, causal, 0, f32)


@pytest.mark.parametrize("rows,keys,Hkv", [(1, 2000, 2), (20, 1300, 2), (90, 230, 64), (200, 230, 90)])
def test_attention_in_place(gpu, rows, keys, Hkv):
    """out is q: the bits of the call with two buffers."""
    rng = np.random.default_rng(80 + rows)
    H, hd, page = 2 * Hkv, 128, 64
    c = Cache(F16, page, Hkv, hd, -(-keys // page))
    b = Batch([rows], [keys], page, c.n_pages)
    fill_keys(c, b, rng)
    for f32 in (False, True):
        q = rng.standard_normal((b.M, H, hd)).astype(np.float32 if f32 else np.float16)
        want = run_attention(c, b, q, H, True, 0)
        cd, bd = c.desc(), b.desc()
        n = L().dfx_paged_attention_ws_bytes(ref(cd), ref(bd), H, F32 if f32 else F16)
        w, dq = dfx.Buf(n + 16), dfx.Buf.of(q)
        dfx.check(L().dfx_paged_attention(ref(cd), ref(bd), dq.ptr, F32 if f32 else F16, H, 1, 0, dq.ptr, w.ptr, None))
        dfx.sync()
        assert np.array_equal(dq.download(q.dtype, shape=q.shape), want)


@pytest.mark.parametrize("Hkv", [2, 60, 250])
@pytest.mark.parametrize("f32", [False, True])
def test_attention_without_keys_pages_or_rows(gpu, f32, Hkv):
    """No keys, fewer keys than rows, pages that are none in the middle and throughout: rows without a visible
    key give zeros, the others leave the missing keys out."""
    rng = np.random.default_rng(9)
    G, hd, page = 2, 128, 16
    H = Hkv * G
    c = Cache(F8, page, Hkv, hd, 12)
    pages = np.array([[0, 1, 2, -1], [3, -1, 4, 5], [6, 7, 12, 8], [-1, 1 << 30, -(1 << 31), 12], [9, 10, 11, -7]])
    b = Batch([3, 2, 20, 4, 50], [0, 60, 64, 50, 33], page, 12, pages=pages)
    fill_keys(c, b, rng)
    q = rng.standard_normal((b.M, H, hd)).astype(np.float32 if f32 else np.float16)
    for causal in (False, True):
        got = run_attention(c, b, q, H, causal, 0)
        check_attention(got, c, b, q, causal, 0, f32)
        assert (got[:3] == 0).all() and (got[25:29] == 0).all()
    b.set(keys=[-5, 1 << 30, 20, -(1 << 31), 4])          # counts out of range are held in it
    for causal in (False, True):
        check_attention(run_attention(c, b, q, H, causal, 0), c, b, q, causal, 0, f32)


@pytest.mark.parametrize("Hkv", [1, 10, 60])
@pytest.mark.parametrize("rows,keys", [(40, 3), (300, 100), (300, 0), (700, 30)])
def test_attention_of_more_rows_than_keys(gpu, rows, keys, Hkv):
    """Rows before the first position see nothing under the causal mask: zeros, however many."""
    rng = np.random.default_rng(rows)
    c = Cache(F8, 16, Hkv, 64, 12)
    b = Batch([rows, 5], [keys, 70], 16, 12)
    fill_keys(c, b, rng)
    q = rng.standard_normal((b.M, 2 * Hkv, 64)).astype(np.float16)
    for causal in (True, False):
        check_attention(run_attention(c, b, q, 2 * Hkv, causal, 0), c, b, q, causal, 0, False)


@pytest.mark.parametrize("Hkv", [1, 250, 1000])
def test_attention_of_extreme_queries(gpu, Hkv):
    """f32 queries from 1e-30 to 1e6, zeros, NaN and infinities: a row's range costs no accuracy and its NaN
    stays its own."""
    rng = np.random.default_rng(12)
    G, hd, page = 4, 64, 16
    c = Cache(F16, page, Hkv, hd, 8)
    b = Batch([9], [100], page, 8)
    fill_keys(c, b, rng)
    q = rng.standard_normal((9, Hkv * G, hd)).astype(np.float32)
    q[1] *= np.float32(1e-30)
    q[2] *= np.float32(1e-5)
    q[3] *= np.float32(300.0)
    q[4] = 0.0
    q[5, 0, 3] = np.nan
    q[6, 1] *= np.float32(1e-38)
    q[7, 2, :] = 1e6 * np.sign(q[7, 2])
    check_attention(run_attention(c, b, q, Hkv * G, True, 0), c, b, q, True, 0, True)
    h = np.clip(q, -60000, 60000).astype(np.float16)
    check_attention(run_attention(c, b, h, Hkv * G, True, 0), c, b, h, True, 0, False)


@pytest.mark.parametrize("Hkv", [2, 100])
@pytest.mark.parametrize("rows", [2, 45, 180])
@pytest.mark.parametrize("typ", [F8, F16])
def test_attention_of_extreme_values(gpu, typ, rows, Hkv):
    """Values at both ends of the cache's range; an f16 result that overflows is infinite."""
    rng = np.random.default_rng(13)
    hd, page = 64, 16
    n_pages = 10 if rows == 2 else 40
    c = Cache(typ, page, Hkv, hd, n_pages)
    b = Batch([rows, rows], [rows + 68, rows + 38], page, n_pages)
    fill_keys(c, b, rng)
    if c.f8:
        c.scale[..., 1] = np.where(rng.random(c.scale.shape[:3]) < 0.5, 2.0 ** 7, 2.0 ** -15)
    else:
        c.v[np.isfinite(c.v)] *= np.float16(10000)
        c.v[:, 1][np.isfinite(c.v[:, 1])] *= np.float16(2.0 ** -20)
    c.upload()
    for f32 in (True, False):
        q = rng.standard_normal((2 * rows, Hkv, hd)).astype(np.float32 if f32 else np.float16)
        check_attention(run_attention(c, b, q, Hkv, False, 0), c, b, q, False, 0, f32)


def test_cache_beyond_32_bits(gpu):
    """Pages whose cells start behind 4 GiB: written and read at their place."""
    rng = np.random.default_rng(14)
    Hkv, G, hd, page = 32, 1, 128, 256
    per = Hkv * page * hd * 2                                    # bytes of a page: 2 MiB
    n_pages = (9 << 30) // 2 // per + 3                          # 4.5 GiB of k, as much of v
    k, v = dfx.Buf(n_pages * per), dfx.Buf(n_pages * per)
    small = Cache(F16, page, Hkv, hd, 3, seed=1)
    ids = [n_pages - 1, 1, n_pages // 2 + 7]                     # small's page j stands for page ids[j]
    b = Batch([30], [300], page, n_pages, pages=np.array([ids[:2]]))
    sb = Batch([30], [300], page, 3, pages=np.array([[0, 1]]))
    fill_keys(small, sb, rng)
    for j, p in enumerate(ids):
        for buf, src in ((k, small.dk), (v, small.dv)):
            dfx.check(L().dfx_memcpy_d2d(C.c_void_p(buf.ptr.value + p * per), C.c_void_p(src.ptr.value + j * per), per, None))
    cd, bd = dfx.PagedCache(F16, page, Hkv, hd, n_pages, k.ptr, v.ptr, None), b.desc()
    tab = rope_table(300, hd)
    qkv = qkv_of(rng, 30, 3 * Hkv, hd)
    want = np.empty((30, Hkv, hd), np.float16)
    ref_append(small, sb, qkv, Hkv, tab, want)
    dq, dx, dt = dfx.Buf(want.nbytes), dfx.Buf.of(qkv), dfx.Buf.of(tab)
    dfx.check(L().dfx_paged_append(ref(cd), ref(bd), dx.ptr, Hkv, dt.ptr, 300, F16, dq.ptr, None), "append")
    do = dfx.Buf(want.nbytes)
    ws = dfx.Buf(max(16, L().dfx_paged_attention_ws_bytes(ref(cd), ref(bd), Hkv, F16)))
    dfx.check(L().dfx_paged_attention(ref(cd), ref(bd), dq.ptr, F16, Hkv, 1, 0, do.ptr, ws.ptr, None), "attention")
    dfx.sync()
    assert np.array_equal(dq.download(np.float16, shape=want.shape), want)
    check_attention(do.download(np.float16, shape=want.shape), small, sb, want, True, 0, False)


# ---------------------------------------------------------------- streams and graphs
def test_two_streams_at_once(gpu):
    """Two batches on two streams, each with its own workspace and pages of one cache: as one after the other."""
    rng = np.random.default_rng(15)
    Hkv, G, hd, page = 2, 2, 64, 16
    H = Hkv * G
    c = Cache(F8, page, Hkv, hd, 200)
    ids = rng.permutation(200)
    bs = [Batch([1, 3], [1500, 40], page, 200, pages=np.stack([ids[:94], ids[94:188]])),
          Batch([20], [150], page, 200, pages=ids[188:200][None])]
    for b in bs:
        fill_keys(c, b, rng)
    qs = [rng.standard_normal((b.M, H, hd)).astype(np.float32) for b in bs]
    want = [run_attention(c, b, q, H, True, 0) for b, q in zip(bs, qs)]
    st = []
    for _ in bs:
        s = C.c_void_p()
        dfx.check(L().dfx_stream_create(C.byref(s)))
        st.append(s)
    cd, bd = c.desc(), [b.desc() for b in bs]
    dq, do = [dfx.Buf.of(q) for q in qs], [dfx.Buf(q.nbytes) for q in qs]
    ws = [dfx.Buf(max(16, L().dfx_paged_attention_ws_bytes(ref(cd), ref(d), H, F32))) for d in bd]
    for _ in range(5):
        for i in range(2):
            dfx.check(L().dfx_paged_attention(ref(cd), ref(bd[i]), dq[i].ptr, F32, H, 1, 0, do[i].ptr, ws[i].ptr, st[i]))
    for i in range(2):
        dfx.sync(st[i])
        assert np.array_equal(do[i].download(np.float32, shape=qs[i].shape), want[i])
        dfx.check(L().dfx_stream_destroy(st[i]))


def test_captured_step_follows_the_device_arrays(gpu):
    """Append and attention of a decoding step captured once and replayed while the key counts grow and
    sequences come and go in the device arrays, with eager work between the replays."""
    hip = C.CDLL("libamdhip64.so")
    rng = np.random.default_rng(16)
    Hkv, G, hd, page, S = 2, 2, 64, 16, 3
    H = Hkv * G
    c = Cache(F8, page, Hkv, hd, 3 * 100)
    b = Batch([1] * S, [700, 30, 16], page, 300, pages=rng.permutation(300).reshape(3, 100), max_keys=1600)
    fill_keys(c, b, rng)
    tab = rope_table(1600, hd)
    qkv = qkv_of(rng, S, H + 2 * Hkv, hd)
    cd, bd = c.desc(), b.desc()
    dx, dt = dfx.Buf.of(qkv), dfx.Buf.of(tab)
    dq, do = dfx.Buf.of(np.zeros((S, H, hd), np.float16)), dfx.Buf.of(np.full((S, H, hd), 7.0, np.float16))
    n = L().dfx_paged_attention_ws_bytes(ref(cd), ref(bd), H, F16)
    assert n > 0
    ws = dfx.Buf(n)
    st, graph, ex = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(st), 1) == 0
    assert hip.hipStreamBeginCapture(st, 0) == 0
    rc = [L().dfx_paged_append(ref(cd), ref(bd), dx.ptr, H, dt.ptr, len(tab), F16, dq.ptr, st),
          L().dfx_paged_attention(ref(cd), ref(bd), dq.ptr, F16, H, 1, 0, do.ptr, ws.ptr, st)]
    assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0 and rc == [0, 0]
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    want_q = np.zeros((S, H, hd), np.float16)
    for n_rows, keys in (([1, 1, 1], [701, 31, 17]), ([1, 1, 1], [702, 32, 18]), ([1, 0, 1], [1500, 32, 19]),
                         ([0, 0, 1], [1500, 0, 20]), ([1, 1, 1], [1501, 1, 21])):
        b.set(n_rows, keys)
        fill_keys(c, b, rng)
        x = qkv_of(rng, S, H + 2 * Hkv, hd)
        dx.upload(x)
        dfx.sync()
        assert hip.hipGraphLaunch(ex, st) == 0 and hip.hipStreamSynchronize(st) == 0
        ref_append(c, b, x, H, tab, want_q)
        assert np.array_equal(dq.download(np.float16, shape=want_q.shape), want_q)
        k, v, sc = c.download()
        assert same_cells(c, k, c.k) and same_cells(c, v, c.v) and np.array_equal(sc, c.scale)
        got = do.download(np.float16, shape=want_q.shape)
        check_attention(got, c, b, want_q, True, 0, False)
        live = int(b.rows[-1])
        assert np.array_equal(got[:live], run_attention(c, b, want_q, H, True, 0)[:live])   # eager, the same split
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    hip.hipStreamDestroy(st)


FIRST_CAPTURE = r"""
import ctypes as C, sys
import numpy as np
sys.path[:0] = sys.argv[1:3]
import dfx
from paged_ref import Batch, Cache, ref, rope_table
from test_gpu_paged import fill_keys
hip, L = C.CDLL("libamdhip64.so"), dfx.lib
rng = np.random.default_rng(5)
st = C.c_void_p()
assert hip.hipStreamCreateWithFlags(C.byref(st), 1) == 0
# the kernels that take more LDS than a launch has by default: some rows, many rows
for n, Hkv, G in ((300, 32, 1), (300, 32, 4)):
    H, hd, page = Hkv * G, 128, 64
    c = Cache(dfx.TYPE_F16, page, Hkv, hd, 6)
    b = Batch([n], [n + 20], page, 6)
    fill_keys(c, b, rng)
    for typ, nt in ((dfx.TYPE_F16, np.float16), (dfx.TYPE_F32, np.float32)):
        q = rng.standard_normal((n, H, hd)).astype(nt)
        dq, do = dfx.Buf.of(q), dfx.Buf.of(np.zeros_like(q))
        cd, bd = c.desc(), b.desc()
        graph, ex = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(st, 0) == 0                # global capture mode, the first call of its kind
        rc = L().dfx_paged_attention(ref(cd), ref(bd), dq.ptr, typ, H, 1, 0, do.ptr, None, st)
        assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
        dfx.check(rc, "attention under capture")
        assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
        de = dfx.Buf.of(np.zeros_like(q))
        for rep in range(3):
            do.upload(np.zeros_like(q))
            dfx.check(L().dfx_paged_attention(ref(cd), ref(bd), dq.ptr, typ, H, 1, 0, de.ptr, None, None))
            dfx.sync()
            assert hip.hipGraphLaunch(ex, st) == 0 and hip.hipStreamSynchronize(st) == 0
            assert np.array_equal(do.download(nt), de.download(nt)) and np.isfinite(do.download(nt)).all()
print("capture ok")
"""


def test_first_call_under_stream_capture(gpu, tmp_path):
    """The first call of a process into the kernels whose LDS limit is raised, inside a global-mode capture."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    script = tmp_path / "first.py"
    script.write_text(FIRST_CAPTURE)
    r = subprocess.run([sys.executable, str(script), here, os.path.join(os.path.dirname(here), "diffuse-cpp_amd")],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "capture ok" in r.stdout, (r.returncode, r.stdout[-2000:], r.stderr[-2000:])


def test_table_of_cells_is_exact(gpu):
    """Every E4M3 code at every scale reaches the attention as its exact value: one key per row, so that
    the result is the value itself."""
    Hkv, hd, page = 1, 128, 16
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    c = Cache(F8, page, Hkv, hd, 2 * 23)
    S = 46
    pages = np.arange(S)[:, None]
    b = Batch([1] * S, [1] * S, page, S, pages=pages)
    for s in range(S):
        c.scale[s] = 2.0 ** (s // 2 - 15)
        c.k[s, 0, 0] = 0
        c.v[s, 0, 0, :, 0] = codes[:128] if s % 2 == 0 else np.concatenate([codes[126:], codes[:0]])
    c.upload()
    q = np.zeros((S, 1, hd), np.float16)
    got = run_attention(c, b, q, 1, True, 0)
    for s in range(S):
        want = (TABLE[c.v[s, 0, 0, :, 0]] * float(c.scale[s, 0, 0, 1]))
        assert np.array_equal(got[s, 0].astype(np.float64), want), s
