"""dfx_token_logprobs against its definition in float64, and together with the operators that come before
it in a step."""
import ctypes as C

import numpy as np
import pytest

import dfx
from paged_ref import Batch, Cache, attention_bound, ref, ref_append, ref_attention, rope_table

pytestmark = pytest.mark.gpu
L = dfx.lib


def run(logits, V=None, rows=None, tokens=None, top=0, entropy=True, n_logits=None, offset=0):
    """(logprob, entropy, top_id, top_logprob) of the library."""
    n_all, ld = logits.shape
    V = ld if V is None else V
    n = n_all if rows is None else len(rows)
    flat = np.concatenate([np.zeros(offset, np.float32), np.ascontiguousarray(logits).ravel()])
    dl = dfx.Buf.of(flat)
    lp = C.c_void_p(dl.ptr.value + 4 * offset)
    dr = dfx.Buf.of(np.asarray(rows, np.int32)) if rows is not None else None
    tokens = np.zeros((n, 0), np.int32) if tokens is None else np.asarray(tokens, np.int32)
    nt = tokens.shape[1]
    dt = dfx.Buf.of(tokens)
    do, de = dfx.Buf.of(np.full((n, max(nt, 1)), 7.0, np.float32)), dfx.Buf.of(np.full(n, 7.0, np.float32))
    di, dv = dfx.Buf.of(np.full((n, max(top, 1)), 7, np.int32)), dfx.Buf.of(np.full((n, max(top, 1)), 7.0, np.float32))
    nb = L().dfx_token_logprobs_ws_bytes(n, V, top)
    ws = dfx.Buf.of(np.full(nb, 0xFF, np.uint8))
    dfx.check(L().dfx_token_logprobs(lp, ld, n_all if n_logits is None else n_logits, dr.ptr if dr else None, n, V,
                                     dt.ptr if nt else None, nt, do.ptr if nt else None, de.ptr if entropy else None,
                                     top, di.ptr if top else None, dv.ptr if top else None, ws.ptr, None), "logprobs")
    dfx.sync()
    return (do.download(np.float32, shape=(n, max(nt, 1)))[:, :nt], de.download(np.float32),
            di.download(np.int32, shape=(n, max(top, 1)))[:, :top], dv.download(np.float32, shape=(n, max(top, 1)))[:, :top])


def define(x, tokens, top):
    """The definition for one row in float64."""
    x = x.astype(np.float64)
    V = len(x)
    with np.errstate(all="ignore"):
        m = np.nanmax(x) if not np.isnan(x).all() else np.nan
        e = np.exp(x - m)
        lp = (x - m) - np.log(e.sum())                       # m + log S would lose log S next to 1e38
        p = np.exp(lp)
        ent = -np.where(p > 0, p * lp, np.where(np.isnan(p), np.nan, 0.0)).sum()
    order = np.lexsort((np.arange(V), -np.where(np.isnan(x), -np.inf, x)))[:top]
    ids = np.concatenate([order, np.full(top - len(order), -1)])
    best = np.concatenate([lp[order], np.full(top - len(order), -np.inf)])
    return np.array([lp[t] if 0 <= t < V else np.nan for t in tokens]), ent, ids, best


def check(got, logits, V=None, rows=None, tokens=None, top=0, n_logits=None):
    """Bounds: exp and its argument are off by 2^-21 of a term at most (|x - m| log2 e below 2^7 matters: beyond,
    the term is 0 in float), a lane's f32 sums of 64 terms by 64 * 2^-24; log S so by 2^-17 in all, and
    the result's rounding is 2^-24 of it.  The entropy is log S - T / S: T's terms and S's error weigh with
    its size, at most |entropy| + log V."""
    n_all = len(logits) if n_logits is None else n_logits
    V = logits.shape[1] if V is None else V
    idx = range(len(logits)) if rows is None else rows
    for i, r in enumerate(idx):
        tk = [] if tokens is None else tokens[i]
        if 0 <= r < n_all:
            lp, ent, ids, best = define(logits[r, :V], tk, top)
        else:
            lp, ent, ids, best = np.full(len(tk), np.nan), np.nan, np.full(top, -1), np.full(top, np.nan)
        assert np.array_equal(got[2][i], ids), (i, r)
        for g, w in ((got[0][i], lp), (got[3][i], best)):
            g, w = np.asarray(g, np.float64), np.asarray(w, np.float64)
            assert np.array_equal(np.isnan(g), np.isnan(w)), (i, g, w)
            with np.errstate(invalid="ignore"):
                fin = np.isfinite(w) & (np.abs(w) < 3.4e38)
            assert np.array_equal(g[~fin & ~np.isnan(w)], w[~fin & ~np.isnan(w)])
            assert (np.abs(g[fin] - w[fin]) <= 2.0 ** -17 + 2.0 ** -24 * np.abs(w[fin])).all(), (i, np.abs(g[fin] - w[fin]).max())
        if np.isnan(ent):
            assert np.isnan(got[1][i])
        else:
            assert abs(got[1][i] - ent) <= 2.0 ** -17 * (1 + abs(ent) + np.log(V)), (i, got[1][i], ent)


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 100, 1021, 4096, 4099, 16384, 32000, 126464, 152064])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_against_the_definition(gpu, V, top):
    rng = np.random.default_rng(V + top)
    n = 3
    x = (rng.standard_normal((n, V)) * rng.uniform(0.5, 4.0, (n, 1))).astype(np.float32)
    x[0, rng.integers(0, V)] += 30.0
    tokens = rng.integers(0, V, (n, 2))
    check(run(x, tokens=tokens, top=top), x, tokens=tokens, top=top)


@pytest.mark.parametrize("n,V", [(300, 70001), (1100, 16384), (150, 126464)])
def test_many_rows(gpu, n, V):
    """The longer pieces that many rows take, both load widths."""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((n, V)) * 3).astype(np.float32)
    tokens = rng.integers(0, V, (n, 1))
    got = run(x, tokens=tokens, top=20)
    pick = sorted({0, 1, n // 2, n - 1} | set(rng.integers(0, n, 8).tolist()))
    check([g[pick] for g in got], x, rows=pick, tokens=tokens[pick], top=20)


@pytest.mark.parametrize("ld,offset", [(1500, 0), (1501, 0), (1500, 1), (1500, 4), (1503, 3)])
def test_strides_rows_and_alignment(gpu, ld, offset):
    """Rows picked in any order and twice, row strides beyond V (NaN between the rows), unaligned rows."""
    rng = np.random.default_rng(ld + offset)
    x = rng.standard_normal((6, ld)).astype(np.float32)
    V = 1499 if ld % 2 else 1496
    x[:, V:] = np.nan
    rows = [5, 0, 0, 3, -1, 6, 5, 1 << 30, -(1 << 31)]
    tokens = rng.integers(-2, V + 2, (len(rows), 3))
    tokens[0] = [-1, V, 1 << 30]
    check(run(x, V=V, rows=rows, tokens=tokens, top=7, offset=offset), x, V=V, rows=rows, tokens=tokens, top=7)
    check(run(x, V=V, rows=[0, 4, 3], top=3, n_logits=4, offset=offset), x, V=V, rows=[0, 4, 3], top=3, n_logits=4)


@pytest.mark.parametrize("V", [50, 5000, 126464])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_equal_masked_and_special_logits(gpu, V, top):
    """Ties throughout, masks of -inf and of the lowest float, +-0, NaN, +inf, rows with nothing left."""
    rng = np.random.default_rng(V + top)
    x = (rng.standard_normal((14, V)) * 2).astype(np.float32)
    x[0] = 1.5                                               # all equal
    x[1] = np.round(x[1])                                    # a few values, many times each
    x[2] = -np.inf                                           # nothing left
    x[3, rng.permutation(V)[3:]] = -np.inf                   # three left
    x[4, rng.permutation(V)[3:]] = np.finfo(np.float32).min  # three left, masked by the lowest value
    x[5] = np.where(rng.random(V) < 0.5, np.float32(0.0), np.float32(-0.0))
    x[6, rng.integers(0, V, 4)] = np.nan
    x[7] = np.nan
    x[8, rng.integers(0, V, 2)] = np.inf
    x[9] *= np.float32(1e30)
    x[10] -= np.float32(1e6)
    x[11] = np.finfo(np.float32).min
    x[12, V // 2:] = -np.inf
    x[13] = -np.float32(1e-40)                               # equal, below the normal range
    x[13, V // 3] = np.float32(1e-41)
    tokens = rng.integers(0, V, (14, 2))
    with np.errstate(all="ignore"):
        check(run(x, tokens=tokens, top=top), x, tokens=tokens, top=top)


@pytest.mark.parametrize("V", [1500, 126464, 126465])
@pytest.mark.parametrize("top", [20, 64])
def test_best_logits_side_by_side(gpu, V, top):
    """The largest logits as neighbours, every fourth, 64 apart and 256 apart (one lane's elements), and runs of
    equal values across lanes: the same order, the lowest index first."""
    rng = np.random.default_rng(V + top)
    x = rng.standard_normal((8, V)).astype(np.float32)
    for r, step in enumerate((1, 2, 4, 64, 256)):
        at = 7 + step * np.arange(min(80, (V - 8) // step))
        x[r, at] = 20 + rng.standard_normal(len(at)).astype(np.float32)
    x[5, 100:1000] = 9.0
    x[6, 5::3] = 4.0
    x[7, V // 2:] = np.float32(np.finfo(np.float32).min)
    x[7, :V // 2] = np.where(rng.random(V // 2) < 30.0 / V, x[7, :V // 2], np.float32(np.finfo(np.float32).min))
    tokens = rng.integers(0, V, (8, 1))
    check(run(x, tokens=tokens, top=top), x, tokens=tokens, top=top)


def test_ids_and_values_against_row_stats(gpu):
    """The best alternative and the entropy are those of dfx_row_stats on the same rows."""
    rng = np.random.default_rng(4)
    n, V = 9, 126464
    x = (rng.standard_normal((n, V)) * 2).astype(np.float32)
    lp, ent, ids, best = run(x, top=2)
    dl, dr, ds = dfx.Buf.of(x), dfx.Buf.of(np.arange(n, dtype=np.int32)), dfx.Buf(n * 16)
    dfx.check(L().dfx_row_stats(dl.ptr, V, dr.ptr, n, V, ds.ptr, None), "row_stats")
    st = ds.download(dfx.ROW_STAT)
    assert np.array_equal(st["token"], ids[:, 0])
    # both within their bounds of the definition (row statistics: 1e-4 relative and 2e-5)
    assert (np.abs(st["entropy"] - ent) <= 1e-4 * np.abs(ent) + 2e-5 + 2.0 ** -17 * 25).all()
    # the difference of the two best is the difference of the logits: two roundings of each
    d = np.abs((best[:, 0] - best[:, 1]) - (st["best"] - st["second"]))
    assert (d <= 2.0 ** -23 * (np.abs(best[:, 0]) + np.abs(best[:, 1]) + np.abs(st["best"]))).all()


def test_captured_scores(gpu):
    """Scores captured once and replayed over other logits and tokens, with eager calls between."""
    hip = C.CDLL("libamdhip64.so")
    rng = np.random.default_rng(17)
    n, V, top = 3, 5000, 20
    dl, dt = dfx.Buf(n * V * 4), dfx.Buf(n * 4)
    do, de, di, dv = dfx.Buf(n * 4), dfx.Buf(n * 4), dfx.Buf(n * top * 4), dfx.Buf(n * top * 4)
    ws = dfx.Buf(L().dfx_token_logprobs_ws_bytes(n, V, top))
    st, graph, ex = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(st), 1) == 0 and hip.hipStreamBeginCapture(st, 0) == 0
    rc = L().dfx_token_logprobs(dl.ptr, V, n, None, n, V, dt.ptr, 1, do.ptr, de.ptr, top, di.ptr, dv.ptr, ws.ptr, st)
    assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0 and rc == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    for rep in range(4):
        x = (rng.standard_normal((n, V)) * 2).astype(np.float32)
        if rep == 2:
            x[1] = 3.0
        tokens = rng.integers(0, V, (n, 1)).astype(np.int32)
        dl.upload(x)
        dt.upload(tokens)
        dfx.sync()
        assert hip.hipGraphLaunch(ex, st) == 0 and hip.hipStreamSynchronize(st) == 0
        got = (do.download(np.float32, shape=(n, 1)), de.download(np.float32), di.download(np.int32, shape=(n, top)),
               dv.download(np.float32, shape=(n, top)))
        check(got, x, tokens=tokens, top=top)
        for g, w in zip(got, run(x, tokens=tokens, top=top)):
            assert np.array_equal(g, w)
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    hip.hipStreamDestroy(st)


@pytest.mark.parametrize("typ", [dfx.TYPE_F8, dfx.TYPE_F16])
def test_a_step_of_many_sequences(gpu, typ):
    """Prompts, then two decoding steps: append, attention with f16 results straight into an F16 GEMM (the
    head), scores of given tokens; the cache and the scores against float64."""
    rng = np.random.default_rng(21)
    Hkv, G, hd, page, V = 2, 4, 64, 32, 1280
    H = Hkv * G
    K = H * hd
    head = (rng.standard_normal((V, K)) * 0.05).astype(np.float16)
    dw = dfx.Buf.of(dfx.repack(dfx.TYPE_F16, head.view(np.uint8), V, K))
    c = Cache(typ, page, Hkv, hd, 12)
    tab = rope_table(100, hd)
    pages = rng.permutation(12).reshape(3, 4)
    past = [0, 0, 0]
    for n in ([40, 17, 3], [1, 1, 1], [1, 0, 1]):
        past = [a + m for a, m in zip(past, n)]
        b = Batch(n, past, page, 12, pages=pages, max_keys=128)
        M = b.M
        qkv = rng.standard_normal((M, H + 2 * Hkv, hd)).astype(np.float32)
        cd, bd = c.desc(), b.desc()
        dx, dt, dq = dfx.Buf.of(qkv), dfx.Buf.of(tab), dfx.Buf(M * K * 2)
        act = dfx.Buf(L().dfx_act_bytes(dfx.TYPE_F16, M, K))
        dfx.check(L().dfx_paged_append(ref(cd), ref(bd), dx.ptr, H, dt.ptr, len(tab), dfx.TYPE_F16, dq.ptr, None))
        ws = dfx.Buf(max(16, L().dfx_paged_attention_ws_bytes(ref(cd), ref(bd), H, dfx.TYPE_F16)))
        dfx.check(L().dfx_paged_attention(ref(cd), ref(bd), dq.ptr, dfx.TYPE_F16, H, 1, 0, act.ptr, ws.ptr, None))
        y = dfx.Buf(M * V * 4)
        dfx.check(L().dfx_gemm(dfx.TYPE_F16, dw.ptr, V, K, act.ptr, M, None, None, y.ptr, None, None))
        dfx.sync()
        tokens = rng.integers(0, V, (M, 1))
        logits = y.download(np.float32, shape=(M, V))
        got = run(logits, tokens=tokens, top=5)
        check(got, logits, tokens=tokens, top=5)
        q = np.zeros((M, H, hd), np.float16)
        ref_append(c, b, qkv, H, tab, q)
        out, A, E = ref_attention(c, b, q, True, 0)
        tol = attention_bound(out, A, E, hd, max(past), False).reshape(M, K)
        w = head.astype(np.float64)
        want = out.reshape(M, K) @ w.T
        # the head: its inputs' error, and K f32 sums
        lim = tol @ np.abs(w).T + 2 * K * 2.0 ** -24 * (np.abs(out.reshape(M, K)) @ np.abs(w).T)
        assert (np.abs(logits - want) <= lim).all()
        z = want - want.max(1, keepdims=True)
        lse = np.log(np.exp(z).sum(1, keepdims=True))
        lp = np.take_along_axis(z - lse, tokens, 1)
        # an error d of every logit moves a log probability by 2 d at most
        assert (np.abs(got[0] - lp) <= 2 * lim.max(1, keepdims=True) + 2.0 ** -16).all()
