"""The operators of serving many sequences and of scoring tokens, in their plain form and as the library's calls.

Kinds of case:

  append    Q and K of a ragged batch rotated, K and V appended to a paged cache (dfx_paged_append)
  attend    attention of a ragged batch over a paged cache (dfx_paged_attention)
  score     log probabilities of given tokens, entropy and best alternatives of logits rows (dfx_token_logprobs)

A batch: the rows of sequence s are rows[s] .. rows[s + 1] - 1 and stand at the last positions of its n_keys[s] keys.
A cache: pages of `page` tokens, k [pages][Hkv][page][hd] and v [pages][Hkv][page / 16][hd][16], in f16 or in
E4M3 with one power of two per block of 16 tokens and head, scale [pages][Hkv][page / 16][K, V].

Head layouts and vocabularies are the benchmark's architectures and the tests' small ones.  Plain forms compute in 32 bits
with elementary torch operations; exact() computes in 64.
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
# heads, KV heads, head size, rope base, vocabulary
ARCH = {"llada-8b": (32, 32, 128, 500000.0, 126464), "dream-7b": (28, 4, 128, 1000000.0, 152064),
        "small": (4, 4, 128, 500000.0, 1536), "small-gqa": (8, 2, 64, 1000000.0, 1280)}
F8 = torch.float8_e4m3fn
TYPE = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token of one sequence: launch latency
        {"name": "append_token", "kind": "append", "arch": "dream-7b", "cache": "f8", "type": "f16", "page": 64,
         "seqs": 1, "rows_lo": 1, "rows_hi": 1, "past_lo": 191, "past_hi": 191},
        # a decoding step of 64 sequences, one token each
        {"name": "append_step_64", "kind": "append", "arch": "llada-8b", "cache": "f8", "type": "f16", "page": 64,
         "seqs": 64, "rows_lo": 1, "rows_hi": 1, "past_lo": 16, "past_hi": 4000},
        # chunks of prompts of eight sequences, continuing earlier ones, for the f32-accurate attention
        {"name": "append_prompts", "kind": "append", "arch": "dream-7b", "cache": "f8", "type": "f32", "page": 64,
         "seqs": 8, "rows_lo": 200, "rows_hi": 1000, "past_lo": 1, "past_hi": 2000},
        # whole prompts into an f16 cache
        {"name": "append_prompts_f16", "kind": "append", "arch": "llada-8b", "cache": "f16", "type": "f16", "page": 128,
         "seqs": 5, "rows_lo": 300, "rows_hi": 1500, "past_lo": 0, "past_hi": 0},
        # one token after a long context: the cache is split over the chip
        {"name": "attend_token_32k", "kind": "attend", "arch": "dream-7b", "cache": "f8", "type": "f16", "page": 64,
         "seqs": 1, "rows_lo": 1, "rows_hi": 1, "past_lo": 32700, "past_hi": 32700, "causal": True, "window": 0},
        # a decoding step of 64 sequences of very different lengths
        {"name": "attend_step_64", "kind": "attend", "arch": "llada-8b", "cache": "f8", "type": "f16", "page": 64,
         "seqs": 64, "rows_lo": 1, "rows_hi": 1, "past_lo": 16, "past_hi": 4000, "causal": True, "window": 0},
        # a denoising step: the active rows of eight sequences see all their positions (512 + 256), f32 as the contexts
        {"name": "attend_denoise", "kind": "attend", "arch": "llada-8b", "cache": "f16", "type": "f32", "page": 16,
         "seqs": 8, "rows_lo": 24, "rows_hi": 96, "past_lo": 512, "past_hi": 700, "causal": False, "window": 0},
        # whole prompts, causal
        {"name": "attend_prompts", "kind": "attend", "arch": "dream-7b", "cache": "f8", "type": "f16", "page": 64,
         "seqs": 4, "rows_lo": 1500, "rows_hi": 4000, "past_lo": 0, "past_hi": 100, "causal": True, "window": 0},
        # chunks of prompts with a sliding window, small heads
        {"name": "attend_window", "kind": "attend", "arch": "small-gqa", "cache": "f16", "type": "f16", "page": 32,
         "seqs": 6, "rows_lo": 100, "rows_hi": 700, "past_lo": 0, "past_hi": 3000, "causal": True, "window": 512},
        # one sampled token with the alternatives that an API returns
        {"name": "score_token", "kind": "score", "arch": "dream-7b", "n": 1, "given": 1, "top": 5},
        # a block of 256 masked positions, 20 alternatives each
        {"name": "score_256", "kind": "score", "arch": "llada-8b", "n": 256, "given": 1, "top": 20},
        # likelihood of a text: the given tokens and entropy only
        {"name": "score_text", "kind": "score", "arch": "dream-7b", "n": 700, "given": 1, "top": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1))))))))


def draw(rng):
    """One more case: 1 to 96 sequences, 1 to 800 rows each, up to 32000 keys; logits of 1 to 700 rows."""
    kind = rng.choice(["append", "attend", "attend", "score"])
    arch = rng.choice(["llada-8b", "dream-7b", "dream-7b", "small", "small-gqa"])
    if kind == "score":
        return {"kind": kind, "arch": arch, "n": _log(rng, 1, 700), "given": rng.choice([1, 1, 1, 4]),
                "top": rng.choice([0, 1, 5, 20, 64])}
    c = {"kind": kind, "arch": arch, "cache": rng.choice(["f8", "f8", "f16"]), "type": rng.choice(["f16", "f16", "f32"]),
         "page": rng.choice([16, 32, 64, 128])}
    if rng.random() < 0.4:                              # decoding: one token of each sequence
        seqs = _log(rng, 1, 96)
        top = 32000 if seqs <= 4 else 4000
        c.update(seqs=seqs, rows_lo=1, rows_hi=1, past_lo=rng.choice([0, 1, 100]), past_hi=_log(rng, 100, top))
    else:                                               # denoising steps and prompts
        seqs = _log(rng, 1, 6)
        hi = _log(rng, 2, 800)
        c.update(seqs=seqs, rows_lo=max(1, hi // 4), rows_hi=hi, past_lo=0,
                 past_hi=0 if rng.random() < 0.2 else _log(rng, 1, 2000))
    if kind == "attend":
        c["causal"] = rng.random() < 0.6
        c["window"] = _log(rng, 16, 2000) if c["causal"] and rng.random() < 0.3 else 0
    return c


def _lengths(case):
    """Rows and keys of each sequence: the case alone decides."""
    rng = random.Random("%s %s %s" % (case["seqs"], case["rows_hi"], case["past_hi"]))
    n, keys = [], []
    for _ in range(case["seqs"]):
        r = _log(rng, case["rows_lo"], case["rows_hi"])
        past = 0 if not case["past_hi"] else max(case["past_lo"], _log(rng, 1, case["past_hi"]))
        n.append(r)
        keys.append(past + r)
    return n, keys


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _scale_of(a):
    """The power of two that a block of largest magnitude a takes: the least with a <= 448 * 2^k, k in -15..7."""
    m, e = torch.frexp(a)                                          # a = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    k = torch.where(a > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -15)).clamp(-15, 7)
    return torch.ldexp(torch.ones_like(a), k)


def _cells(x, scale):
    """E4M3 cells of x / scale as bytes; what is not finite becomes NaN."""
    y = torch.where(torch.isfinite(x), (x / scale).clamp(-448.0, 448.0), torch.full_like(x, math.nan))
    return y.to(F8).view(torch.uint8)


def _filled(g, case, n_pages, Hkv, hd):
    """A pool of pages that holds keys with uneven channels and values, as a model leaves them."""
    P, B = case["page"], case["page"] // 16
    ch = 0.5 + 1.5 * torch.rand(Hkv, 1, 1, hd, generator=g, device=DEV)
    kx = _randn(g, n_pages, Hkv, B, 16, hd) * ch
    vx = _randn(g, n_pages, Hkv, B, hd, 16)
    if case["cache"] == "f16":
        return kx.half().reshape(n_pages, Hkv, P, hd), vx.half(), None
    sc = torch.stack([_scale_of(kx.abs().amax((3, 4))), _scale_of(vx.abs().amax((3, 4)))], -1)
    k = _cells(kx, sc[..., 0, None, None]).reshape(n_pages, Hkv, P, hd)
    return k, _cells(vx, sc[..., 1, None, None]), sc


def _rope_table(n_pos, hd, base):
    theta = torch.arange(n_pos, dtype=torch.float64)[:, None] * base ** (-torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
    return torch.stack([theta.cos(), theta.sin()], -1).float().to(DEV)


def prepare(case, seed):
    g = _gen(seed)
    H, Hkv, hd, base, V = ARCH[case["arch"]]
    if case["kind"] == "score":
        n = case["n"]
        logits = _randn(g, n, V) * (0.5 + 3.5 * torch.rand(n, 1, generator=g, device=DEV))
        # the head's rows in the order of the pass; the sampler reads them in another
        rows = torch.randperm(n, generator=g, device=DEV).int()
        tokens = torch.randint(0, V, (n, case["given"]), generator=g, device=DEV, dtype=torch.int32)
        likely = logits[rows.long()].argmax(1).int()
        tokens[::2, 0] = likely[::2]
        return {"kind": "score", "V": V, "top": case["top"], "logits": logits, "rows": rows, "tokens": tokens}
    P, S = case["page"], case["seqs"]
    n, keys = _lengths(case)
    rows = torch.tensor([0] + n).cumsum(0)
    M = int(rows[-1])
    per_seq = [-(-x // P) for x in keys]
    # an append touches its last pages; the pages before them are a prefix that the sequences share
    own_from = [(x - m) // P if case["kind"] == "append" else 0 for x, m in zip(keys, n)]
    n_pages = 3 + sum(a - b for a, b in zip(per_seq, own_from))
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    shared, free = order[0], order[1:]
    pages = torch.zeros(S, max(per_seq), dtype=torch.int32)
    for s in range(S):
        mine = [shared] * own_from[s] + [free.pop() for _ in range(per_seq[s] - own_from[s])]
        pages[s, :per_seq[s]] = torch.tensor(mine, dtype=torch.int32)
    k, v, scale = _filled(g, case, n_pages, Hkv, hd)
    st = {"kind": case["kind"], "H": H, "Hkv": Hkv, "hd": hd, "page": P, "S": S, "M": M, "max_keys": max(keys),
          "max_rows": max(n), "f8": case["cache"] == "f8", "type": case["type"], "k": k, "v": v, "scale": scale,
          "rows": rows.int().to(DEV), "n_keys": torch.tensor(keys, dtype=torch.int32, device=DEV), "pages": pages.to(DEV)}
    if case["kind"] == "append":
        st["qkv"] = _randn(g, M, H + 2 * Hkv, hd) * (0.3 + 1.7 * torch.rand(1, H + 2 * Hkv, 1, generator=g, device=DEV))
        st["tab"] = _rope_table(max(keys), hd, base)
    else:
        st["q"] = (_randn(g, M, H, hd) * 1.5).to(TYPE[case["type"]])
        st["causal"], st["window"] = case["causal"], case["window"]
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _places(st):
    """Sequence and position of every row."""
    r = torch.arange(st["M"], device=DEV)
    s = torch.searchsorted(st["rows"][1:].long(), r, right=True)
    return s, st["n_keys"].long()[s] - (st["rows"].long()[s + 1] - r)


def _append(st):
    H, Hkv, hd, P = st["H"], st["Hkv"], st["hd"], st["page"]
    half = hd // 2
    s, pos = _places(st)
    c, sn = st["tab"][pos].unbind(-1)
    qk = st["qkv"][:, :H + Hkv]
    x0, x1, c, sn = qk[..., :half], qk[..., half:], c[:, None], sn[:, None]
    y = torch.cat([x0 * c - x1 * sn, x0 * sn + x1 * c], -1)
    q = y[:, :H].to(TYPE[st["type"]])
    kx, vx = y[:, H:], st["qkv"][:, H + Hkv:]
    page, tok = st["pages"].long()[s, pos // P], pos % P
    k, v = st["k"], st["v"]
    if not st["f8"]:
        k[page, :, tok] = kx.half()
        v[page, :, tok // 16, :, tok % 16] = vx.half()
        return q, k, v
    B = P // 16
    scale = st["scale"]                                                    # [pages][Hkv][B][2]
    flat = scale.transpose(1, 2).reshape(-1, Hkv, 2)                       # by block
    blk = page * B + tok // 16
    amax = torch.stack([torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1) for x in (kx, vx)], -1)
    new = torch.zeros_like(flat).scatter_reduce(0, blk[:, None, None].expand_as(amax), amax, "amax")
    new = _scale_of(new)
    # a sequence's first row may stand inside a block: its earlier tokens keep their places
    first = st["rows"].long()[:-1]
    at, kept = blk[first], pos[first] % 16
    old = flat[at]
    both = torch.where((kept > 0)[:, None, None], torch.maximum(old, new[at]), new[at])
    new[at] = both
    ratio = old / both
    stays = torch.arange(16, device=DEV) < kept[:, None]                   # [S][16]
    pg, b = at // B, at % B
    kb = k.view(-1, Hkv, B, 16, hd)
    kc, vc = kb[pg, :, b], v[pg, :, b]                                     # [S][Hkv][16][hd], [S][Hkv][hd][16]
    kn = (kc.view(F8).float() * ratio[:, :, 0, None, None]).to(F8).view(torch.uint8)
    vn = (vc.view(F8).float() * ratio[:, :, 1, None, None]).to(F8).view(torch.uint8)
    kb[pg, :, b] = torch.where(stays[:, None, :, None], kn, kc)
    v[pg, :, b] = torch.where(stays[:, None, None, :], vn, vc)
    sc = new[blk]
    k[page, :, tok] = _cells(kx, sc[:, :, 0, None])
    v[page, :, tok // 16, :, tok % 16] = _cells(vx, sc[:, :, 1, None])
    scale[page, :, tok // 16] = sc
    return q, k.view(F8), v.view(F8), scale


def _attend(st):
    H, Hkv, hd, S, L, R = st["H"], st["Hkv"], st["hd"], st["S"], st["max_keys"], st["max_rows"]
    pg = st["pages"].long()
    k, v = st["k"][pg], st["v"][pg]                        # [S][pages][Hkv][P][hd], [S][pages][Hkv][B][hd][16]
    if st["f8"]:
        sc = st["scale"][pg]
        k = k.view(F8).float().unflatten(3, (-1, 16)) * sc[..., 0, None, None]
        k = k.flatten(3, 4)
        v = v.view(F8).float() * sc[..., 1, None, None]
    k = k.float().permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :L]
    v = v.float().permute(0, 2, 1, 3, 5, 4).flatten(2, 4)[:, :, :L]
    s, pos = _places(st)
    i = torch.arange(st["M"], device=DEV) - st["rows"].long()[s]
    q = torch.zeros(S, R, H, hd, device=DEV)
    q[s, i] = st["q"].float()
    q = q.view(S, R, Hkv, H // Hkv, hd).permute(0, 2, 3, 1, 4).reshape(S, Hkv, -1, hd)
    x = (q @ k.transpose(2, 3).contiguous()).view(S, Hkv, -1, R, L) * (1.0 / math.sqrt(hd))
    p = torch.zeros(S, R, dtype=torch.long, device=DEV)
    p[s, i] = pos
    j = torch.arange(L, device=DEV)
    seen = (j < st["n_keys"].long()[:, None])[:, None]      # [S][1][L]
    if st["causal"]:
        seen = seen & (j <= p[..., None])
    if st["window"]:
        seen = seen & (j > p[..., None] - st["window"])
    x = torch.where(seen[:, None, None], x, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    o = (e / e.sum(-1, keepdim=True)).view(S, Hkv, -1, L) @ v
    o = o.view(S, H, R, hd)[s, :, i]
    return o.to(TYPE[st["type"]])


def _score(st):
    x = st["logits"][st["rows"].long()]
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    p = e / z
    entropy = -torch.where(p > 0, p * (d - log_z), 0.0).sum(1)
    out = [d.gather(1, st["tokens"].long()) - log_z, entropy]
    if st["top"]:
        best, at = torch.sort(d, dim=1, descending=True, stable=True)
        out += [at[:, :st["top"]].int(), best[:, :st["top"]] - log_z]
    return out


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
def _plan(st):
    """The descriptors, outputs and workspace that a program keeps beside its batch."""
    pkg = os.path.join(ROOT, "diffuse-cpp_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import dfx

    L = dfx.lib()
    if st["kind"] == "score":
        n, given = st["tokens"].shape
        top = st["top"]
        out = [torch.empty(n, given, device=DEV), torch.empty(n, device=DEV)]
        if top:
            out += [torch.empty(n, top, dtype=torch.int32, device=DEV), torch.empty(n, top, device=DEV)]
        ws = torch.empty(max(1, L.dfx_token_logprobs_ws_bytes(n, st["V"], top)), dtype=torch.uint8, device=DEV)
        ptr = [t.data_ptr() for t in out] + [None] * (4 - len(out))
        args = (st["logits"].data_ptr(), st["V"], n, st["rows"].data_ptr(), n, st["V"], st["tokens"].data_ptr(), given,
                ptr[0], ptr[1], top, ptr[2], ptr[3], ws.data_ptr(), None)
        return L.dfx_token_logprobs, args, dfx.check, out, ws
    cache = dfx.PagedCache(dfx.TYPE_F8 if st["f8"] else dfx.TYPE_F16, st["page"], st["Hkv"], st["hd"], st["k"].shape[0],
                           st["k"].data_ptr(), st["v"].data_ptr(), st["scale"].data_ptr() if st["f8"] else None)
    batch = dfx.PagedBatch(st["S"], st["M"], st["rows"].data_ptr(), st["n_keys"].data_ptr(), st["pages"].data_ptr(),
                           st["pages"].shape[1], st["max_keys"])
    cr, br = ctypes.byref(cache), ctypes.byref(batch)
    typ = dfx.TYPE_F16 if st["type"] == "f16" else dfx.TYPE_F32
    y = torch.empty(st["M"], st["H"], st["hd"], dtype=TYPE[st["type"]], device=DEV)
    if st["kind"] == "append":
        out = (y, st["k"].view(F8), st["v"].view(F8), st["scale"]) if st["f8"] else (y, st["k"], st["v"])
        args = (cr, br, st["qkv"].data_ptr(), st["H"], st["tab"].data_ptr(), st["tab"].shape[0], typ, y.data_ptr(), None)
        return L.dfx_paged_append, args, dfx.check, out, (cache, batch)
    ws = torch.empty(max(1, L.dfx_paged_attention_ws_bytes(cr, br, st["H"], typ)), dtype=torch.uint8, device=DEV)
    args = (cr, br, st["q"].data_ptr(), typ, st["H"], int(st["causal"]), st["window"], y.data_ptr(), ws.data_ptr(), None)
    return L.dfx_paged_attention, args, dfx.check, y, (cache, batch, ws)


def run(state):
    if own:
        if "plan" not in state:
            state["plan"] = _plan(state)
        call, args, check, out, _ = state["plan"]
        check(call(*args), state["kind"])
        return out
    return {"append": _append, "attend": _attend, "score": _score}[state["kind"]](state)


def work(case):
    H, Hkv, hd, _, V = ARCH[case["arch"]]
    if case["kind"] == "score":
        n, out = case["n"], 8 * case["top"] + 8 * case["given"] + 8
        return {"bytes": n * (4 * V + out), "flops": 4 * n * V}
    n, keys = _lengths(case)
    M, cb = sum(n), 1 if case["cache"] == "f8" else 2
    qb = 2 if case["type"] == "f16" else 4
    if case["kind"] == "append":
        return {"bytes": M * hd * (4 * (H + 2 * Hkv) + 4 + qb * H + 2 * cb * Hkv), "flops": 3 * M * (H + Hkv) * hd}
    w = case["window"]
    pairs = read = 0
    for m, x in zip(n, keys):
        if not case["causal"]:
            pairs, read = pairs + m * x, read + x
        else:
            first = x - m                                   # position of the first row
            full = m * first + m * (m + 1) // 2
            if w:
                seen = sum(min(p + 1, w) for p in range(first, x))
                pairs, read = pairs + seen, read + min(x, m + w - 1)
            else:
                pairs, read = pairs + full, read + x
    return {"bytes": 2 * M * H * hd * qb + 2 * read * Hkv * hd * cb, "flops": 4 * pairs * H * hd}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _e4m3_scale(a):
    """2^k of a block's largest magnitude."""
    if not a > 0:
        return 2.0 ** -15
    k = math.ceil(math.log2(a) - math.log2(448.0) - 1e-12)
    return 2.0 ** min(7, max(-15, k))


def _exact_append(st):
    H, Hkv, hd, P = st["H"], st["Hkv"], st["hd"], st["page"]
    qkv, tab = st["qkv"].double(), st["tab"].double()
    rows, keys, pages = st["rows"].tolist(), st["n_keys"].tolist(), st["pages"].tolist()
    z = torch.view_as_complex(tab.contiguous())
    f8 = st["f8"]
    k = (st["k"].view(F8) if f8 else st["k"]).double()
    v = (st["v"].view(F8) if f8 else st["v"]).double()
    scale = st["scale"].double().cpu() if f8 else None
    qs = []
    for s in range(st["S"]):
        m = rows[s + 1] - rows[s]
        p0 = keys[s] - m
        x = qkv[rows[s]:rows[s + 1]]
        zz = z[p0:keys[s], None] * torch.complex(x[:, :H + Hkv, :hd // 2], x[:, :H + Hkv, hd // 2:])
        y = torch.cat([zz.real, zz.imag], -1)
        qs.append(y[:, :H])
        kx, vx = y[:, H:], x[:, H + Hkv:]
        if not f8:
            pos = torch.arange(p0, keys[s], device=DEV)
            pg = st["pages"][s].long()[pos // P]
            k[pg, :, pos % P] = kx
            v[pg, :, (pos % P) // 16, :, pos % 16] = vx
            continue
        edges = [p0] + list(range(p0 // 16 * 16 + 16, keys[s], 16)) + [keys[s]]
        top = torch.stack([torch.stack([t[a - p0:b - p0].abs().amax((0, 2)) for t in (kx, vx)], -1)
                           for a, b in zip(edges, edges[1:])]).cpu().tolist()
        fac = torch.empty(m, Hkv, 2, dtype=torch.float64)
        for i, (a, b) in enumerate(zip(edges, edges[1:])):
            page, blk = pages[s][a // P], a % P // 16
            sc = torch.tensor([[_e4m3_scale(t) for t in h] for h in top[i]], dtype=torch.float64)
            if a % 16:
                old = scale[page, :, blk].clone()
                sc = torch.maximum(sc, old)
                r = (old / sc).to(DEV)
                k[page, :, 16 * blk:16 * blk + a % 16] *= r[:, 0, None, None]
                v[page, :, blk, :, :a % 16] *= r[:, 1, None, None]
            scale[page, :, blk] = sc
            fac[a - p0:b - p0] = sc
        pos = torch.arange(p0, keys[s], device=DEV)
        pg = st["pages"][s].long()[pos // P]
        fac = fac.to(DEV)
        k[pg, :, pos % P] = kx / fac[:, :, 0, None]
        v[pg, :, (pos % P) // 16, :, pos % 16] = vx / fac[:, :, 1, None]
    q = torch.cat(qs)
    return (q, k, v, scale.to(DEV)) if f8 else (q, k, v)


def _exact_attend(st):
    H, Hkv, hd, G = st["H"], st["Hkv"], st["hd"], st["H"] // st["Hkv"]
    rows, keys = st["rows"].tolist(), st["n_keys"].tolist()
    out = torch.empty(st["M"], H, hd, dtype=torch.float64, device=DEV)
    for s in range(st["S"]):
        n = keys[s]
        pg = st["pages"][s, :-(-n // st["page"])].long()
        if st["f8"]:
            k = st["k"][pg].view(F8).double().view(len(pg), Hkv, -1, 16, hd) * st["scale"][pg][..., 0, None, None].double()
            v = st["v"][pg].view(F8).double() * st["scale"][pg][..., 1, None, None].double()
        else:
            k, v = st["k"][pg].double().view(len(pg), Hkv, -1, 16, hd), st["v"][pg].double()
        for h in range(Hkv):
            kh = k[:, h].reshape(-1, hd)[:n]
            vh = v[:, h].transpose(2, 3).reshape(-1, hd)[:n]
            for a in range(rows[s], rows[s + 1], 1024):
                b = min(a + 1024, rows[s + 1])
                qh = st["q"][a:b, h * G:h * G + G].double().reshape(-1, hd)
                x = (qh @ kh.T / math.sqrt(hd)).view(b - a, G, n)
                pos = torch.arange(n - rows[s + 1] + a, n - rows[s + 1] + b, device=DEV)[:, None, None]
                j = torch.arange(n, device=DEV)
                if st["causal"]:
                    x = x.masked_fill(j > pos, -math.inf)
                if st["window"]:
                    x = x.masked_fill(j <= pos - st["window"], -math.inf)
                out[a:b, h * G:h * G + G] = (torch.softmax(x, -1).view(-1, n) @ vh).view(b - a, G, hd)
    return out


def _exact_score(st):
    outs = []
    for a in range(0, st["rows"].numel(), 128):             # 128 rows at a time
        x = st["logits"][st["rows"][a:a + 128].long()].double()
        lp = x - torch.logsumexp(x, 1, keepdim=True)
        o = [lp.gather(1, st["tokens"][a:a + 128].long()), -(lp.exp() * lp).sum(1)]
        if st["top"]:
            best, at = torch.sort(x, dim=1, descending=True, stable=True)
            o += [at[:, :st["top"]].int(), lp.gather(1, at[:, :st["top"]])]
        outs.append(o)
    return [torch.cat(t) for t in zip(*outs)]


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "score": _exact_score}[st["kind"]](st)
