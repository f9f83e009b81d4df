"""The paged key-value cache (append, attention of single tokens, attention of packed
prompts) against plain forms in 64 bits on the same, already rounded inputs.

Tolerances.  u is the rounding to nearest of the element type, finfo.eps / 2: a
significand of b bits has steps of 2^(1-b) relative to a power of two, half of which
is 2^-b (bf16, 8 bits: 2^-8; fp16, 11: 2^-11; fp32, 24: 2^-24).  Appended vectors are rounded once from fp32: u relative,
and 16 2^-24 of the vector's largest value for the norm, the rotation's sines (their
argument is exact to 2^-25 turns) and its two products.  Attention: a score is an
fp32 sum of hd products, off by at most (hd + 4) 2^-24 sum|q k| scale = e, so each
probability by a factor e^(+-e) and the exponential's own 2^-22; numerator and
denominator give twice that, their sums of n terms n 2^-24 more; 16-bit caches round
each probability once (u; fp16's below 2^-14 by 2^-25 absolute) before the second
product; all of it times the weighted mean of |v|.  The result's rounding and the
gate's few units come on top."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _round(a, kind):
    from shiftwing_amd.paged import from_kind, to_kind
    return from_kind(to_kind(a, kind), kind)


def _tables(rng, lens, ps, extra=2):
    """Page tables over a shuffled pool; entries behind a sequence's pages name none."""
    need = [-(-n // ps) for n in lens]
    width, pages = max(need + [1]) + 1, sum(need) + extra
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, pages, width


def _cache(be, kind, nh, nkv, hd, ps, lens, rng):
    from shiftwing_amd.paged import PagedCache
    table, pages, width = _tables(rng, lens, ps)
    c = PagedCache(be, kind=kind, query_heads=nh, kv_heads=nkv, head_dim=hd, page_size=ps, pages=pages, table_pages=width,
                   sequences=len(lens))
    c.set_table(table)
    return c, table


def _fill(c, table, lens, rng, kind, junk=np.nan):
    """Random keys and values in every position a sequence has, `junk` elsewhere."""
    pages, ps, nkv, hd = c.shape
    K, V = (np.full(c.shape, junk, np.float32) for _ in range(2))
    for s, n in enumerate(lens):
        for p in range(0, n, ps):
            m = min(ps, n - p)
            if 0 <= table[s, p // ps] < pages:
                K[table[s, p // ps], :m] = rng.standard_normal((m, nkv, hd))
                V[table[s, p // ps], :m] = rng.standard_normal((m, nkv, hd))
    K, V = _round(K, kind), _round(V, kind)
    c.write(K, V)
    return K, V


def _want(q, K, V, table, seq, visible, scale, gate, kind):
    """One row's attention in 64 bits and its tolerance, per head and dim."""
    pages, ps, nkv, hd = K.shape
    nh = q.shape[0]
    pos = np.array([p for p in range(visible) if 0 <= table[seq, p // ps] < pages], int)
    if len(pos) == 0:
        return np.zeros((nh, hd)), np.zeros((nh, hd))
    k, v = (X[table[seq, pos // ps], pos % ps].astype(np.float64) for X in (K, V))
    kvh = np.arange(nh) * nkv // nh
    s = np.einsum("hd,phd->hp", q.astype(np.float64), k[:, kvh]) * scale
    mass = np.einsum("hd,phd->hp", np.abs(q).astype(np.float64), np.abs(k[:, kvh])).max(1) * abs(scale)
    p = np.exp(s - s.max(1, keepdims=True))
    l = p.sum(1)
    o = np.einsum("hp,phd->hd", p, v[:, kvh]) / l[:, None]
    w = np.einsum("hp,phd->hd", p, np.abs(v[:, kvh])) / l[:, None]
    n, u = len(pos), U[kind]
    e = (hd + 4) * 2.0 ** -24 * mass + 2.0 ** -22 + 2.0 ** -24 * np.abs(s).max(1)
    tol = (2 * e + (n + 8) * 2.0 ** -24 + (u if kind != "f32" else 0))[:, None] * w
    if kind == "f16":
        tol = tol + n * 2.0 ** -25 * np.abs(v[:, kvh]).max(0)
    if gate is not None:
        g = 1 / (1 + np.exp(-gate.astype(np.float64)))
        o, tol = o * g, tol * g + 2.0 ** -20 * np.abs(o * g)
    return o, tol + u * (np.abs(o) + tol) + (2.0 ** -25 if kind == "f16" else 1e-37)


def _check(got, want, tol, what):
    assert np.all(np.isfinite(got)), what
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - want) / tol):.3g} x the tolerance"


# ---- append ---------------------------------------------------------------------------------------------


def _turned(x, norm, pos, rd, theta, eps, hd):
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 + norm.astype(np.float64))
    h = rd // 2
    if h:
        ang = pos[:, None, None] * float(np.float32(theta)) ** (-2.0 * np.arange(h) / rd)
        a, b = x[..., :h].copy(), x[..., h:rd].copy()
        x = x.copy()
        x[..., :h], x[..., h:rd] = a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)
    return x


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,rd,norms,start,length", [
    (4, 2, 64, 16, 64, True, [0, 1], [1]),                                # the first token of a sequence
    (6, 2, 64, 5, 24, True, [2, 9, 9, 10, 47], [7, 0, 90001, 38]),        # a gap in front, an empty one, a far position
    (2, 2, 128, 1, 2, False, [0, 3, 4], [300, 1000000]),                  # one position a page, one pair
    (32, 2, 256, 16, 64, True, [0, 1, 2, 3], [17, 16, 400]),              # the large decoder's heads
    (5, 1, 256, 48, 0, True, [0, 20, 131], [20, 4000]),                   # no rotation
    (3, 3, 128, 64, 128, False, [1, 130], [129]),
])
def test_append(be, kind, nh, nkv, hd, ps, rd, norms, start, length):
    from shiftwing_amd.paged import PagedCache
    rng = np.random.default_rng(71)
    new = np.diff(start)
    # pages of the last positions only; the rest of the table names none
    first = [(n - m) // ps for n, m in zip(length, new)]
    used = [range(f, -(-n // ps)) if m else range(0) for f, n, m in zip(first, length, new)]
    pages, width = sum(len(u) for u in used) + 2, max(-(-n // ps) for n in length) + 1
    ids, table, at = rng.permutation(pages).astype(np.int32), np.full((len(length), width), -1, np.int32), 0
    for s, u in enumerate(used):
        table[s, list(u)] = ids[at:at + len(u)]
        at += len(u)
    c = PagedCache(be, kind=kind, query_heads=nh, kv_heads=nkv, head_dim=hd, page_size=ps, pages=pages, table_pages=width,
                   sequences=len(length))
    c.set_table(table)
    rows = start[-1] + 3  # rows behind the last sequence
    q, k, v = (_round(rng.standard_normal((rows, h, hd)) * 3, kind) for h in (nh, nkv, nkv))
    w = [(rng.standard_normal(hd) * 0.1).astype(np.float32) if norms else None for _ in range(2)]
    K0, V0 = (_round(rng.standard_normal(c.shape), kind) for _ in range(2))
    c.write(K0, V0)
    print(f"[append] {kind} heads {nh}/{nkv} x {hd} page {ps} rotary {rd} rows {start}", flush=True)
    theta = 1e7 if rd == 64 else 1e4
    got = c.append(start, length, k, v, q, q_norm=w[0], k_norm=w[1], rotary_dim=rd, theta=theta)
    gk, gv = c.read()
    wq, wk, wv = np.zeros((rows, nh, hd)), K0.astype(np.float64), V0.astype(np.float64)
    tol_k = np.zeros(c.shape)
    tol_q = np.zeros((rows, nh, hd))
    for s, m in enumerate(new):
        r = np.arange(start[s], start[s + 1])
        if len(r) == 0:
            continue
        pos = np.arange(length[s] - m, length[s])
        cells = table[s, pos // ps], pos % ps
        for x, norm, out, tol, where in ((q, w[0], wq, tol_q, r), (k, w[1], wk, tol_k, cells)):
            y = _turned(x[r], norm, pos.astype(np.float64), rd, theta, 1e-6, hd)
            out[where] = y
            # the rotation's frequencies: (i + 3) 2^-53 relative, times the angle
            far = 2.0 ** -45 * pos[:, None, None]
            tol[where] = U[kind] * np.abs(y) + (16 * 2.0 ** -24 + far) * np.abs(y).max(-1, keepdims=True) + 2.0 ** -25
        wv[cells] = v[r]
    assert np.array_equal(gv, wv), "values"
    untouched = tol_k == 0
    assert np.array_equal(gk[untouched], K0[untouched]), "cells of no row"
    _check(gk[~untouched], wk[~untouched], tol_k[~untouched], "keys")
    outside = np.r_[np.arange(start[0]), np.arange(start[-1], rows)]
    assert np.all(got[outside] == 0), "rows of no sequence"
    inside = np.arange(start[0], start[-1])
    _check(got[inside], wq[inside], tol_q[inside], "queries")


def test_append_leaves_out_absent_pages_and_takes_keys_alone(be):
    from shiftwing_amd.paged import PagedCache
    rng = np.random.default_rng(72)
    c = PagedCache(be, kind="bf16", query_heads=4, kv_heads=2, head_dim=64, page_size=4, pages=3, table_pages=4, sequences=1)
    c.set_table(np.array([[2, 3, -1, 0]], np.int32))  # 3 and -1 name no page
    K0 = _round(rng.standard_normal(c.shape), "bf16")
    c.write(K0, K0)
    k, v = (_round(rng.standard_normal((14, 2, 64)), "bf16") for _ in range(2))
    assert c.append([0, 14], [14], k, v) is None
    gk, gv = c.read()
    for got, x in ((gk, k), (gv, v)):
        assert np.array_equal(got[2], x[:4]) and np.array_equal(got[0, :2], x[12:14])
        assert np.array_equal(got[1], K0[1]) and np.array_equal(got[0, 2:], K0[0, 2:])


def test_append_strided_rows_and_interleaved_pools(be):
    """Query | gate rows of a fused projection, keys and values in one row, both pools in one allocation."""
    import ctypes as C

    from shiftwing_amd.abi import ColiPaged
    rng = np.random.default_rng(73)
    nh, nkv, hd, ps, T, pages = 4, 2, 64, 8, 13, 3
    page = ps * nkv * hd
    c = ColiPaged(0, nh, nkv, hd, ps, pages, 2, 2 * page)
    pool = be.upload(np.zeros((pages, 2, ps, nkv, hd), np.float32))
    table = be.upload(np.array([[2, 0]], np.int32))
    qg = rng.standard_normal((T, nh, 2, hd)).astype(np.float32)
    kv = rng.standard_normal((T, 2 * nkv * hd + 8)).astype(np.float32)
    dq, dkv, out = be.upload(qg), be.upload(kv), be.alloc(T * nh * hd * 4)
    start, length = (C.c_int * 2)(0, T), (C.c_int * 1)(T)
    be.check(be.lib.coli_cuda_paged_append(
        be.ctx, C.byref(c), pool.p, C.c_void_p(pool.ptr + page * 4), table.p, start, length, 1, out.p, dq.p, nh * 2 * hd, 2 * hd,
        dkv.p, kv.shape[1], C.c_void_p(dkv.ptr + nkv * hd * 4), kv.shape[1], None, None, 0.0, 0, 0.0), "append")
    got = be.download(pool, (pages, 2, ps, nkv, hd), np.float32)
    rows = np.concatenate([got[2], got[0]], 1)[:, :T]  # [k | v][position]
    assert np.array_equal(rows.reshape(2, T, -1).transpose(1, 0, 2).reshape(T, -1), kv[:, :-8])
    assert np.all(got[1] == 0) and np.all(got[0][:, T - ps:] == 0)
    assert np.array_equal(be.download(out, (T, nh, hd), np.float32), qg[:, :, 0])


# ---- attention of single tokens -----------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,lens,gated", [
    (2, 2, 64, 16, [1], False),
    (8, 2, 64, 16, [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 700], True),
    (16, 2, 256, 16, [1, 300, 0, 64], True),
    (32, 2, 256, 64, [1025], False),
    (12, 3, 128, 48, [5, 191, 193, 2000], False),
    (40, 2, 128, 32, [140, 33], True),                  # 20 query heads a kv head: two groups
    (7, 1, 64, 1, [3, 100], True),                      # one position a page
    (3, 1, 128, 7, [130, 29, 7], False),                # pages that end inside every run
    (6, 2, 256, 24, [555], True),
])
def test_decode(be, kind, nh, nkv, hd, ps, lens, gated):
    rng = np.random.default_rng(81)
    c, table = _cache(be, kind, nh, nkv, hd, ps, lens, rng)
    K, V = _fill(c, table, lens, rng, kind)
    q = _round(rng.standard_normal((len(lens), nh, hd)) * 2, kind)
    gate = _round(rng.standard_normal((len(lens), nh, hd)) * 3, kind) if gated else None
    scale = float(np.float32(hd ** -0.5))
    print(f"[decode] {kind} heads {nh}/{nkv} x {hd} page {ps} lengths {lens}", flush=True)
    got = c.decode(q, lens, scale, gate)
    for s, n in enumerate(lens):
        want, tol = _want(q[s], K, V, table, s, n, scale, gate[s] if gated else None, kind)
        _check(got[s], want, tol, f"sequence {s} of length {n}")


def test_decode_leaves_out_absent_pages(be):
    for ps in (16, 6):
        rng = np.random.default_rng(82)
        lens = [100, 40, 33]
        c, table = _cache(be, "bf16", 4, 2, 64, ps, lens, rng)
        table[0, 2], table[0, 5], table[1, 0] = -1, c.shape[0], 1 << 30
        table[2, :] = -5  # nothing left
        c.set_table(table)
        K, V = _fill(c, table, lens, rng, "bf16")
        q = _round(rng.standard_normal((3, 4, 64)), "bf16")
        got = c.decode(q, lens, 0.125)
        for s, n in enumerate(lens):
            want, tol = _want(q[s], K, V, table, s, n, 0.125, None, "bf16")
            _check(got[s], want, tol, f"page {ps} sequence {s}")
        assert np.all(got[2] == 0)


def test_decode_more_sequences_than_a_launch(be):
    rng = np.random.default_rng(83)
    lens = [int(n) for n in rng.integers(0, 90, 300)]
    c, table = _cache(be, "f16", 2, 1, 64, 16, lens, rng)
    K, V = _fill(c, table, lens, rng, "f16")
    q, gate = (_round(rng.standard_normal((300, 2, 64)), "f16") for _ in range(2))
    got = c.decode(q, lens, 0.125, gate)
    for s, n in enumerate(lens):
        want, tol = _want(q[s], K, V, table, s, n, 0.125, gate[s], "f16")
        _check(got[s], want, tol, f"sequence {s}")


def test_decode_extreme_scores(be):
    """Scores of +-3e4 (the rest of the softmax vanishes) and keys of minus infinity behind finite ones."""
    rng = np.random.default_rng(84)
    lens = [200]
    c, table = _cache(be, "f32", 2, 2, 64, 16, lens, rng)
    K, V = _fill(c, table, lens, rng, "f32")
    q = np.zeros((1, 2, 64), np.float32)
    q[:, :, 0] = 1e3
    pos = np.arange(200)
    K[table[0, pos // 16], pos % 16, :, 0] = np.where(pos == 77, 30.0, -30.0)[:, None]
    K[table[0, 150 // 16], 150 % 16, :, 0] = -np.inf
    c.write(K, V)
    got = c.decode(q, lens, 1.0)
    assert np.allclose(got[0], V[table[0, 77 // 16], 77 % 16], rtol=2.0 ** -22, atol=0)


# ---- attention of packed prompts -------------------------------------------------------------------------


PROMPTS = [
    (2, 2, 64, 16, [0, 1], [1], False),                                         # one token
    (4, 2, 64, 16, [0, 31, 31, 95, 96, 161], [31, 9, 64, 1, 65], True),          # tile edges, an empty sequence
    (16, 2, 256, 16, [3, 40, 57, 58], [37, 300, 1], True),                       # a gap in front, a cached prefix
    (6, 2, 128, 24, [0, 129, 200], [129, 71], False),                            # three heads a kv head
    (3, 3, 128, 5, [0, 65, 130], [200, 65], True),                               # pages that end inside tiles
    (8, 1, 64, 64, [0, 7, 11], [3000, 2500], True),                              # few rows behind long caches: splits
    (20, 1, 128, 16, [0, 33], [4000], False),
    (2, 1, 256, 32, [0, 190], [190], False),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,start,lens,gated", PROMPTS)
def test_prompt(be, kind, nh, nkv, hd, ps, start, lens, gated):
    rng = np.random.default_rng(91)
    c, table = _cache(be, kind, nh, nkv, hd, ps, lens, rng)
    K, V = _fill(c, table, lens, rng, kind)
    rows = start[-1] + 2
    q = _round(rng.standard_normal((rows, nh, hd)) * 2, kind)
    gate = _round(rng.standard_normal((rows, nh, hd)) * 3, kind) if gated else None
    scale = float(np.float32(hd ** -0.5))
    print(f"[prompt] {kind} heads {nh}/{nkv} x {hd} page {ps} rows {start} lengths {lens}", flush=True)
    got = c.prompt(q, start, lens, scale, gate)
    seen = np.zeros(rows, bool)
    for s, n in enumerate(lens):
        for r in range(start[s], start[s + 1]):
            seen[r] = True
            want, tol = _want(q[r], K, V, table, s, n - (start[s + 1] - r) + 1, scale, gate[r] if gated else None, kind)
            _check(got[r], want, tol, f"row {r} of sequence {s}")
    assert np.all(got[~seen] == 0), "rows of no sequence"


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("ps", [16, 6])
def test_prompt_leaves_out_absent_pages(be, kind, ps):
    rng = np.random.default_rng(92)
    start, lens = [0, 150, 190, 200], [150, 700, 10]
    c, table = _cache(be, kind, 4, 2, 64, ps, lens, rng)
    table[0, 0], table[0, 5], table[1, 20], table[1, 3], table[1, 7] = -1, c.shape[0], 1 << 30, -7, -1
    table[2, :] = -5
    c.set_table(table)
    K, V = _fill(c, table, lens, rng, kind)
    q = _round(rng.standard_normal((200, 4, 64)), kind)
    got = c.prompt(q, start, lens, 0.125)
    for s, n in enumerate(lens):
        for r in range(start[s], start[s + 1]):
            want, tol = _want(q[r], K, V, table, s, n - (start[s + 1] - r) + 1, 0.125, None, kind)
            _check(got[r], want, np.maximum(tol, 1e-37), f"row {r} of sequence {s}")


def test_prompt_more_sequences_than_a_launch(be):
    rng = np.random.default_rng(93)
    new = rng.integers(0, 4, 290)
    start = [0] + [int(x) for x in np.cumsum(new)]
    lens = [int(n + b) for n, b in zip(new, rng.integers(0, 60, 290))]
    c, table = _cache(be, "bf16", 4, 2, 64, 16, lens, rng)
    K, V = _fill(c, table, lens, rng, "bf16")
    q = _round(rng.standard_normal((start[-1], 4, 64)), "bf16")
    got = c.prompt(q, start, lens, 0.125)
    for s, n in enumerate(lens):
        for r in range(start[s], start[s + 1]):
            want, tol = _want(q[r], K, V, table, s, n - (start[s + 1] - r) + 1, 0.125, None, "bf16")
            _check(got[r], want, tol, f"row {r} of sequence {s}")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,ps", [(64, 16), (64, 5), (128, 16), (128, 5)])
def test_prompt_more_tiles_than_compute_units(be, kind, hd, ps):
    """96 kv heads x 4 tiles of rows, which no smaller case has: every ninth row is looked at, and the last."""
    rng = np.random.default_rng(96)
    nh, nkv, start, lens = 192, 96, [0, 100, 161], [100, 130]
    c, table = _cache(be, kind, nh, nkv, hd, ps, lens, rng)
    K, V = _fill(c, table, lens, rng, kind)
    V[table[1, 125 // ps], 125 % ps, :, 3] = np.nan  # seen by the last rows alone
    clean = np.where(np.isnan(V), 0, V)
    c.write(K, V)
    q, gate = (_round(rng.standard_normal((161, nh, hd)), kind) for _ in range(2))
    print(f"[prompt] {kind} heads {nh}/{nkv} x {hd} page {ps} rows {start}", flush=True)
    got = c.prompt(q, start, lens, 0.11, gate)
    for s, n in enumerate(lens):
        for r in [*range(start[s], start[s + 1], 9), start[s + 1] - 1]:
            sees = n - (start[s + 1] - r) + 1
            want, tol = _want(q[r], K, clean, table, s, sees, float(np.float32(0.11)), gate[r], kind)
            dims = [d for d in range(hd) if d != 3 or s == 0 or sees <= 125]
            assert len(dims) == hd or np.all(np.isnan(got[r, :, 3]))
            _check(got[r][:, dims], want[:, dims], tol[:, dims], f"row {r} of sequence {s}")


# ---- values that are not finite ---------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("call", ["decode", "prompt"])
def test_a_nan_of_weight_zero(be, kind, call):
    """A visible NaN (a key's, or a value's) among scores 400 below the largest: its weight is zero in fp32, in its
    split and as its split's in the join, and zero times NaN is NaN."""
    for what in ("key", "value"):
        rng = np.random.default_rng(94)
        lens, rows = [5000], 1 if call == "decode" else 3
        c, table = _cache(be, kind, 2, 1, 64, 16, lens, rng)
        K, V = _fill(c, table, lens, rng, kind)
        q = np.zeros((rows, 2, 64), np.float32)
        q[:, :, 0] = 8
        pos = np.arange(5000)
        K[table[0, pos // 16], pos % 16, :, 0] = np.where(pos < 2500, -25, 25)[:, None]
        if what == "key":
            K[table[0, 30 // 16], 30 % 16, 0, 5] = np.nan
        else:
            V[table[0, 30 // 16], 30 % 16, 0, 5] = np.nan
        c.write(K, V)
        got = c.decode(q, lens, 1.0) if call == "decode" else c.prompt(q, [0, rows], lens, 1.0)
        hit = np.isnan(got)
        assert np.all(hit if what == "key" else hit[:, :, 5] & (hit.sum(-1) == 1)), what


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh,nkv,hd,ps,start,lens,at", [
    (2, 2, 64, 16, [0, 70], [70], [69]),                    # the last row's own
    (4, 2, 128, 16, [0, 150, 180], [150, 400], [77, 395]),  # within a prompt, and behind a cached prefix
    (16, 2, 256, 16, [0, 45], [45], [20]),
    (6, 2, 256, 6, [0, 90], [130], [100]),                  # pages that end inside tiles
    (8, 1, 64, 64, [0, 7], [3000], [2996]),                 # splits
    (3, 1, 128, 16, [0, 40], [50], [3]),                    # seen by every row
])
def test_prompt_values_that_are_not_seen(be, kind, nh, nkv, hd, ps, start, lens, at):
    """A NaN among the values of one position, an infinity beside it: rows before it are as they would be, the others
    have it in that dim alone."""
    rng = np.random.default_rng(95)
    c, table = _cache(be, kind, nh, nkv, hd, ps, lens, rng)
    K, V = _fill(c, table, lens, rng, kind)
    clean = V.copy()
    for s, p in enumerate(at):
        V[table[s, p // ps], p % ps, :, 3], V[table[s, p // ps], p % ps, :, hd - 2] = np.nan, -np.inf
    c.write(K, V)
    q = _round(rng.standard_normal((start[-1], nh, hd)), kind)
    for scale in (hd ** -0.5, -0.03):
        got = c.prompt(q, start, lens, scale)
        for s, n in enumerate(lens):
            for r in range(start[s], start[s + 1]):
                sees = n - (start[s + 1] - r) + 1
                want, tol = _want(q[r], K, clean, table, s, sees, float(np.float32(scale)), None, kind)
                if s < len(at) and sees > at[s]:
                    assert np.all(np.isnan(got[r, :, 3])) and np.all(got[r, :, hd - 2] == -np.inf)
                    rest = [d for d in range(hd) if d not in (3, hd - 2)]
                else:
                    rest = list(range(hd))
                _check(got[r][:, rest], want[:, rest], tol[:, rest], f"row {r} of sequence {s}, scale {scale}")


# ---- together ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompts_then_tokens(be, kind):
    """Prompts are appended and attended, then a prompt chunk and two turns of single tokens follow in the same
    cache: the rows' outputs equal attention over the whole history of rotated, rounded keys."""
    rng = np.random.default_rng(95)
    nh, nkv, hd, ps, rd = 8, 2, 128, 16, 64
    final = [70, 21, 48]
    c, table = _cache(be, kind, nh, nkv, hd, ps, final, rng)
    hist = [[], [], []]
    have = [0, 0, 0]
    w = [(rng.standard_normal(hd) * 0.1).astype(np.float32) for _ in range(2)]
    scale = float(np.float32(hd ** -0.5))
    for new in ([40, 19, 0], [28, 0, 46], [1, 1, 1], [1, 1, 1]):
        start = np.r_[0, np.cumsum(new)].tolist()
        have = [a + b for a, b in zip(have, new)]
        q, k, v = (_round(rng.standard_normal((start[-1], h, hd)), kind) for h in (nh, nkv, nkv))
        gate = _round(rng.standard_normal((start[-1], nh, hd)), kind)
        rq = c.append(start, have, k, v, q, q_norm=w[0], k_norm=w[1], rotary_dim=rd, theta=1e7)
        got = c.decode(rq, have, scale, gate) if new == [1, 1, 1] else c.prompt(rq, start, have, scale, gate)
        K, V = c.read()
        for s in range(3):
            pos = np.arange(have[s] - new[s], have[s])
            if len(pos):
                y = _turned(k[start[s]:start[s + 1]], w[1], pos.astype(np.float64), rd, 1e7, 1e-6, hd)
                _check(K[table[s, pos // ps], pos % ps], y,
                       U[kind] * np.abs(y) + 2.0 ** -20 * np.abs(y).max(-1, keepdims=True) + 1e-9, "keys")
            for r in range(start[s], start[s + 1]):
                want, tol = _want(rq[r], K, V, table, s, have[s] - (start[s + 1] - r) + 1, scale, gate[r], kind)
                _check(got[r], want, tol, f"row {r}")
    assert have == final


# ---- calls that the wrapper does not make --------------------------------------------------------------------


class Raw:
    """The C calls on device buffers of one's own, on any context."""

    def __init__(self, be, kind, nh, nkv, hd, ps, pages, width, stride=0):
        import ctypes as C

        from shiftwing_amd.abi import ColiPaged
        from shiftwing_amd.paged import KINDS
        self.C, self.be, self.kind, self.nh, self.hd = C, be, kind, nh, hd
        self.c = ColiPaged(KINDS[kind], nh, nkv, hd, ps, pages, width, stride or ps * nkv * hd)

    def ints(self, a):
        return (self.C.c_int * len(a))(*a)

    def call(self, name, *args):
        self.be.check(getattr(self.be.lib, name)(self.be.ctx, self.C.byref(self.c), *args), name)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_gates_behind_the_queries(be, kind):
    """Gates as the projection leaves them, behind each head's query, in rows wider than that; an output that is
    not clear, whose rows of no sequence stay; scales of zero and below."""
    from shiftwing_amd.paged import from_kind, to_kind, word
    rng = np.random.default_rng(101)
    nh, nkv, hd, ps, start, lens = 6, 2, 128, 16, [1, 40, 43], [39, 900]
    c, table = _cache(be, kind, nh, nkv, hd, ps, lens, rng)
    K, V = _fill(c, table, lens, rng, kind)
    r = Raw(be, kind, nh, nkv, hd, ps, c.shape[0], table.shape[1])
    rows, wide, size = 45, nh * 2 * hd + 20, np.dtype(word(kind)).itemsize
    mix = _round(rng.standard_normal((rows, wide)) * 2, kind)
    gate = mix[:, :nh * 2 * hd].reshape(rows, nh, 2, hd)[:, :, 1]
    q = _round(rng.standard_normal((rows, nh, hd)), kind)
    dmix, dq = be.upload(to_kind(mix, kind)), be.upload(to_kind(q, kind))
    for scale in (0.0, -0.05):
        for name, args, n in (("prompt", (r.ints(start), r.ints(lens), 2), rows), ("decode", (r.ints(lens), 2), 2)):
            out = be.upload(to_kind(np.full((rows, nh, hd), 7.0), kind))
            r.call("coli_cuda_paged_" + name, out.p, dq.p, r.C.c_void_p(dmix.ptr + hd * size), wide, 2 * hd, c.k_pool.p,
                   c.v_pool.p, c.table.p, *args, scale)
            got = from_kind(be.download(out, (rows, nh, hd), word(kind)), kind)
            seen = np.zeros(rows, bool)
            for s, length in enumerate(lens):
                mine = range(start[s], start[s + 1]) if name == "prompt" else [s]
                for i, row in enumerate(mine):
                    seen[row] = True
                    sees = length - len(mine) + i + 1
                    want, tol = _want(q[row], K, V, table, s, sees, float(np.float32(scale)), gate[row], kind)
                    _check(got[row], want, tol, f"{name} row {row} scale {scale}")
            assert np.all(got[~seen] == 7.0)


def test_a_pool_beyond_32_bits(be):
    """Pages 2^30 elements apart: the last one begins 2^32 elements (8 GiB) behind the first."""
    from shiftwing_amd.paged import from_kind, to_kind
    rng = np.random.default_rng(102)
    nh, nkv, hd, ps, T = 4, 2, 64, 16, 40
    row, far = nkv * hd, 1 << 30
    r = Raw(be, "bf16", nh, nkv, hd, ps, 5, 3, far)
    pool = be.alloc((4 * far + 2 * ps * row) * 2)
    v_pool = r.C.c_void_p(pool.ptr + ps * row * 2)  # behind each page's keys
    table = be.upload(np.array([[4, 0, 3]], np.int32))
    k, v = (_round(rng.standard_normal((T, nkv, hd)), "bf16") for _ in range(2))
    q = _round(rng.standard_normal((T, nh, hd)), "bf16")
    dk, dv, dq = (be.upload(to_kind(x, "bf16")) for x in (k, v, q))
    r.call("coli_cuda_paged_append", pool.p, v_pool, table.p, r.ints([0, T]), r.ints([T]), 1, None, None, 0, 0, dk.p, row, dv.p,
           row, None, None, 0.0, 0, 0.0)
    out = be.alloc(T * nh * hd * 2)
    r.call("coli_cuda_paged_prompt", out.p, dq.p, None, 0, 0, pool.p, v_pool, table.p, r.ints([0, T]), r.ints([T]), 1, 0.125)
    prompt = from_kind(be.download(out, (T, nh, hd), np.uint16), "bf16")
    r.call("coli_cuda_paged_decode", out.p, dq.p, None, 0, 0, pool.p, v_pool, table.p, r.ints([T]), 1, 0.125)
    token = from_kind(be.download(out, (1, nh, hd), np.uint16), "bf16")
    flat = np.zeros((3, ps, nkv, hd), np.float32), np.zeros((3, ps, nkv, hd), np.float32)
    for x, y in zip(flat, (k, v)):
        x.reshape(-1, nkv, hd)[:T] = y
    plain = np.arange(3)[None]
    for i in range(T):
        want, tol = _want(q[i], *flat, plain, 0, i + 1, 0.125, None, "bf16")
        _check(prompt[i], want, tol, f"row {i}")
    want, tol = _want(q[0], *flat, plain, 0, T, 0.125, None, "bf16")
    _check(token[0], want, tol, "the token")


def test_two_contexts_and_the_same_call_again(be):
    """Calls queued on two contexts in turn, with different sizes of workspace, repeated: the same bits each time."""
    from shiftwing_amd import Backend
    rng = np.random.default_rng(103)
    other = Backend(0)
    cases = []
    for b, lens in ((be, [3000, 17]), (other, [901, 64, 1, 2500])):
        c, table = _cache(b, "bf16", 8, 2, 128, 16, lens, rng)
        _fill(c, table, lens, rng, "bf16")
        r = Raw(b, "bf16", 8, 2, 128, 16, c.shape[0], table.shape[1])
        q = b.upload(rng.integers(0, 2, (len(lens), 8, 128)).astype(np.uint16) + 0x3F80)
        outs = [b.alloc(len(lens) * 8 * 128 * 2) for _ in range(6)]
        cases.append((b, c, r, q, outs, lens))
    for turn in range(6):
        for b, c, r, q, outs, lens in cases:
            n = len(lens)
            extra = (r.ints(list(range(n + 1))),) if turn % 2 else ()
            r.call("coli_cuda_paged_" + ("prompt" if turn % 2 else "decode"), outs[turn].p, q.p, None, 0, 0, c.k_pool.p,
                   c.v_pool.p, c.table.p, *extra, r.ints(lens), n, 0.09)
    for b, c, r, q, outs, lens in cases:
        got = [b.download(o, (len(lens) * 8 * 128,), np.uint16) for o in outs]
        for turn in range(2, 6):
            assert np.array_equal(got[turn], got[turn % 2]), f"turn {turn}"
        assert np.any(got[0] != 0)
