"""fp16 attention: scores as large as fp16 vectors make them, and weights far below the
largest one, of very many positions: a key of
much higher score whose values are zero (a sink), and behind it a long tail of equal
scores that makes up the whole output.

Tolerances, relative to the output, which is the tail's weight times a mean value: the
scores' difference is gap, one fp32 product scaled by log2(e) rounded, which moves a
weight by e^(+-e), e = 3 2^-24 gap, its exponential by 2^-22, numerator and sum of n
terms by n 2^-24 each; a weight is rounded to fp16 (2^-11).  A weight below fp16's
normal numbers loses half of its last place: weights are held 2^15 (single tokens) or
2^13 (prompts) above one, so 2^-25 is 2^-40 or 2^-38 of the largest weight, n times that
of the largest value.  The output's rounding is 2^-11, below 2^-14 2^-25 absolute."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

N, PS = 100_000, 16


class Sink:
    """A pool of two pages for any number of sequences: one that holds the sink, one that every other table entry
    names."""

    def __init__(self, be, nkv, hd, sequences, length, at, gap):
        from shiftwing_amd.paged import PagedCache
        rng = np.random.default_rng(111)
        width = -(-length // PS)
        self.c = PagedCache(be, kind="f16", query_heads=nkv, kv_heads=nkv, head_dim=hd, page_size=PS, pages=2,
                            table_pages=width, sequences=sequences)
        self.table = np.zeros((sequences, width), np.int32)
        self.table[:, at // PS] = 1
        self.c.set_table(self.table)
        K = np.zeros((2, PS, nkv, hd), np.float32)
        K[1, at % PS, :, 0] = gap / 8
        V = np.repeat(rng.uniform(0.5, 1.5, (1, PS, 1, hd)), 2, 0).astype(np.float16).astype(np.float32)
        V = np.tile(V, (1, 1, nkv, 1))
        V[1, at % PS] = 0
        self.c.write(K, V)
        self.at, self.gap, self.V = at, gap, V[:, :, 0].astype(np.float64)

    def queries(self, rows):
        q = np.zeros((rows, self.c.nh, self.c.hd), np.float32)
        q[..., 0] = 8
        return q

    def want(self, length, least):
        """The output of a row that sees `length` positions, and its tolerance; `least`: the largest weight's
        multiple at which fp16 ends."""
        p = np.arange(length)
        times = np.zeros((2, PS))
        np.add.at(times, (self.table[0, p // PS], p % PS), 1)
        w = times * np.exp(-float(self.gap))
        if length > self.at:
            w[1, self.at % PS] = 1.0
        else:
            w /= np.exp(-float(self.gap))
        o = (w[..., None] * self.V).sum((0, 1)) / w.sum()
        tol = o * (2 * (3 * 2.0 ** -24 * self.gap + 2.0 ** -22 + (length + 8) * 2.0 ** -24) + 2.0 ** -11)
        tol = tol + length * least * 1.5 / max(w.sum(), 1)
        return o, tol + 2.0 ** -11 * (o + tol) + 2.0 ** -25


def _check(got, want, tol, what):
    got = got.astype(np.float64)
    assert np.all(np.isfinite(got)), what
    off = np.abs(got - want) / tol
    assert np.all(off <= 1), f"{what}: {np.max(off):.3g} x the tolerance, {got.flat[0]:.6g} for {want.flat[0]:.6g}"


@pytest.mark.parametrize("gap", [10.0, 16.0, 17.5, 20.0])
@pytest.mark.parametrize("nkv,hd,sequences,at", [
    (1, 64, 1, 0),          # in splits
    (4, 256, 128, 0),       # one split a sequence: 512 workgroups of a compute unit each
    (4, 256, 128, 70_003),
    (25, 64, 128, 3),
])
def test_decode(be, nkv, hd, sequences, at, gap):
    print(f"[decode] {sequences} sequences x {nkv} heads of {hd}, the sink at {at}, gap {gap}", flush=True)
    s = Sink(be, nkv, hd, sequences, N, at, gap)
    got = s.c.decode(s.queries(sequences), [N] * sequences, 1.0)
    want, tol = s.want(N, 2.0 ** -40)
    _check(got, np.broadcast_to(want, got.shape), tol, f"gap {gap}")


@pytest.mark.parametrize("gap", [10.0, 16.0, 17.5, 20.0])
@pytest.mark.parametrize("nkv,hd,at", [
    (1, 64, 0),             # in splits
    (130, 64, 0),           # 16 rows a wave
    (300, 128, 0),          # 32 rows a wave
    (300, 64, 70_003),
    (130, 256, 0),
])
def test_prompt(be, nkv, hd, at, gap):
    print(f"[prompt] {nkv} heads of {hd}, the sink at {at}, gap {gap}", flush=True)
    s = Sink(be, nkv, hd, 1, N, at, gap)
    got = s.c.prompt(s.queries(3), [0, 3], [N], 1.0)
    for i in range(3):
        want, tol = s.want(N - 2 + i, 2.0 ** -38)
        _check(got[i], want[None], tol, f"row {i}, gap {gap}")


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("call", ["decode", "prompt"])
@pytest.mark.parametrize("nkv,hd", [(1, 64), (130, 64), (300, 128), (130, 256)])
def test_scores_whose_last_place_is_large(be, call, nkv, hd, sign):
    """Scores of about 2^27.5 in powers of two, 16 and 32 apart from tile to tile, where fp32 numbers lie 16 apart: no
    reference beside the largest score is exact there.  The output is a mean of the values all the same."""
    from shiftwing_amd.paged import PagedCache
    rng = np.random.default_rng(112)
    pages, per = 40, 64
    n = pages * per
    c = PagedCache(be, kind="f16", query_heads=nkv, kv_heads=nkv, head_dim=hd, page_size=per, pages=pages, table_pages=pages,
                   sequences=1)
    c.set_table(np.arange(pages)[None])
    K = np.zeros((pages, per, nkv, hd), np.float32)
    K[..., 0] = 8192.0 * sign
    K[..., 1] = 16.0 * np.arange(pages)[:, None, None]
    V = np.tile(rng.uniform(0.5, 1.5, (pages, per, 1, hd)), (1, 1, nkv, 1))
    c.write(K, V)
    rows = 1 if call == "decode" else 5
    q = np.zeros((rows, nkv, hd), np.float32)
    q[..., 0], q[..., 1] = 16384.0, 1.0
    print(f"[{call}] {nkv} heads of {hd}, scores of {'-' if sign < 0 else ''}2^27", flush=True)
    got = c.decode(q, [n], 1.0) if call == "decode" else c.prompt(q, [0, rows], [n], 1.0)
    # weights and their sum are rounded apart: 2^-11 and n 2^-24 a side, and the output
    slack = 2 * 2.0 ** -11 + 2 * n * 2.0 ** -24
    assert np.all((got >= 0.5 * (1 - slack)) & (got <= 1.5 * (1 + slack))), (got.min(), got.max())
