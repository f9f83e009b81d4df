"""The gated delta rule on packed prompts and single tokens against its definition,
token by token in 64 bits, on the same, already rounded inputs.

Tolerance.  A token's update S <- (1 - beta k k^T) e^g S + beta k v^T never grows a
column's norm beyond what v adds (|k| = 1, beta <= 1, g <= 0), so errors of earlier
tokens pass on undiminished at most and add up.  A chunk of 64 tokens forms its
columns by sums of at most key_dim + 3 x 64 terms of that column's size m (the larger
of its norm and |v|): (key_dim + 192) 2^-24 m a chunk, worst case; single tokens are
held to the same per 64.  The decays' own error, 2^-22 |g|, adds 2^-22 x 128 at most
where e^g is not yet negligible (|g| e^g <= 0.4: 2^-23).  An output is a unit vector's
product with the state, over sqrt(key_dim), and its rounding, finfo.eps / 2 relative
(bf16 2^-8, fp16 2^-11, fp32 2^-24; fp16 below 2^-14 2^-25 absolute)."""
import numpy as np
import pytest

from test_gpu_paged import U, _round

pytestmark = pytest.mark.gpu


class Rule:
    """Inputs of a case and the definition in 64 bits, all sequences and heads side by side."""

    def __init__(self, be, kind, kh, vh, dk, dv, slots, seed, decay=(1.0, 16.0)):
        from shiftwing_amd.delta import DeltaRule
        self.rng = np.random.default_rng(seed)
        self.kind, self.kh, self.vh, self.dk, self.dv = kind, kh, vh, dk, dv
        self.a_log = np.log(self.rng.uniform(*decay, vh)).astype(np.float32)
        self.dt_bias = self.rng.uniform(-4, 1, vh).astype(np.float32)
        self.dev = DeltaRule(be, kind=kind, key_heads=kh, value_heads=vh, key_dim=dk, value_dim=dv, slots=slots,
                             a_log=self.a_log, dt_bias=self.dt_bias)
        self.S = self.rng.standard_normal((slots, vh, dk, dv)).astype(np.float32)
        self.dev.write(self.S)
        self.S = self.S.astype(np.float64)
        self.size = np.sqrt((self.S ** 2).sum(2, keepdims=True))  # largest column norm so far
        self.chunks = np.zeros(slots)

    def rows(self, n):
        mix = _round(self.rng.standard_normal((n, 2 * self.kh * self.dk + self.vh * self.dv)), self.kind)
        return mix, *(self.rng.standard_normal((n, self.vh)).astype(np.float32) * 2 for _ in range(2))

    def token(self, mix, a, b, slot):
        """One token of each row's slot; the outputs."""
        n, kd = len(mix), self.kh * self.dk
        m = mix.astype(np.float64)
        q, k = (m[:, i * kd:(i + 1) * kd].reshape(n, self.kh, self.dk).repeat(self.vh // self.kh, 1) for i in (0, 1))
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6) for x in (q, k))
        v = m[:, 2 * kd:].reshape(n, self.vh, self.dv)
        g = -np.exp(self.a_log.astype(np.float64)) * np.logaddexp(0, a.astype(np.float64) + self.dt_bias)
        S = self.S[slot] * np.exp(g)[..., None, None]
        d = (v - np.einsum("nhk,nhkv->nhv", k, S)) / (1 + np.exp(-b.astype(np.float64)))[..., None]
        S = S + k[..., None] * d[:, :, None]
        self.S[slot] = S
        self.size[slot] = np.maximum(self.size[slot], np.maximum(np.sqrt((S ** 2).sum(2, keepdims=True)), np.abs(v)[:, :, None]))
        return np.einsum("nhk,nhkv->nhv", q, S) / np.sqrt(self.dk)

    def prompt(self, mix, a, b, start, slot):
        out = np.zeros((len(mix), self.vh, self.dv))
        start, slot = np.asarray(start), np.asarray(slot)
        for t in range(int(np.diff(start).max(initial=0))):
            live = np.flatnonzero(np.diff(start) > t)
            r = start[live] + t
            out[r] = self.token(mix[r], a[r], b[r], slot[live])
        self.chunks[slot] += -(-np.diff(start) // 64)
        return out

    def tol(self, slot):
        """State tolerance [slot][vh][1][dv]."""
        return ((self.dk + 192) * 2.0 ** -24 + 2.0 ** -22) * (self.chunks[slot][:, None, None, None] + 1) * self.size[slot]

    def check_out(self, got, want, slot, what):
        tol = self.tol(slot)[:, :, 0] * self.dk ** -0.5 * 2
        tol = tol + U[self.kind] * (np.abs(want) + tol) + (2.0 ** -25 if self.kind == "f16" else 0)
        assert np.all(np.isfinite(got)), what
        assert np.all(np.abs(got - want) <= tol), f"{what}: {np.max(np.abs(got - want) / tol):.3g} x the tolerance"

    def check_state(self):
        got, tol = self.dev.read(), self.tol(np.arange(len(self.S)))
        tol = np.where(self.chunks[:, None, None, None] > 0, tol, 0)  # slots no call named are as they were
        assert np.all(np.isfinite(got))
        assert np.all(np.abs(got - self.S) <= tol), f"state: {np.max(np.abs(got - self.S) / np.maximum(tol, 1e-30)):.3g} x"

    def run_prompt(self, mix, a, b, start, slot):
        got, want = self.dev.prompt(mix, a, b, start, slot), self.prompt(mix, a, b, start, slot)
        seen = np.zeros(len(mix), bool)
        for s, n in enumerate(np.diff(start)):
            r = np.arange(start[s], start[s + 1])
            seen[r] = True
            if n:
                self.check_out(got[r], want[r], np.full(n, slot[s]), f"sequence {s}")
        assert np.all(got[~seen] == 0), "rows of no sequence"
        self.check_state()

    def run_step(self, mix, a, b, slot):
        got, want = self.dev.step(mix, a, b, slot), self.token(mix, a, b, np.asarray(slot))
        self.chunks[slot] += 1
        self.check_out(got, want, np.asarray(slot), "step")
        self.check_state()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kh,vh,dk,dv,start,slot,slots", [
    (1, 1, 128, 128, [0, 1], [0], 1),                                       # one token
    (2, 4, 128, 128, [0, 64, 64, 127, 192, 257], [4, 0, 6, 1, 3], 8),        # around a chunk, an empty one, free slots
    (1, 8, 64, 32, [3, 203], [1], 2),                                       # a gap in front; more value heads than waves
    (3, 3, 8, 256, [0, 130, 131], [1, 0], 2),                               # smallest key dim
    (2, 2, 104, 96, [0, 70, 300], [0, 2], 3),
    (1, 2, 24, 64, [0, 500], [0], 1),
])
def test_prompt(be, kind, kh, vh, dk, dv, start, slot, slots):
    print(f"[delta prompt] {kind} heads {kh}/{vh} dims {dk} x {dv} rows {start}", flush=True)
    r = Rule(be, kind, kh, vh, dk, dv, slots, 21)
    r.run_prompt(*r.rows(start[-1] + 2), start, slot)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kh,vh,dk,dv,slot,slots", [
    (1, 1, 128, 128, [0], 1), (16, 64, 128, 128, [2, 0], 3), (2, 6, 40, 160, [5, 1, 3], 7), (1, 1, 8, 32, [1], 4),
    (1, 2, 16, 32, list(range(139, -1, -1)), 150),   # more rows than a launch
])
def test_step(be, kind, kh, vh, dk, dv, slot, slots):
    print(f"[delta step] {kind} heads {kh}/{vh} dims {dk} x {dv} rows {len(slot)}", flush=True)
    r = Rule(be, kind, kh, vh, dk, dv, slots, 22)
    for _ in range(2):
        r.run_step(*r.rows(len(slot)), slot)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompts_then_tokens(be, kind):
    """Prompts, single tokens, chunks that end anywhere, in the same slots."""
    r = Rule(be, kind, 2, 4, 128, 64, 4, 23)
    r.run_prompt(*r.rows(100), [0, 37, 100], [2, 0])
    r.run_step(*r.rows(2), [0, 2])
    r.run_prompt(*r.rows(140), [0, 65, 65, 139], [0, 1, 2])
    r.run_step(*r.rows(3), [2, 1, 0])


@pytest.mark.parametrize("how", ["same keys", "no decay", "all decay", "mixed decay", "zero rows"])
def test_hard_inputs(be, how):
    """Equal keys make the chunk's system as far from the identity as it gets; decays from none to all, and tokens of
    either kind side by side, where sums of g are large and their differences small."""
    r = Rule(be, "f32", 1, 2, 128, 32, 1, 24)
    mix, a, b = r.rows(200)
    if how == "same keys":
        mix[:, 128:256] = mix[0, 128:256]
        a[:] = -30.0
        b[:] = 20.0
    elif how == "no decay":
        a[:] = -50.0
    elif how == "all decay":
        a[:] = 3e4
    elif how == "mixed decay":
        a[:] = np.where(np.arange(200) % 7 == 3, 40.0, -9.0)[:, None]
    else:
        mix[::3] = 0.0
    r.run_prompt(mix, a, b, [0, 200], [0])


def test_prompt_in_passes(be):
    """More records than one pass holds: 128 sequences of up to five chunks, in groups of two launches."""
    r = Rule(be, "bf16", 16, 64, 8, 32, 140, 25)
    new = np.r_[r.rng.integers(0, 150, 138), 300, 64]
    start = np.r_[0, np.cumsum(new)].tolist()
    r.run_prompt(*r.rows(start[-1]), start, r.rng.permutation(140).tolist())


def test_state_out_apart(be):
    """With a second state the first one stays, and only the call's slots are written."""
    import ctypes as C

    from shiftwing_amd.abi import ColiDelta
    r = Rule(be, "f32", 2, 2, 64, 32, 3, 26)
    mix, a, b = r.rows(70)
    before = r.dev.read()
    other = be.upload(np.full(before.shape, 7.0, np.float32))
    d = ColiDelta(0, 2, 2, 64, 32, 3, *[mix.shape[1]] * 3)
    x, da, db = be.upload(mix), be.upload(a), be.upload(b)
    out = be.alloc(70 * 2 * 32 * 4)
    given = (out.p, x.p, C.c_void_p(x.ptr + 128 * 4), C.c_void_p(x.ptr + 256 * 4), da.p, db.p, r.dev.a_log.p, r.dev.dt_bias.p,
             r.dev.state.p, other.p)
    be.check(be.lib.coli_cuda_delta_prompt(be.ctx, C.byref(d), *given, (C.c_int * 3)(0, 70, 70), (C.c_int * 2)(2, 0), 2), "prompt")
    got = be.download(other, before.shape, np.float32)
    assert np.array_equal(r.dev.read(), before)
    assert np.all(got[1] == 7.0) and np.array_equal(got[0], before[0])
    r.prompt(mix, a, b, [0, 70, 70], [2, 0])
    assert np.all(np.abs(got[2] - r.S[2]) <= r.tol([2])[0])
    be.check(be.lib.coli_cuda_delta_step(be.ctx, C.byref(d), *given, (C.c_int * 1)(1), 1), "step")
    got = be.download(other, before.shape, np.float32)
    r.token(mix[:1], a[:1], b[:1], np.array([1]))
    assert np.all(np.abs(got[1] - r.S[1]) <= r.tol([1])[0]) and np.array_equal(r.dev.read(), before)


def test_same_state_as_the_layer(be, oracle):
    """The states are the Gated DeltaNet layer's: a prompt here leaves what its own steps leave."""
    from oracle import pyoracle as po
    from test_gpu_mixers import _dev_gdn, _x
    g = po.HostGdn(51, 128, 1, 4, 128, 32, K=4)
    dev = _dev_gdn(be, g, slots=2)
    rng = np.random.default_rng(27)
    cs, st = dev.read_state()
    assert st.shape == (2, 4, 128, 32)
    X = _x(rng, 3, 128)
    ab = [po.oracle_gdn_gates(oracle, g, X[i]) for i in range(3)]
    for i in range(3):
        dev.slots_step(X[i:i + 1], ab[i][0][None], ab[i][1][None], [1], [i])
    _, st = dev.read_state()
    # the layer's own convolution outputs are inside it; its state continues here
    r = Rule(be, "f32", 1, 4, 128, 32, 2, 28)
    r.dev.state, r.S = dev.state, st.astype(np.float64)
    r.size = np.sqrt((r.S ** 2).sum(2, keepdims=True))
    r.run_prompt(*r.rows(66), [0, 66], [1])
    assert np.array_equal(dev.read_state()[1], r.dev.read())


class Raw:
    """The C calls on q, k and v of their own."""

    def __init__(self, be, r, strides):
        import ctypes as C

        from shiftwing_amd.abi import ColiDelta
        from shiftwing_amd.paged import KINDS
        self.C, self.be, self.r = C, be, r
        self.d = ColiDelta(KINDS[r.kind], r.kh, r.vh, r.dk, r.dv, r.dev.slots, *strides)

    def call(self, name, out, q, k, v, a, b, *rest):
        ints = [(self.C.c_int * len(x))(*x) if isinstance(x, list) else x for x in rest]
        dev = self.r.dev
        self.be.check(getattr(self.be.lib, "coli_cuda_delta_" + name)(
            self.be.ctx, self.C.byref(self.d), out.p, q.p, k.p, v.p, a.p, b.p, dev.a_log.p, dev.dt_bias.p, dev.state.p,
            dev.state.p, *ints), name)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_tensors_apart(be, kind):
    """q, k and v in arrays and strides of their own, an output that is not clear, rows of no sequence, which may hold
    anything."""
    from shiftwing_amd.paged import from_kind, to_kind, word
    r = Rule(be, kind, 2, 6, 72, 96, 5, 31)
    T, kd, vd = 150, 2 * 72, 6 * 96
    mix, a, b = r.rows(T)
    start, slot = [4, 70, 147], [3, 1]
    mix[:4], mix[147:], a[:4], b[147:] = np.nan, np.inf, np.nan, np.nan
    parts = [mix[:, :kd], mix[:, kd:2 * kd], mix[:, 2 * kd:]]
    wide = [kd + 8, kd, vd + 40]
    dev = [be.upload(to_kind(np.concatenate([x, np.full((T, w - x.shape[1]), np.nan, np.float32)], 1), kind))
           for x, w in zip(parts, wide)]
    da, db = be.upload(a), be.upload(b)
    raw = Raw(be, r, wide)
    out = be.upload(to_kind(np.full((T, 6, 96), 7.0), kind))
    raw.call("prompt", out, *dev, da, db, start, slot, 2)
    got = from_kind(be.download(out, (T, 6, 96), word(kind)), kind)
    assert np.all(got[:4] == 7.0) and np.all(got[147:] == 7.0)
    mix[:4], mix[147:], a[:4], b[147:] = 0, 0, 0, 0
    want = r.prompt(mix, a, b, start, slot)
    for s in range(2):
        rows = slice(start[s], start[s + 1])
        r.check_out(got[rows], want[rows], np.full(start[s + 1] - start[s], slot[s]), f"sequence {s}")
    r.check_state()
    mix, a, b = r.rows(2)
    dev = [be.upload(to_kind(np.concatenate([x, np.full((2, w - x.shape[1]), np.nan, np.float32)], 1), kind))
           for x, w in zip((mix[:, :kd], mix[:, kd:2 * kd], mix[:, 2 * kd:]), wide)]
    da, db = be.upload(a), be.upload(b)
    raw.call("step", out, *dev, da, db, [4, 3], 2)
    want = r.token(mix, a, b, np.array([4, 3]))
    r.chunks[[4, 3]] += 1
    got = from_kind(be.download(out, (T, 6, 96), word(kind)), kind)
    r.check_out(got[:2], want, np.array([4, 3]), "step")
    r.check_state()


def test_what_is_not_finite_stays_with_its_sequence(be):
    """A NaN in one sequence: another, and the slots no call names, are as without it, to the bit; from the NaN on its
    own outputs and its state are NaN."""
    got = []
    for bad in (False, True):
        r = Rule(be, "bf16", 2, 4, 128, 64, 3, 32)
        mix, a, b = r.rows(300)
        if bad:
            mix[100, :2 * 2 * 128] = np.nan  # q and k
        got.append((r.dev.prompt(mix, a, b, [0, 170, 300], [2, 0]), r.dev.read()))
    (clean, state), (out, after) = got
    assert np.array_equal(out[170:], clean[170:]) and np.array_equal(out[:64], clean[:64])
    assert np.array_equal(after[[0, 1]], state[[0, 1]])
    assert np.all(np.isnan(out[100:170])) and np.all(np.isnan(after[2]))


def test_the_same_bits_again(be):
    r = Rule(be, "bf16", 2, 8, 128, 128, 4, 33)
    mix, a, b = r.rows(700)
    before, seen = r.dev.read(), []
    for _ in range(3):
        r.dev.write(before)
        out = r.dev.prompt(mix, a, b, [0, 333, 334, 700], [1, 3, 0])
        seen.append((out, r.dev.step(mix[:4], a[:4], b[:4], [0, 1, 2, 3]), r.dev.read()))
    for other in seen[1:]:
        assert all(np.array_equal(x, y) for x, y in zip(seen[0], other))
