"""Performance cases of the serving operators behind the hybrid decoder's mixers: the paged key-value cache
(append with the position rotation, attention of single new tokens, attention of packed prompts) and the gated
delta rule (packed prompts in chunks, single tokens).

`own` chooses who computes: the plain torch form (elementary operations in 32 bits, rounded once at the end), or
the framework's C ABI.  Shapes are those of the repository's two decoders (query heads / kv heads of 256, rotary
dim 64; DeltaNet heads of 128 x 128) and generic ones of head dims 64 and 128.

  s35    16 query heads over 2 kv heads, DeltaNet 16 key / 32 value heads
  s397   32 query heads over 2 kv heads, DeltaNet 16 key / 64 value heads
  gen128 32 query heads over 8 kv heads of 128
  gen64  12 query heads over 12 kv heads of 64

The framework's calls go to the stream of their own context, which no torch stream waits for, nor it for them.  So
prepare() returns inputs that are finished, and whoever reads the results of run(), or lets go of a state that it has
run, waits for the device first (torch.cuda.synchronize()).

Lengths of a batch come from the case's `longest` and `sequences` alone (a spread from long to short), so work()
knows them.
"""
import ctypes
import math

import torch

own = False

SHAPES = {
    "s35": dict(nh=16, nkv=2, hd=256, rd=64, kh=16, vh=32),
    "s397": dict(nh=32, nkv=2, hd=256, rd=64, kh=16, vh=64),
    "gen128": dict(nh=32, nkv=8, hd=128, rd=128),
    "gen64": dict(nh=12, nkv=12, hd=64, rd=32),
}
DK = DV = 128            # DeltaNet key and value dims
THETA, EPS = 1e7, 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
CHUNK = 64               # the plain delta rule's chunk


def listed():
    return [
        # One sequence's next token enters the cache: the smallest call, all latency.
        dict(name="append-1", kind="append", model="s397", type="bf16", sequences=1, longest=1, before=4096, page=16),
        # Eleven prompts of different lengths enter the cache, fp32 as the framework's activations are.
        dict(name="append-prompts-f32", kind="append", model="s35", type="f32", sequences=11, longest=1300, before=0, page=64),
        # One sequence's next token at 4,097 positions: single-user decoding.
        dict(name="decode-1", kind="decode", model="s397", type="bf16", sequences=1, longest=4097, page=16),
        # Continuous batching, 48 sequences of very different lengths.
        dict(name="decode-48-ragged", kind="decode", model="gen128", type="f16", sequences=48, longest=9001, page=16),
        # The framework's own type: thirteen sequences of an fp32 cache.
        dict(name="decode-13-f32", kind="decode", model="s35", type="f32", sequences=13, longest=6000, page=32),
        # Three very long contexts: bandwidth.
        dict(name="decode-long", kind="decode", model="s397", type="bf16", sequences=3, longest=131071, page=64),
        # Short prompts packed together, multi-head, an odd total.
        dict(name="prompt-short", kind="prompt", model="gen64", type="f16", sequences=9, longest=333, before=0, page=16),
        # Long prompts of the large decoder: matrix products.
        dict(name="prompt-long", kind="prompt", model="s397", type="bf16", sequences=3, longest=4999, before=0, page=64),
        # Draft tokens under verification: few rows of each of four sequences behind long caches.
        dict(name="prompt-verify", kind="prompt", model="s397", type="bf16", sequences=4, longest=7, before=20000, page=16),
        # Single tokens of sixteen sequences through the delta rule.
        dict(name="delta-step-16", kind="step", model="s397", type="bf16", sequences=16),
        # Prompts through the small decoder's delta rule in the framework's own type.
        dict(name="delta-prompts-f32", kind="delta", model="s35", type="f32", sequences=5, longest=700),
        # One long prompt through the large decoder's delta rule, every state of it in order.
        dict(name="delta-prompt-long", kind="delta", model="s397", type="bf16", sequences=1, longest=8191),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "prompt", "prompt", "prompt", "step", "delta", "delta"])
    typ = rng.choice(sorted(TYPES))
    if kind in ("step", "delta"):
        model = rng.choice(["s35", "s397"])
        if kind == "step":
            return dict(kind=kind, model=model, type=typ, sequences=_log(rng, 1, 64))
        n = _log(rng, 1, 16)
        return dict(kind=kind, model=model, type=typ, sequences=n, longest=_log(rng, 1, 8191 // n))
    model, page = rng.choice(sorted(SHAPES)), rng.choice([8, 16, 32, 48, 64, 128])
    if kind == "append":
        n = _log(rng, 1, 100)
        return dict(kind=kind, model=model, type=typ, sequences=n, longest=_log(rng, 1, max(1, 6000 // n)),
                    before=rng.choice([0, _log(rng, 1, 2000)]), page=page)
    if kind == "decode":
        n = _log(rng, 1, 128)
        return dict(kind=kind, model=model, type=typ, sequences=n, longest=_log(rng, 1, 130000 // n), page=page)
    n = _log(rng, 1, 24)
    if rng.random() < 0.3:
        return dict(kind=kind, model=model, type=typ, sequences=n, longest=_log(rng, 1, 16), before=_log(rng, 1, 40000 // n),
                    page=page)
    longest = _log(rng, 1, (3500 if typ != "f32" else 2000) // (1 + n // 4))
    return dict(kind=kind, model=model, type=typ, sequences=n, longest=longest, before=0, page=page)


def _spread(n, longest):
    """n lengths from `longest` down to a fraction of it, none below one token, in a mixed order."""
    lens = [max(1, int(longest * (1 - i / n) ** 1.5)) for i in range(n)]
    return lens[::2] + lens[1::2][::-1]


def _lengths(case):
    """(new tokens, cached positions with them) of each sequence."""
    if case["kind"] == "step":
        return [1] * case["sequences"], [1] * case["sequences"]
    new = _spread(case["sequences"], case["longest"])
    if case["kind"] == "decode":
        return [1] * len(new), new
    before = case.get("before", 0)
    old = [max(1, before - before * i // (3 * len(new))) if before else 0 for i in range(len(new))]
    return new, [a + b for a, b in zip(new, old)]


# ---- inputs -------------------------------------------------------------------------------------------


class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(1 + (int(seed) * 1000003) % (1 << 40))

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda").mul_(std)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=self.g, device="cuda").mul_(hi - lo).add_(lo)


def prepare(case, seed):
    torch.cuda.synchronize()  # calls on earlier states, whose memory this one may get
    s = _inputs(case, seed)
    torch.cuda.synchronize()  # the inputs, before another stream reads them
    return s


def _inputs(case, seed):
    r, m, dt = _Rand(seed), SHAPES[case["model"]], TYPES[case["type"]]
    new, length = _lengths(case)
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    T, n = start[-1], len(new)
    s = dict(case=case, m=m, dt=dt, new=new, length=length, start=start, T=T,
             h_start=(ctypes.c_int * (n + 1))(*start), h_length=(ctypes.c_int * n)(*length))
    if case["kind"] in ("step", "delta"):
        kh, vh = m["kh"], m["vh"]
        kd, vd = kh * DK, vh * DV
        # the rows that the causal convolution leaves: q | k | v after SiLU
        mix = torch.nn.functional.silu(r.normal(T, 2 * kd + vd)).to(dt)
        slots = n + 2
        order = torch.randperm(slots, generator=r.g, device="cuda")[:n]
        rate = r.uniform(vh, lo=math.log(1e-3), hi=math.log(1e-1)).exp_()
        s.update(mix=mix, a=r.normal(T, vh), b=r.normal(T, vh), a_log=r.uniform(vh, lo=1.0, hi=16.0).log_(),
                 dt_bias=rate + torch.log(-torch.expm1(-rate)), state=r.normal(slots, vh, DK, DV, std=0.1),
                 slot=order, h_slot=(ctypes.c_int * n)(*order.tolist()), slots=slots)
        # the rows of slots that no sequence has stay as they were
        s["state_out"] = s["state"].clone()
        s["out"] = torch.empty(T, vh, DV, device="cuda", dtype=dt)
        return s
    nh, nkv, hd, ps = m["nh"], m["nkv"], m["hd"], case["page"]
    need = [-(-x // ps) for x in length]
    width, pages = max(need) + 1, sum(need) + 3
    ids = torch.randperm(pages, generator=r.g, device="cuda").to(torch.int32)
    table = torch.full((n, width), -1, device="cuda", dtype=torch.int32)
    at = torch.arange(width, device="cuda")
    need_t = torch.tensor(need, device="cuda")
    table[at[None, :] < need_t[:, None]] = ids[: sum(need)]
    s.update(table=table, width=width, pages=pages)
    shape = (pages, ps, nkv, hd)
    if case["kind"] == "append":
        # query and gate of a head side by side, as the fused projection leaves them
        s.update(q=r.normal(T, nh, 2 * hd).to(dt), k=r.normal(T, nkv * hd).to(dt), v=r.normal(T, nkv * hd).to(dt),
                 q_norm=r.normal(hd, std=0.1), k_norm=r.normal(hd, std=0.1),
                 q_out=torch.empty(T, nh, hd, device="cuda", dtype=dt),
                 k_pool=r.normal(*shape).to(dt), v_pool=r.normal(*shape).to(dt))
        return s
    # positions that no sequence has written hold whatever was there
    cells = _cells(table, torch.tensor(length, device="cuda"), ps)
    k_pool, v_pool = (torch.full((pages * ps, nkv, hd), float("nan"), device="cuda", dtype=dt) for _ in range(2))
    real = cells[cells >= 0]
    k_pool[real] = r.normal(real.numel(), nkv, hd).to(dt)
    v_pool[real] = r.normal(real.numel(), nkv, hd).to(dt)
    s.update(k_pool=k_pool.view(shape), v_pool=v_pool.view(shape), q=r.normal(T, nh, hd, std=2.0).to(dt),
             gate=r.normal(T, nh, 2 * hd).to(dt), out=torch.empty(T, nh, hd, device="cuda", dtype=dt))
    return s


def _cells(table, length, ps):
    """[sequence, position]: the pool's row of each position, -1 behind a sequence's end."""
    p = torch.arange(table.shape[1] * ps, device=table.device)[: int(length.max())]
    rows = table.long()[:, p // ps] * ps + p % ps
    return torch.where(p[None, :] < length[:, None], rows, -1)


# ---- the plain forms -------------------------------------------------------------------------------


def _norm_rotate(x, w, pos, rd):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + w)
    half = rd // 2
    # far positions need their angle in 64 bits
    freq = THETA ** (-torch.arange(half, device=x.device, dtype=torch.float64) * 2 / rd)
    ang = pos.double()[:, None, None] * freq
    co, si = torch.cos(ang).float(), torch.sin(ang).float()
    a, b = x[..., :half], x[..., half:rd]
    return torch.cat([a * co - b * si, b * co + a * si, x[..., rd:]], -1)


def _token_rows(s):
    dev = s["table"].device
    new, length = torch.tensor(s["new"], device=dev), torch.tensor(s["length"], device=dev)
    seq = torch.repeat_interleave(torch.arange(len(s["new"]), device=dev), new, output_size=s["T"])
    first = torch.tensor(s["start"][:-1], device=dev)
    pos = torch.arange(s["T"], device=dev) - first[seq] + (length - new)[seq]
    return seq, pos


def _plain_append(s):
    m, ps = s["m"], s["case"]["page"]
    seq, pos = _token_rows(s)
    q = _norm_rotate(s["q"][..., : m["hd"]], s["q_norm"], pos, m["rd"]).to(s["dt"])
    k = _norm_rotate(s["k"].view(s["T"], m["nkv"], m["hd"]), s["k_norm"], pos, m["rd"]).to(s["dt"])
    cell = s["table"][seq, pos // ps].long() * ps + pos % ps
    for pool, x in ((s["k_pool"], k), (s["v_pool"], s["v"].view(s["T"], m["nkv"], m["hd"]))):
        pool.view(-1, m["nkv"], m["hd"])[cell] = x
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _gathered(s):
    """Keys and values of every sequence, padded to the longest: [sequence, kv head, position, dim]."""
    m = s["m"]
    cells = _cells(s["table"], torch.tensor(s["length"], device=s["table"].device), s["case"]["page"])
    there = cells >= 0
    cells = torch.where(there, cells, cells[:, :1])
    k, v = (p.view(-1, m["nkv"], m["hd"])[cells].permute(0, 2, 1, 3).float().contiguous() for p in (s["k_pool"], s["v_pool"]))
    return k, v, there


def _softmax_values(scores, v):
    scores = scores - scores.amax(-1, keepdim=True)
    p = scores.exp_()
    return (p @ v) / p.sum(-1, keepdim=True)


def _plain_decode(s):
    m, n = s["m"], len(s["new"])
    k, v, there = _gathered(s)
    q = s["q"].view(n, m["nkv"], m["nh"] // m["nkv"], m["hd"]).float()
    scores = (q @ k.transpose(-1, -2)) / math.sqrt(m["hd"])
    o = _softmax_values(scores.masked_fill_(~there[:, None, None], -math.inf), v).reshape(n, m["nh"], m["hd"])
    return {"out": (o * torch.sigmoid(s["gate"][..., m["hd"] :].float())).to(s["dt"])}


def _plain_prompt(s):
    m, dev = s["m"], s["q"].device
    n, g, most = len(s["new"]), m["nh"] // m["nkv"], max(s["new"])
    seq, pos = _token_rows(s)
    place = torch.arange(s["T"], device=dev) - torch.tensor(s["start"][:-1], device=dev)[seq]
    k, v, there = _gathered(s)
    q = torch.zeros(n, most, m["nkv"], g, m["hd"], device=dev)
    q[seq, place] = s["q"].view(s["T"], m["nkv"], g, m["hd"]).float()
    at = torch.zeros(n, most, dtype=torch.long, device=dev)
    at[seq, place] = pos
    sees = torch.arange(k.shape[2], device=dev) <= at[..., None]        # [sequence, query, position]
    q = q.permute(0, 2, 3, 1, 4).reshape(n, m["nkv"], g * most, m["hd"])
    scores = ((q @ k.transpose(-1, -2)) / math.sqrt(m["hd"])).view(n, m["nkv"], g, most, -1)
    scores = scores.masked_fill_(~sees[:, None, None], -math.inf).view(n, m["nkv"], g * most, -1)
    o = _softmax_values(scores, v).view(n, m["nkv"], g, most, m["hd"]).permute(0, 3, 1, 2, 4)[seq, place]
    o = o.reshape(s["T"], m["nh"], m["hd"])
    return {"out": (o * torch.sigmoid(s["gate"][..., m["hd"] :].float())).to(s["dt"])}


def _delta_inputs(s):
    """q, k (unit length, per value head), v, log decay and beta of every token."""
    m, T = s["m"], s["T"]
    kd, rep = m["kh"] * DK, m["vh"] // m["kh"]
    mix = s["mix"].float()
    q, k = (x.view(T, m["kh"], DK) for x in (mix[:, :kd], mix[:, kd : 2 * kd]))
    q = q * torch.rsqrt(q.square().sum(-1, keepdim=True) + 1e-6) / math.sqrt(DK)
    k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) + 1e-6)
    g = -s["a_log"].exp() * torch.nn.functional.softplus(s["a"] + s["dt_bias"])
    return (q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1), mix[:, 2 * kd :].reshape(T, m["vh"], DV), g,
            torch.sigmoid(s["b"]))


def _plain_step(s):
    q, k, v, g, beta = _delta_inputs(s)
    S = s["state"][s["slot"]] * g.exp()[..., None, None]
    d = beta[..., None] * (v - (k[..., None, :] @ S)[..., 0, :])
    S = S + k[..., None] * d[..., None, :]
    s["state_out"][s["slot"]] = S
    return {"out": (q[..., None, :] @ S)[..., 0, :].to(s["dt"]), "state": s["state_out"]}


def _plain_delta(s):
    """Chunks of 64 tokens: within a chunk the tokens' corrections solve a triangular system, from chunk to chunk
    the state is carried."""
    m, n, dev = s["m"], len(s["new"]), s["mix"].device
    x = _delta_inputs(s)
    seq = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(s["new"], device=dev), output_size=s["T"])
    place = torch.arange(s["T"], device=dev) - torch.tensor(s["start"][:-1], device=dev)[seq]
    chunks = -(-max(s["new"]) // CHUNK)

    def laid(t):  # [sequence, head, chunk, token, ...], zeros behind a sequence's end
        y = torch.zeros(n, chunks * CHUNK, *t.shape[1:], device=dev)
        y[seq, place] = t
        return y.transpose(1, 2).reshape(n, m["vh"], chunks, CHUNK, *t.shape[2:])

    q, k, v, g, beta = (laid(t) for t in x)
    G = g.double().cumsum(-1)
    D = (G[..., :, None] - G[..., None, :]).tril().exp().float().tril()
    kk = k @ k.transpose(-1, -2)
    A = (beta[..., None] * D * kk).tril(-1)
    # (1 + A)^-1, row by row for all chunks at once
    R = torch.eye(CHUNK, device=dev).expand_as(A).clone()
    for t in range(1, CHUNK):
        R[..., t : t + 1, :t] = -(A[..., t : t + 1, :t] @ R[..., :t, :t])
    eG, eR = G.exp().float()[..., None], (G[..., -1:] - G).exp().float()[..., None]
    U, W = R @ (v * beta[..., None]), R @ (k * eG * beta[..., None])
    P, qg, kr = D * (q @ k.transpose(-1, -2)), q * eG, (k * eR).transpose(-1, -2).contiguous()
    S, o = s["state"][s["slot"]], torch.empty_like(v)
    for c in range(chunks):
        d = U[:, :, c] - W[:, :, c] @ S
        o[:, :, c] = qg[:, :, c] @ S + P[:, :, c] @ d
        S = S * eG[:, :, c, -1:] + kr[:, :, c] @ d
    s["state_out"][s["slot"]] = S
    o = o.view(n, m["vh"], chunks * CHUNK, DV).transpose(1, 2)[seq, place]
    return {"out": o.to(s["dt"]), "state": s["state_out"]}


# ---- the framework's calls ---------------------------------------------------------------------------

_held = []


def _backend():
    if not _held:
        from shiftwing_amd import Backend
        _held.append(Backend(torch.cuda.current_device()))
    return _held[0]


def _own(s):
    from shiftwing_amd.abi import ColiDelta, ColiPaged
    be, m, case = _backend(), s["m"], s["case"]
    lib, ctx, kind, n = be.lib, be.ctx, s["case"]["kind"], len(s["new"])
    code, hd = CODES[case["type"]], m.get("hd")
    if kind in ("step", "delta"):
        kd, size = m["kh"] * DK, s["mix"].element_size()
        d = ColiDelta(code, m["kh"], m["vh"], DK, DV, s["slots"], *[s["mix"].shape[1]] * 3)
        p = s["mix"].data_ptr()
        given = (s["out"].data_ptr(), p, p + kd * size, p + 2 * kd * size, s["a"].data_ptr(), s["b"].data_ptr(),
                 s["a_log"].data_ptr(), s["dt_bias"].data_ptr(), s["state"].data_ptr(), s["state_out"].data_ptr())
        if kind == "step":
            be.check(lib.coli_cuda_delta_step(ctx, ctypes.byref(d), *given, s["h_slot"], n), "coli_cuda_delta_step")
        else:
            be.check(lib.coli_cuda_delta_prompt(ctx, ctypes.byref(d), *given, s["h_start"], s["h_slot"], n),
                     "coli_cuda_delta_prompt")
        return {"out": s["out"], "state": s["state_out"]}
    c = ColiPaged(code, m["nh"], m["nkv"], hd, case["page"], s["pages"], s["width"], case["page"] * m["nkv"] * hd)
    k_pool, v_pool, table = s["k_pool"].data_ptr(), s["v_pool"].data_ptr(), s["table"].data_ptr()
    if kind == "append":
        be.check(lib.coli_cuda_paged_append(
            ctx, ctypes.byref(c), k_pool, v_pool, table, s["h_start"], s["h_length"], n, s["q_out"].data_ptr(),
            s["q"].data_ptr(), m["nh"] * 2 * hd, 2 * hd, s["k"].data_ptr(), m["nkv"] * hd, s["v"].data_ptr(), m["nkv"] * hd,
            s["q_norm"].data_ptr(), s["k_norm"].data_ptr(), EPS, m["rd"], THETA), "coli_cuda_paged_append")
        return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    gate = (s["gate"].data_ptr() + hd * s["gate"].element_size(), m["nh"] * 2 * hd, 2 * hd)
    if kind == "decode":
        be.check(lib.coli_cuda_paged_decode(ctx, ctypes.byref(c), s["out"].data_ptr(), s["q"].data_ptr(), *gate, k_pool, v_pool,
                                            table, s["h_length"], n, 1 / math.sqrt(hd)), "coli_cuda_paged_decode")
    else:
        be.check(lib.coli_cuda_paged_prompt(ctx, ctypes.byref(c), s["out"].data_ptr(), s["q"].data_ptr(), *gate, k_pool, v_pool,
                                            table, s["h_start"], s["h_length"], n, 1 / math.sqrt(hd)), "coli_cuda_paged_prompt")
    return {"out": s["out"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "step": _plain_step,
            "delta": _plain_delta}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    m, size = SHAPES[case["model"]], BYTES[case["type"]]
    new, length = _lengths(case)
    T = sum(new)
    if case["kind"] in ("step", "delta"):
        kd, vd = m["kh"] * DK, m["vh"] * DV
        moved = T * ((2 * kd + 2 * vd) * size + 2 * m["vh"] * 4) + 2 * len(new) * m["vh"] * DK * DV * 4 + 2 * m["vh"] * 4
        return {"bytes": moved, "flops": 7 * T * m["vh"] * DK * DV}
    nh, nkv, hd = m["nh"], m["nkv"], m["hd"]
    if case["kind"] == "append":
        return {"bytes": 2 * T * (nh + 2 * nkv) * hd * size + 8 * hd + 4 * sum(-(-x // case["page"]) for x in length),
                "flops": T * (nh + nkv) * (4 * hd + 3 * m["rd"])}
    seen = sum(a * b - a * (a - 1) // 2 for a, b in zip(new, length))
    return {"bytes": 3 * T * nh * hd * size + 2 * sum(length) * nkv * hd * size + 4 * sum(-(-x // case["page"]) for x in length),
            "flops": 4 * nh * hd * seen}


# ---- the same results in 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    m = s["m"]
    if case["kind"] in ("step", "delta"):
        return _exact_delta(s, m)
    hd, nkv, ps = m["hd"], m["nkv"], case["page"]
    pages = s["table"].tolist()
    rows = [torch.tensor([pages[i][p // ps] * ps + p % ps for p in range(n)], device="cuda") for i, n in enumerate(s["length"])]
    if case["kind"] == "append":
        pos = torch.cat([torch.arange(n - t, n, device="cuda") for t, n in zip(s["new"], s["length"])])
        turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64),
                           pos.double()[:, None] / THETA ** (torch.arange(0, m["rd"], 2, device="cuda").double() / m["rd"]))

        def turned(x, w):
            x = x.double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * (w.double() + 1)
            pair = torch.complex(x[..., : m["rd"] // 2], x[..., m["rd"] // 2 : m["rd"]]) * turn[:, None]
            return torch.cat([pair.real, pair.imag, x[..., m["rd"] :]], -1)

        cells = torch.cat([r[n - t :] for r, t, n in zip(rows, s["new"], s["length"])])
        kp, vp = s["k_pool"].double(), s["v_pool"].double()
        kp.view(-1, nkv, hd)[cells] = turned(s["k"].reshape(s["T"], nkv, hd), s["k_norm"])
        vp.view(-1, nkv, hd)[cells] = s["v"].double().reshape(s["T"], nkv, hd)
        return {"q": turned(s["q"][..., :hd], s["q_norm"]), "k_pool": kp, "v_pool": vp}
    outs = []
    for i, (t, n) in enumerate(zip(s["new"], s["length"])):
        lo = s["start"][i]
        q = s["q"][lo : lo + t].double()
        here = torch.empty(t, m["nh"], hd, device="cuda", dtype=torch.float64)
        mask = torch.arange(n, device="cuda")[None, :] > torch.arange(n - t, n, device="cuda")[:, None]
        for h in range(m["nh"]):
            k, v = (p.view(-1, nkv, hd)[rows[i], h * nkv // m["nh"]].double() for p in (s["k_pool"], s["v_pool"]))
            w = torch.softmax((q[:, h] @ k.t() / math.sqrt(hd)).masked_fill_(mask, -math.inf), -1)
            here[:, h] = w @ v
        outs.append(here)
    return {"out": torch.cat(outs) / (1 + torch.exp(-s["gate"][..., hd:].double()))}


def _exact_delta(s, m):
    """Token by token, all sequences and heads side by side."""
    mix, kh, vh = s["mix"].double(), m["kh"], m["vh"]
    first, new = torch.tensor(s["start"][:-1], device="cuda"), s["new"]
    A = torch.exp(s["a_log"].double())
    S = s["state"][s["slot"]].double()
    out = torch.empty(s["T"], vh, DV, device="cuda", dtype=torch.float64)
    for t in range(max(new)):
        live = torch.tensor([i for i, n in enumerate(new) if n > t], device="cuda") if t >= min(new) else slice(None)
        row = first[live] + t
        x = mix[row]
        q, k = (x[:, i * kh * DK : (i + 1) * kh * DK].reshape(-1, kh, 1, DK).expand(-1, kh, vh // kh, DK).reshape(-1, vh, DK)
                for i in (0, 1))
        q, k = (y / (y.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt() for y in (q, k))
        decay = torch.exp(-A * torch.log1p(torch.exp(s["a"][row].double() + s["dt_bias"].double())))
        X = S[live] * decay[:, :, None, None]
        d = x[:, 2 * kh * DK :].reshape(-1, vh, DV) - (k[..., None] * X).sum(-2)
        X = X + k[..., None] * (d / (1 + torch.exp(-s["b"][row].double()))[..., None])[:, :, None]
        out[row] = (q[..., None] * X).sum(-2) / DK ** 0.5
        S[live] = X
    state = s["state_out"].double()
    state[s["slot"]] = S
    return {"out": out, "state": state}
