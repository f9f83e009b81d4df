"""The refusals of the paged-cache calls: every check of their arguments fails with
a message before the device (here there is none) is touched."""
import ctypes as C

import pytest

BUF = (C.c_char * 4096)()
AT = (C.addressof(BUF) + 255) & ~255


def _lib():
    from shiftwing_amd import abi
    return abi.load()


def _cache(**kw):
    from shiftwing_amd.abi import ColiPaged
    d = dict(type=2, query_heads=4, kv_heads=2, head_dim=64, page_size=16, pages=8, table_pages=4, page_stride=16 * 2 * 64)
    d.update(kw)
    return ColiPaged(*[d[f] for f, _ in ColiPaged._fields_])


def _ints(a):
    return (C.c_int * max(1, len(a)))(*a)


def _append(cache=None, **kw):
    d = dict(k_pool=AT, v_pool=AT, table=AT, start=[0, 2, 3], length=[5, 1], sequences=2, q_out=AT, q=AT, q_stride=256,
             q_head=64, k=AT, k_stride=128, v=AT, v_stride=128, q_norm=AT, k_norm=AT, eps=1e-6, rd=32, theta=1e4)
    d.update(kw)
    d["start"], d["length"] = (_ints(d[n]) if d[n] is not None else None for n in ("start", "length"))
    return _lib().coli_cuda_paged_append(None, C.byref(cache or _cache()), *d.values())


def _decode(cache=None, **kw):
    d = dict(out=AT, q=AT, gate=AT, gate_stride=256, gate_head=64, k_pool=AT, v_pool=AT, table=AT, length=[5, 0], sequences=2,
             scale=0.125)
    d.update(kw)
    d["length"] = _ints(d["length"]) if d["length"] is not None else None
    return _lib().coli_cuda_paged_decode(None, C.byref(cache or _cache()), *d.values())


def _prompt(cache=None, **kw):
    d = dict(out=AT, q=AT, gate=AT, gate_stride=256, gate_head=64, k_pool=AT, v_pool=AT, table=AT, start=[0, 2, 2],
             length=[5, 0], sequences=2, scale=0.125)
    d.update(kw)
    d["start"], d["length"] = (_ints(d[n]) if d[n] is not None else None for n in ("start", "length"))
    return _lib().coli_cuda_paged_prompt(None, C.byref(cache or _cache()), *d.values())


def _refused(rc, word):
    assert rc == -1
    said = _lib().coli_cuda_last_error().decode()
    assert word in said, said


@pytest.mark.parametrize("call", [_append, _decode, _prompt])
def test_a_sound_call_lacks_only_its_context(call):
    _refused(call(), "null context")
    _refused(call(sequences=0), "null context")


@pytest.mark.parametrize("call", [_append, _decode, _prompt])
@pytest.mark.parametrize("bad,word", [
    (dict(type=3), "element type"), (dict(type=-1), "element type"), (dict(head_dim=96), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=3), "kv_heads"),
    (dict(query_heads=0), "kv_heads"), (dict(query_heads=-4, kv_heads=-2), "kv_heads"),
    (dict(page_size=0), "page_size"), (dict(pages=0), "page_size"), (dict(table_pages=0), "page_size"),
    (dict(pages=1 << 28), "page_size"), (dict(table_pages=1 << 28), "page_size"),
    (dict(page_stride=16 * 2 * 64 - 8), "page_stride"), (dict(page_stride=16 * 2 * 64 + 4), "page_stride"),
    (dict(page_stride=1 << 62), "page_stride"), (dict(page_stride=-(16 * 2 * 64)), "page_stride"),
])
def test_cache_descriptions(call, bad, word):
    _refused(call(_cache(**bad)), word)


@pytest.mark.parametrize("call", [_append, _decode, _prompt])
def test_pools_and_tables(call):
    for n in ("k_pool", "v_pool", "table"):
        _refused(call(**{n: None}), "null pool")
    _refused(call(k_pool=AT + 8), "16-byte")
    _refused(call(v_pool=AT + 2), "16-byte")
    _refused(call(table=AT + 2), "4-byte")
    _refused(call(sequences=-1), "sequence count")
    _refused(call(length=None), "null lengths")
    _refused(call(length=[65, 1]), "length[0]")
    _refused(call(length=[5, -1]), "length[1]")


@pytest.mark.parametrize("call", [_append, _prompt])
def test_packed_rows(call):
    _refused(call(start=None), "null start")
    _refused(call(start=[-1, 1, 1]), "negative")
    _refused(call(start=[0, 2, 1], length=[5, 5]), "sequence 1")
    _refused(call(start=[0, 6, 6]), "sequence 0")


@pytest.mark.parametrize("call", [_decode, _prompt])
def test_attention_operands(call):
    for n in ("out", "q"):
        _refused(call(**{n: None}), "16-byte")
        _refused(call(**{n: AT + 8}), "16-byte")
    _refused(call(gate=AT + 4), "gates")
    _refused(call(gate_stride=254), "gates")
    _refused(call(gate_head=-64), "gates")
    _refused(call(scale=float("nan")), "scale")
    _refused(call(scale=float("inf")), "scale")


def test_append_operands():
    _refused(_append(k=None), "null keys")
    _refused(_append(v=None), "null keys")
    _refused(_append(q=None), "one of q and q_out")
    _refused(_append(q_out=None), "one of q and q_out")
    _refused(_append(k=AT + 4), "16-byte")
    _refused(_append(q=AT + 4), "16-byte")
    _refused(_append(k_stride=132), "strides")
    _refused(_append(v_stride=-128), "strides")
    _refused(_append(q_head=60), "strides")
    _refused(_append(q_norm=AT + 1), "norms")
    for rd in (-2, 33, 66):
        _refused(_append(rd=rd), "rotary_dim")
    for theta in (0.0, -1.0, float("nan"), float("inf")):
        _refused(_append(theta=theta), "theta")
    for eps in (-1e-6, float("nan"), float("inf")):
        _refused(_append(eps=eps), "eps")
    # what is not used is not looked at
    _refused(_append(rd=0, theta=0.0), "null context")
    _refused(_append(q_norm=None, k_norm=None, eps=-1.0), "null context")


def test_largest_sizes():
    """Sizes whose indexes or launches would not fit: refused before anything runs."""
    many = _cache(table_pages=(1 << 26) + 1)
    for call in (_append, _decode, _prompt):
        _refused(call(many), "2^30")
    most = dict(table_pages=1 << 26)
    _refused(_append(_cache(**most), start=[0, 1 << 23, 1 << 24], length=[1 << 30, 1 << 23]), "2^24 - 1")
    _refused(_prompt(_cache(**most), start=[0, 1 << 23, 1 << 24], length=[1 << 30, 1 << 23]), "2^24 - 1")
    _refused(_append(_cache(**most), start=[5, 1 << 23, (1 << 24) + 4], length=[1 << 30, 1 << 30]), "null context")
    _refused(_prompt(_cache(**most), start=[5, 1 << 23, (1 << 24) + 4], length=[1 << 30, 1 << 30]), "null context")
    heads = dict(query_heads=1024, kv_heads=2, **most)  # 512 a kv head: 2^20 tokens of 1,024 heads
    _refused(_prompt(_cache(**heads), start=[0, 1 << 19, (1 << 19) + 1], length=[1 << 20, 1]), "2^29")
    _refused(_prompt(_cache(**heads), start=[0, 1 << 18, 1 << 19], length=[1 << 20, 1 << 20]), "null context")


class _NoDevice:
    """Takes uploads and fails any call: what the wrapper checks, it checks before one."""

    class lib:
        pass

    ctx = None

    def upload(self, a):
        return None


def test_shapes_that_do_not_fit():
    import numpy as np

    from shiftwing_amd.paged import PagedCache
    c = PagedCache(_NoDevice(), kind="bf16", query_heads=4, kv_heads=2, head_dim=64, page_size=16, pages=8, table_pages=4,
                   sequences=2)
    k, q = np.zeros((5, 2, 64)), np.zeros((5, 4, 64))
    calls = [lambda: c.set_table(np.zeros((2, 3), int)), lambda: c.set_table(np.zeros((1, 4), int)),
             lambda: c.append([0, 3], [3], k, k[:4]), lambda: c.append([0, 6], [6], k, k), lambda: c.append([0], [3], k, k),
             lambda: c.append([0, 3], [3], k, k, q[:, :3]), lambda: c.append([0, 3], [3], k, k, k_norm=np.ones(63)),
             lambda: c.append([0, 1, 2, 3], [3, 3, 3], k, k), lambda: c.decode(q[:3], [5, 5, 5], 1.0),
             lambda: c.decode(q, [5, 5], 1.0), lambda: c.decode(q[:2, :2], [5, 5], 1.0), lambda: c.decode(q[:2], [5, 5], 1.0, q),
             lambda: c.prompt(q, [0, 6], [6], 1.0), lambda: c.prompt(q, [0, 1, 2], [6], 1.0),
             lambda: c.prompt(q, [0, 5], [6], 1.0, k), lambda: c.write(k, k)]
    for call in calls:
        with pytest.raises(ValueError):
            call()
