"""The refusals of the packed Gated DeltaNet calls, before the device (here there is
none) is touched."""
import ctypes as C

import pytest

from test_paged_cpu import AT, _ints, _lib, _refused


def _desc(**kw):
    from shiftwing_amd.abi import ColiDelta
    d = dict(type=1, key_heads=2, value_heads=4, key_dim=64, value_dim=32, slots=100, q_stride=512, k_stride=512, v_stride=512)
    d.update(kw)
    return ColiDelta(*[d[f] for f, _ in ColiDelta._fields_])


def _tensors(kw):
    d = dict(out=AT, q=AT, k=AT, v=AT, a=AT, b=AT, a_log=AT, dt_bias=AT, state=AT, state_out=AT)
    d.update({n: v for n, v in kw.items() if n in d})
    return list(d.values())


def _step(desc=None, **kw):
    slot = kw.get("slot", [3, 1])
    return _lib().coli_cuda_delta_step(None, C.byref(desc or _desc()), *_tensors(kw), _ints(slot) if slot is not None else None,
                                       kw.get("n", len(slot or [0])))


def _prompt(desc=None, **kw):
    slot, start = kw.get("slot", [3, 1]), kw.get("start", [0, 5, 5])
    return _lib().coli_cuda_delta_prompt(None, C.byref(desc or _desc()), *_tensors(kw),
                                         _ints(start) if start is not None else None,
                                         _ints(slot) if slot is not None else None, kw.get("n", len(slot or [0])))


@pytest.mark.parametrize("call", [_step, _prompt])
def test_a_sound_call_lacks_only_its_context(call):
    _refused(call(), "null context")
    _refused(call(n=0), "null context")
    _refused(call(_desc(slots=200), slot=list(range(150)), start=[0] * 151), "null context")


@pytest.mark.parametrize("call", [_step, _prompt])
@pytest.mark.parametrize("bad,word", [
    (dict(type=3), "element type"), (dict(key_heads=0), "key_heads"), (dict(value_heads=3), "key_heads"),
    (dict(value_heads=-4, key_heads=-2), "key_heads"), (dict(key_dim=136), "key_dim"), (dict(key_dim=12), "key_dim"),
    (dict(key_dim=0), "key_dim"), (dict(value_dim=48), "key_dim"), (dict(value_dim=288), "key_dim"), (dict(value_dim=0), "key_dim"),
    (dict(slots=0), "slots"), (dict(q_stride=516), "strides"), (dict(k_stride=-512), "strides"), (dict(v_stride=4), "strides"),
])
def test_descriptions(call, bad, word):
    _refused(call(_desc(**bad)), word)


@pytest.mark.parametrize("call", [_step, _prompt])
def test_tensors_and_slots(call):
    for n in ("out", "q", "k", "v", "a", "b", "a_log", "dt_bias", "state", "state_out"):
        _refused(call(**{n: None}), "null tensor")
        _refused(call(**{n: AT + 2}), "aligned")
    _refused(call(n=-1), "null slots")
    _refused(call(slot=None), "null slots")
    _refused(call(slot=[3, 100]), "slot[1]")
    _refused(call(slot=[-1, 3]), "slot[0]")
    _refused(call(slot=[3, 3]), "named twice")
    _refused(call(slot=list(range(80)) + [7], start=[0] * 82), "named twice")


def test_prompt_rows():
    _refused(_prompt(start=None), "null start")
    _refused(_prompt(start=[-1, 5, 5]), "negative")
    _refused(_prompt(start=[0, 5, 4]), "sequence 1")
    _refused(_prompt(start=[0, 5, (1 << 31) - 64]), "sequence 1")
    _refused(_prompt(start=[0, 5, (1 << 31) - 65]), "null context")


def test_shapes_that_do_not_fit():
    import numpy as np

    from shiftwing_amd.delta import DeltaRule
    from test_paged_cpu import _NoDevice

    def rule(heads=4):
        return DeltaRule(_NoDevice(), kind="f32", key_heads=2, value_heads=4, key_dim=64, value_dim=32, slots=3,
                         a_log=np.zeros(heads), dt_bias=np.zeros(heads))
    r, x, a = rule(), np.zeros((5, 2 * 128 + 128)), np.zeros((5, 4))
    calls = [lambda: rule(3), lambda: r.write(np.zeros((3, 4, 32, 64))), lambda: r.prompt(x, a, a, [0, 6], [0]),
             lambda: r.prompt(x, a, a, [0, 5], [0, 1]), lambda: r.prompt(x[:, 1:], a, a, [0, 5], [0]),
             lambda: r.prompt(x, a[:4], a, [0, 5], [0]), lambda: r.prompt(x, a, a[:, :2], [0, 5], [0]),
             lambda: r.step(x, a, a, [0, 1]), lambda: r.step(x[:2], a, a, [0, 1])]
    for call in calls:
        with pytest.raises(ValueError):
            call()
