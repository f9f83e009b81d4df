"""Further refusals of the paged-cache calls and their wrappers, before the device is touched."""
import pytest

from test_paged_cpu import _decode, _prompt, _refused


@pytest.mark.parametrize("call", [_decode, _prompt])
def test_scales_that_overflow_as_powers_of_two(call):
    """3e38 is finite, 3e38 log2(e) is not, and infinity times a score of zero is NaN."""
    for scale in (3e38, -3e38, 2.4e38):
        _refused(call(scale=scale), "log2(e)")
    for scale in (2.3e38, -2.3e38, 0.0, 1e-45):
        _refused(call(scale=scale), "null context")


def test_bounds_that_are_no_ints():
    """Lengths, starts and slots are C ints: 2^32 + 5 is not 5, and 2.5 is not 2."""
    import numpy as np

    from shiftwing_amd.delta import DeltaRule
    from shiftwing_amd.paged import PagedCache, ints
    from test_paged_cpu import _NoDevice
    c = PagedCache(_NoDevice(), kind="f32", query_heads=4, kv_heads=2, head_dim=64, page_size=16, pages=8, table_pages=4,
                   sequences=2)
    r = DeltaRule(_NoDevice(), kind="f32", key_heads=1, value_heads=1, key_dim=64, value_dim=32, slots=3,
                  a_log=np.zeros(1), dt_bias=np.zeros(1))
    k, q, mix, a = np.zeros((5, 2, 64)), np.zeros((5, 4, 64)), np.zeros((5, 160)), np.zeros((5, 1))
    far = np.array([(1 << 32) + 5])
    calls = [lambda: c.append([0, 5], far, k, k), lambda: c.append([0, 4.5], [5], k, k), lambda: c.append([0, 5], [[5]], k, k),
             lambda: c.decode(q[:1], far, 1.0), lambda: c.decode(q[:1], [np.nan], 1.0), lambda: c.prompt(q, [[0], [5]], [5], 1.0),
             lambda: c.prompt(q, np.array([0, (1 << 32) + 5]), [5], 1.0), lambda: r.prompt(mix, a, a, [0, 5], far - 5),
             lambda: r.step(mix[:1], a[:1], a[:1], [1 + (1 << 33)])]
    for call in calls:
        with pytest.raises(ValueError):
            call()
    assert ints([])[0].size == 0 and ints([0.0, 3])[0].tolist() == [0, 3] and ints(range(3))[0].dtype == np.int32
