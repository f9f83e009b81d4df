"""The workspace of split attention grows when a context first needs it, not with every few hundred tokens."""
import numpy as np
import pytest

from test_gpu_paged import _cache, _check, _fill, _round, _want

pytestmark = pytest.mark.gpu


def test_a_growing_context_keeps_its_workspace():
    from shiftwing_amd import Backend
    be = Backend(0)
    rng = np.random.default_rng(121)
    nh, nkv, hd, most = 32, 2, 256, 16000
    c, table = _cache(be, "bf16", nh, nkv, hd, 16, [most, most], rng)
    K, V = _fill(c, table, [most, most], rng, "bf16")
    q = _round(rng.standard_normal((3, nh, hd)), "bf16")

    def turn(n):
        return (c.decode(q[:1], [n], 0.0625), c.decode(q[:2], [n, n // 2], 0.0625),
                c.prompt(q, [0, 3], [n], 0.0625), c.prompt(q, [0, 1, 3], [n // 3, n], 0.0625))
    turn(200)  # the calls' own arrays; single tokens are split
    free = be.memory_info()[0]
    for n in [*range(300, 3000, 137), *range(3000, most, 1009), most]:
        got = turn(n)
        assert abs(free - be.memory_info()[0]) < 1 << 20, f"at {n} positions"
    want, tol = _want(q[0], K, V, table, 0, most, 0.0625, None, "bf16")
    _check(got[0][0], want, tol, "the longest")
