"""fp16 attention whose scores are as large as fp16 vectors make them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


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
