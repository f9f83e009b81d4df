"""Packed Gated DeltaNet prompts whose records take several passes: ragged batches, and the workspace they go through."""
import numpy as np
import pytest

from test_gpu_delta import Rule

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_long_prompts_beside_many_tokens(be, kind):
    """Two long prompts, one that ends in the second pass's middle, empty sequences and single tokens: more records
    than the workspace holds (266 of bf16, 222 of fp32, at 64 heads)."""
    r = Rule(be, kind, 16, 64, 8, 32, 100, 41)
    new = [1] * 40 + [0, 6011] + [1] * 20 + [65, 6400] + [0, 1, 4700]
    start = np.r_[0, np.cumsum(new)].tolist()
    print(f"[delta prompt] {kind} {len(new)} sequences, {start[-1]} rows", flush=True)
    r.run_prompt(*r.rows(start[-1] + 1), start, r.rng.permutation(100)[:len(new)].tolist())


def test_workspace_of_many_heads():
    """128 sequences of one token at 128 fp32 heads: a chunk of each is 588 MiB of records, the workspace 512."""
    from shiftwing_amd import Backend
    be = Backend(0)
    r = Rule(be, "f32", 128, 128, 8, 32, 128, 42)
    mix, a, b = r.rows(128)
    r.dev.prompt(mix, a, b, [0] + [1] * 128, list(range(128)))  # the arrays of a call, and one record
    before = r.dev.read()
    free = be.memory_info()[0]
    out = r.dev.prompt(mix, a, b, list(range(129)), list(range(128)))
    assert free - be.memory_info()[0] <= 544 << 20
    r.dev.write(before)
    r.S[0] = before[0]
    r.chunks[0] = 1
    want = r.token(mix, a, b, np.arange(128))
    r.chunks += 1
    r.check_out(out, want, np.arange(128), "tokens")
