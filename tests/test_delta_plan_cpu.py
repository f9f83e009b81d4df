"""The passes that coli_cuda_delta_prompt makes over packed prompts (sw_delta_plan.h, compiled here): every chunk in
one pass, its records within the workspace, no pass shorter than it has to be."""
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT

FIT = 512 << 20  # bytes
PROGRAM = """
#include <stdio.h>
#include <vector>
#include "sw_delta_plan.h"
int main() {  // most, bytes of a chunk, sequences, their rows longest first; then the passes of the first launch
  int most, n;
  size_t bytes;
  while (scanf("%d %zu %d", &most, &bytes, &n) == 3) {
    std::vector<int> rows(n);
    for (int &r : rows)
      if (scanf("%d", &r) != 1) return 1;
    printf("%d", sw::delta_sequences(most, bytes));
    for (long long first = 0;;) {
      const long long c = sw::delta_pass(rows.data(), n, first, bytes);
      printf(" %lld/%d", c, sw::delta_live(rows.data(), n, first));
      first += c;
      if (n == 0 || first >= sw::chunks_of(rows[0])) break;
    }
    printf("\\n");
  }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "shiftwing_amd", "csrc"),
                    str(at / "plan.cpp"), "-o", str(at / "plan")], check=True)

    def run(bytes_, rows, most=128):
        rows = sorted(rows, reverse=True)
        text = subprocess.run([str(at / "plan")], input=" ".join(map(str, [most, bytes_, len(rows), *rows])),
                              capture_output=True, text=True, check=True).stdout.split()
        return int(text[0]), [tuple(int(x) for x in p.split("/")) for p in text[1:]]
    return run


BF16, F32 = 31504, 37648  # bytes of a chunk and value head


def test_one_long_prompt_beside_many_tokens(plan):
    rows = [8191] + [1] * 127
    assert plan(64 * BF16, rows)[1] == [(128, 128)]           # 255 records, 490 MiB
    assert [c for c, _ in plan(64 * F32, rows)[1]] == [95, 33]  # 222 records fit


@pytest.mark.parametrize("heads", [1, 32, 64, 128, 300])
@pytest.mark.parametrize("each", [BF16, F32])
def test_passes(plan, heads, each):
    rng = np.random.default_rng(5)
    for n in (1, 2, 17, 128):
        n = min(n, plan(heads * each, [])[0])
        rows = np.sort((rng.uniform(size=n) ** 4 * 20000).astype(int))[::-1]
        rows[n // 2:] = rng.integers(0, 2, n - n // 2)
        rows = np.sort(rows)[::-1]
        left, fit = -(-rows // 64), FIT // (heads * each)
        for c, live in plan(heads * each, rows.tolist())[1]:
            assert live == np.sum(left > 0)
            assert np.minimum(left, c).sum() <= fit
            assert c == left.max() or np.minimum(left, c + 1).sum() > fit, "more would have fit"
            left = np.maximum(left - c, 0)
        assert not left.any()


def test_launches(plan):
    for each, heads, n in ((BF16, 64, 128), (F32, 128, 111), (F32, 7000, 2), (F32, 65535, 1)):
        assert plan(each * heads, [])[0] == n
    assert plan(F32 * 65535, [130])[1] == [(1, 1)] * 3  # a chunk larger than the workspace: one at a time
    assert plan(BF16, [0, 0])[1] == [(0, 0)]
