"""CPU tests of which kernels the rows of a 4-bit product run in (csrc/mx_plan.h, compiled with the host
compiler), and that the GPU tests' sizes reach the ways of dealing them out that they are for."""
import subprocess

import pytest

from icsa_hip import build
from test_gpu_mx_split import SPLITS

pytestmark = pytest.mark.cpu

MAIN = """
#include <cstdio>
#include "mx_plan.h"
int main() {
  long long m, n, cols; int groups, gelu;
  while (std::scanf("%lld %lld %lld %d %d", &m, &n, &cols, &groups, &gelu) == 5) {
    const long long big = mx_large_rows(m, cols, groups, gelu != 0);
    std::printf("%d %lld %d\\n", mx_rows_takes(m, n), big, mx_rows_takes(m - big, n));
  }
}
"""


def _up(x, n):
    return -(-x // n) * n


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", build.CSRC_DIR, str(d / "main.cpp"), "-o", str(d / "main")],
                   check=True)

    def run(sizes):
        """(all rows in the kernel of few rows, rows of large tiles, the others in the kernel of few rows) of each
        (M, N, K, result in 4 bits, GELU)."""
        lines = ["%d %d %d %d %d" % (m, n, _up(n, 256) if mx else n, -(-k // 256), gelu) for m, n, k, mx, gelu in sizes]
        out = subprocess.run([str(d / "main")], input="\n".join(lines), capture_output=True, text=True, check=True).stdout
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]
    return run


@pytest.mark.parametrize("M,N,K,first,rest", SPLITS)
def test_sizes_of_the_gpu_tests_split(plan, M, N, K, first, rest):
    for all_few, big, few in plan([(M, N, K, mx, gelu) for mx in (0, 1) for gelu in (0, 1)]):
        assert not all_few and big == 256 * first < M
        assert few == (rest == "rows")


def test_every_row_is_taken_once(plan):
    """Large rows are whole tiles, or all of them; the kernel of few rows gets at most 64."""
    sizes = [(m, n, k, mx, g) for m in (1, 2, 33, 64, 65, 127, 256, 257, 1560, 3120, 4099, 9360, 14040, 65520, 1 << 20)
             for n in (1, 130, 2000, 5120, 13824, 30720) for k in (1, 256, 1300, 5120, 13824) for mx in (0, 1) for g in (0, 1)]
    for (m, n, k, mx, g), (all_few, big, few) in zip(sizes, plan(sizes)):
        assert 0 <= big <= m and (big == m or big % 256 == 0)
        assert all_few == (m <= 64 and n <= 8192 or m <= 32 and n <= 16384)
        if few and 0 < big < m:
            assert m - big <= 64
