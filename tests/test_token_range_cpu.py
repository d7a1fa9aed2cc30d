"""The cut of a K-grouped product's token ranges at the rows that exist, compiled for the host: sizes of any value, whose
plain sums would leave 32 or 64 bits, give ranges inside the rows."""

import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "triton_grouped_gemm_b200" / "csrc"

PROGRAM = """
#include <cstdio>
#define __host__
#define __device__
#define __forceinline__ inline
#include "token_range.cuh"
int main() {
  char kind;
  long long a, b, total;
  while (std::scanf(" %c %lld %lld %lld", &kind, &a, &b, &total) == 4) {
    const b200::TokenSpan s = kind == 's' ? b200::span_of_size(a, b, total) : b200::span_of_bounds(a, b, total);
    std::printf("%lld %lld %d\\n", s.start, s.tokens, s.cut ? 1 : 0);
  }
}
"""


@pytest.fixture(scope="module")
def spans(tmp_path_factory):
    folder = tmp_path_factory.mktemp("token_range")
    (folder / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", str(CSRC),
                    str(folder / "main.cpp"), "-o", str(folder / "main")], check=True)

    def run(queries):
        text = "\n".join(" ".join(map(str, q)) for q in queries)
        out = subprocess.run([str(folder / "main")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


HUGE = [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 62, 2 ** 63 - 1]
SMALL = [0, 1, 5, 90, 91, 4000, -1, -(2 ** 31), -(2 ** 63)]


@pytest.mark.parametrize("total", [0, 1, 90, 2 ** 31 - 1])
def test_running_sizes(spans, total):
    for sizes in ([40, 30, 20], [40, 30, 4000, 5], HUGE, [5] + HUGE[::-1], SMALL, HUGE + SMALL):
        start = 0
        for size in sizes:
            got_start, tokens, cut = spans([("s", start, size, total)])[0]
            want = min(max(size, 0), total - start)
            assert (got_start, tokens, cut) == (start, want, int(max(size, 0) > want))
            start += tokens
        assert start <= total < 2 ** 31


@pytest.mark.parametrize("total", [0, 90, 2 ** 31 - 1])
def test_explicit_bounds(spans, total):
    ends = [0, 1, 40, 89, 90, 91, 2 ** 31 - 1, -1, -40, -(2 ** 31)]
    queries = [("b", lo, hi, total) for lo in ends for hi in ends]
    for (_, lo, hi, _), (start, tokens, cut) in zip(queries, spans(queries)):
        rows = [r for r in (max(lo, 0), min(hi, total))]
        want = max(rows[1] - rows[0], 0)
        assert tokens == want and 0 <= start and start + tokens <= total
        assert tokens == 0 or start == lo or lo < 0
        assert cut == int(hi > lo and want != hi - lo)
