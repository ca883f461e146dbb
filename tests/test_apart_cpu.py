"""csrc/apart.cuh, which finds operands that share memory, against a search byte by byte."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <stdio.h>
#include "apart.cuh"
using namespace ennx;
int main() {  // per line: base, run, counts and strides of a, then of b
  long long v[16];
  for (;;) {
    for (int i = 0; i < 16; ++i)
      if (scanf("%lld", v + i) != 1) return 0;
    Memory m[2];
    for (int k = 0; k < 2; ++k) {
      const long long* x = v + 8 * k;
      m[k].base = (const void*)x[0];
      m[k].run = x[1];
      for (int d = 0; d < 3; ++d) { m[k].count[d] = x[2 + d]; m[k].stride[d] = x[5 + d]; }
    }
    printf("%d %d\n", (int)share_bytes(m[0], m[1]), (int)shares_own_bytes(m[0]));
  }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    cxx = os.environ.get("CXX", "g++")
    if shutil.which(cxx) is None:
        pytest.skip("no C++ compiler")
    at = tmp_path_factory.mktemp("apart")
    (at / "apart.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT}/ennx_b200/csrc", str(at / "apart.cpp"), "-o",
                    str(at / "apart")], check=True)

    def run(pairs):
        text = "\n".join(" ".join(str(n) for m in p for n in (m[0], m[1], *m[2], *m[3])) for p in pairs)
        out = subprocess.run([str(at / "apart")], input=text, capture_output=True, text=True, check=True, timeout=60).stdout
        return [tuple(int(n) for n in line.split()) for line in out.splitlines()]
    return run


def runs(m):
    base, run, (a, b, c), (s, t, u) = m
    return [range(base + i * s + j * t + k * u, base + i * s + j * t + k * u + run)
            for i in range(a) for j in range(b) for k in range(c)]


def test_against_every_byte(ask):
    rng = random.Random(1)
    pairs = []
    for _ in range(4000):
        one = [(rng.randint(200, 300), rng.randint(0, 6), [rng.choice([0, 1, 1, 2, 3, 5]) for _ in range(3)],
                [rng.choice([0, 1, 4, 6, 8, 12, 24, 48, rng.randint(0, 60)]) for _ in range(3)]) for _ in range(2)]
        if rng.random() < 0.5:
            one[1] = (one[1][0], one[1][1], one[1][2], one[0][3])
        pairs.append(one)
    both = own = 0
    for (a, b), got in zip(pairs, ask(pairs)):
        ra, rb = runs(a), runs(b)
        seen = [n for r in ra for n in r]
        want = int(bool(set(seen) & {n for r in rb for n in r})), int(len(set(seen)) < len(seen))
        assert got == want, (a, b)
        both, own = both + want[0], own + want[1]
    assert 300 < both < 3700 and 300 < own < 3700


def test_large_strides_and_the_layouts_of_one_tensor(ask):
    far = 1 << 40
    q = (far, 4096, (16384, 1, 1), (6144, 0, 0))       # columns of a projection
    k = (far + 4096, 1024, (16384, 1, 1), (6144, 0, 0))
    v = (far + 5120, 1024, (16384, 1, 1), (6144, 0, 0))
    shifted = (far + 4094, 1024, (16384, 1, 1), (6144, 0, 0))
    behind = (far + 16384 * 6144, 4096, (16384, 1, 1), (6144, 0, 0))
    other = (far + 4096, 2048, (8192, 1, 1), (12288, 0, 0))   # every second row, other columns
    # key and value caches side by side, [batch, room, 2, heads, 128] and [2, batch, heads, room, 128]
    kc = (far, 256, (32, 1 << 20, 8), ((1 << 20) * 4096, 4096, 256))
    vc = (far + 2048, 256, (32, 1 << 20, 8), ((1 << 20) * 4096, 4096, 256))
    kh = (far, 256, (32, 1 << 20, 8), ((1 << 20) * 2048, 256, (1 << 20) * 256))
    vh = (far + (32 << 20) * 2048, 256, (32, 1 << 20, 8), ((1 << 20) * 2048, 256, (1 << 20) * 256))
    crossed = (far, 256, (32, 1 << 20, 8), ((1 << 20) * 2048, 128, (1 << 20) * 256))
    none = (0, 4096, (16384, 1, 1), (6144, 0, 0))
    cases = [((q, k), (0, 0)), ((k, v), (0, 0)), ((v, q), (0, 0)), ((q, shifted), (1, 0)), ((shifted, v), (0, 0)),
             ((shifted, k), (1, 0)), ((q, behind), (0, 0)), ((q, other), (0, 0)), ((k, other), (1, 0)), ((q, q), (1, 0)),
             ((kc, vc), (0, 0)), ((kc, kc), (1, 0)), ((kh, vh), (0, 0)), ((kc, kh), (1, 0)), ((crossed, q), (1, 1)),
             ((none, q), (0, 0)), ((q, none), (0, 0))]
    assert ask([c for c, _ in cases]) == [w for _, w in cases]
