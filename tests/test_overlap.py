"""CPU: the host's test of whether two strided tensors share memory, against the bytes themselves."""
import random
import shutil
import subprocess

import pytest

from conftest import ROOT

MAIN = r"""
#include <cstdio>
#include "overlap.h"
int main() {
  long long v[16];
  for (;;) {
    b200moe::StridedRows r[2];
    for (int k = 0; k < 2; ++k) {
      for (int i = 0; i < 8; ++i) if (scanf("%lld", &v[i]) != 1) return 0;
      r[k].base = (uintptr_t)v[0]; r[k].width = v[1];
      for (int a = 0; a < 3; ++a) r[k].axis(v[2 + 2 * a], v[3 + 2 * a]);
    }
    printf("%d %d\n", (int)b200moe::rows_meet(r[0], r[1]), (int)r[0].same(r[1]));
  }
}
"""


@pytest.fixture(scope="module")
def meet(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("overlap")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", str(ROOT / "on_device_sd_b200" / "csrc"), str(d / "main.cpp"), "-o", str(d / "main")], check=True)

    def ask(pairs):
        text = "\n".join(" ".join(str(x) for t in p for x in (t[0], t[1], *[y for ax in t[2] for y in ax])) for p in pairs)
        out = subprocess.run([str(d / "main")], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
        return [tuple(int(x) for x in line.split()) for line in out if line]

    return ask


def held(t):
    base, width, axes = t
    starts = [base]
    for n, s in axes:
        starts = [x + i * s for x in starts for i in range(n)]
    return {x + k for x in starts for k in range(width)}


def test_random_layouts_against_the_bytes(meet):
    rng = random.Random(5)
    pairs = []
    for _ in range(4000):
        pair = []
        for _ in range(2):
            width = rng.choice([1, 2, 4, 8, 16])
            axes = [(rng.choice([0, 1, 1, 2, 3, 5]) if rng.random() < 0.1 else rng.randint(1, 5), rng.choice([0, 4, 8, 16, 24, 32, 48, 64, 100, 160, 320])) for _ in range(3)]
            pair.append((1000 + rng.choice([0, 4, 8, 16, 32, 64, 200, 500, 900]), width, axes))
        if rng.random() < 0.5:
            pair[1] = (pair[1][0], pair[1][1], pair[0][2])       # the same strides, as views of one buffer have
        pairs.append(pair)
    got = meet(pairs)
    for p, (yes, _) in zip(pairs, got):
        assert yes == int(bool(held(p[0]) & held(p[1]))), p
    assert 0.2 < sum(y for y, _ in got) / len(got) < 0.8


def test_layouts_of_the_operators(meet):
    """Heads of 128 16-bit elements: 256 bytes."""
    d, hq, hk, T = 256, 32, 4, 8191
    row = (hq + 2 * hk) * d
    one, base = (1, 0), 1 << 40
    q, k, v = ((base + o * d, d, [(T, row), (n, d), one]) for o, n in ((0, hq), (hq, hk), (hq + hk, hk)))
    other = (base + T * row, d, [(T, hq * d), (hq, d), one])
    shifted = (base + 16, d, [(T, row), (hq, d), one])
    later = (base + 3 * row, d, [(T - 3, row), (hq, d), one])
    dense = (base, d, [(T, hq * d), (hq, d), one])
    blocks, page = 1000, 256
    k_half = (base, d, [(blocks, 2 * page * hk * d), (page, hk * d), (hk, d)])
    v_half = (base + page * hk * d, d, [(blocks, 2 * page * hk * d), (page, hk * d), (hk, d)])
    k_heads = (base, d, [(blocks, 2 * page * hk * d), (page, 2 * hk * d), (hk, 2 * d)])
    v_heads = (base + d, d, [(blocks, 2 * page * hk * d), (page, 2 * hk * d), (hk, 2 * d)])
    cases = [(q, k, 0), (q, v, 0), (k, v, 0), (q, other, 0), (q, q, 1), (q, shifted, 1), (q, later, 1), (q, dense, 1), (k, dense, 1), (k_half, v_half, 0),
             (k_heads, v_heads, 0), (k_half, k_half, 1), (k_half, k_heads, 1), (k_half, (base + 64, *v_half[1:]), 1)]
    got = meet([c[:2] for c in cases])
    assert [g[0] for g in got] == [c[2] for c in cases]
    assert got[4][1] == 1 and sum(g[1] for g in got) == 2
