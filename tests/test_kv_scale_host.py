"""How a page's scale grows (csrc/kv_scale.h), compiled for the CPU: every pair of a stored scale and a need ends,
in as few doublings as the need asks for, whatever the scale's sign."""
import math
import os
import subprocess

import numpy as np
import pytest

from project_willamette_b200 import build

MAIN = r"""
#include <cstdio>
#include "kv_scale.h"
int main() {
    float old, need;
    while (std::scanf("%a %a", &old, &need) == 2) {
        const wl::PageScale g = wl::grown_scale(old, need);
        std::printf("%a %d\n", (double)g.scale, g.doublings);
    }
}
"""

TINY, MOST = np.float32(2.0 ** -149), np.finfo(np.float32).max
NEEDS = [0.0, TINY, 3 * TINY, 2.0 ** -126, 1e-20, 0.00787, 1.0, 1.0000001, 127.0, 1e30, MOST / np.float32(127)]
SIZES = [TINY, 3 * TINY, 2.0 ** -127, 1e-20, 0.004, 0.5, 1.0, 3.0, 1e30, MOST]


@pytest.fixture(scope="module")
def grown(tmp_path_factory):
    d = tmp_path_factory.mktemp("scale")
    (d / "m.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", build.CSRC, str(d / "m.cpp"), "-o", str(d / "m")], check=True)

    def call(pairs):
        text = "".join(f"{float(a).hex()} {float(b).hex()}\n" for a, b in pairs)
        r = subprocess.run([str(d / "m")], input=text, capture_output=True, text=True, check=True, timeout=20)
        return [(float.fromhex(x.split()[0]), int(x.split()[1])) for x in r.stdout.splitlines()]
    return call


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_doublings(grown, sign):
    rng = np.random.default_rng(3)
    pairs = [(s, n) for s in SIZES for n in NEEDS]
    pairs += [(a, b) for a, b in zip(np.exp(rng.uniform(-80, 80, 500)), np.exp(rng.uniform(-80, 80, 500)))]
    pairs = [(np.float32(sign) * np.float32(a), np.float32(b)) for a, b in pairs]
    for (old, need), (scale, k) in zip(pairs, grown(pairs)):
        assert math.copysign(1, scale) == sign and abs(scale) >= float(need)
        assert scale == float(old) * 2.0 ** k  # exact: doublings round nothing
        assert k == 0 or abs(scale) / 2 < float(need)  # and no more than needed


def test_no_scale_yet_and_not_finite(grown):
    nan, inf = math.nan, math.inf
    assert grown([(0.0, 0.5), (-0.0, 0.5), (0.0, 0.0)]) == [(0.5, 0), (0.5, 0), (0.0, 0)]
    assert grown([(inf, 1.0), (-inf, 1.0)]) == [(inf, 0), (-inf, 0)]
    for scale, k in grown([(nan, 1.0), (nan, 0.0), (1.0, nan), (-1.0, nan), (0.0, nan), (inf, nan), (nan, nan)]):
        assert math.isnan(scale) and k == 0
