"""A uniform number's or top_p's part of a weight (csrc/sample_parts.h) is exact for every float of 0 <= p < 1: the header
is compiled alone on the host and compared with fractions."""
import math
import os
import random
import shutil
import struct
import subprocess
from fractions import Fraction

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def part_of(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host C++ compiler")
    exe = str(tmp_path_factory.mktemp("parts") / "driver")
    subprocess.run([cxx, "-std=c++20", "-O2", "-I" + os.path.join(ROOT, "sandyrt_amd", "csrc"),
                    os.path.join(ROOT, "tests", "binding", "sample_parts_driver.cpp"), "-o", exe], check=True)

    def run(cases):
        text = "\n".join(f"{bits} {w} {int(up)}" for bits, w, up in cases)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True, timeout=60).stdout
        return [int(x) for x in out.split()]
    return run


def bits_of(p):
    return struct.unpack("<I", struct.pack("<f", p))[0]


def test_parts_are_exact(part_of):
    r = random.Random(3)
    edges = [bits_of(p) for p in (0.0, -0.0, 2.0 ** -149, 2.0 ** -126, 2.0 ** -126 - 2.0 ** -149, 2.0 ** -100, 2.0 ** -24, 0.5,
                                  0.5 - 2.0 ** -25, 1 - 2.0 ** -24)]
    assert edges[1] == 0x80000000
    drawn = [bits_of(r.random() * (1 - 2.0 ** -24)) for _ in range(200)] + [r.randrange(bits_of(1.0)) for _ in range(200)]
    cases = [(u, w, up) for u in edges + drawn for w in (0, 1, 2, 3, (1 << 50), (1 << 62), (1 << 62) - 1, r.randrange(1 << 62)) for up in (0, 1)]
    for (u, w, up), got in zip(cases, part_of(cases)):
        exact = Fraction(struct.unpack("<f", struct.pack("<I", u))[0]) * w
        assert got == (math.ceil(exact) if up else math.floor(exact)), (hex(u), w, up)
        assert w == 0 or got < w or up  # a target that the sum of all passes
