"""The bin of a logit's weight (sample_bins.h), with the undefined-behaviour sanitizer: whatever the logits and the
temperature are, no float leaves the range of the whole number that it becomes."""

import ctypes
import math
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fusor-ai_amd", "csrc")
SOURCE = """
#include "sample_bins.h"
extern "C" double bins(float x, float top, double scale) { return fg::bins_of(x, fg::top_of(top), scale); }
extern "C" int bin(float x, float top, double scale) { return fg::bin_of(fg::bins_of(x, fg::top_of(top), scale)); }
"""


@pytest.fixture(scope="module")
def bins(tmp_path_factory):
    where = tmp_path_factory.mktemp("bins")
    source, lib = where / "bins.cpp", where / "bins.so"
    source.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined,float-cast-overflow", "-fno-sanitize-recover",
                    "-I", CSRC, str(source), "-o", str(lib)], check=True)
    lib = ctypes.CDLL(str(lib))
    for f in (lib.bins, lib.bin):
        f.argtypes = [ctypes.c_float, ctypes.c_float, ctypes.c_double]
    lib.bins.restype = ctypes.c_double
    return lib


def test_ordinary_logits(bins):
    for temperature in (0.01, 0.7, 1.0, 100.0):
        for x in (5.0, 4.999, 4.0, 0.0, -3.5, -27.0):
            t = 32 * (5 - ctypes.c_float(x).value) / temperature
            assert bins.bins(x, 5.0, 32 / temperature) == pytest.approx(t, rel=1e-15)
            assert bins.bin(x, 5.0, 32 / temperature) == min(int(bins.bins(x, 5.0, 32 / temperature)), 1023)


@pytest.mark.parametrize("scale", [1e-290, 1e-30, 1.0, 32.0, 3200.0, 1e38, 2.5e46])  # 32 over any f32 temperature
def test_every_logit_has_a_bin(bins, scale):
    inf = math.inf
    for top in (inf, 3.4e38, 1.0, 0.0, -3.4e38):
        for x in (inf, 3.4e38, 1.0, 1e-45, 0.0, -1.0, -1e10, -3.4e38, -inf):
            if x <= top:
                b = bins.bin(x, top, scale)
                t = bins.bins(x, top, scale)
                assert b == (1023 if t >= 1023 else int(t))
    assert bins.bin(-inf, 1.0, scale) == 1023
    assert bins.bin(1.0, 1.0, scale) == bins.bin(inf, inf, scale) == 0
