"""csrc/rope_rule.h, the turns of a rotary pair's angle, on the CPU against more digits than they have."""
import ctypes
import os
import random
import shutil
import subprocess
from fractions import Fraction

import numpy as np
import pytest

from helpers import ROOT

DRIVER = """
#include "rope_rule.h"
extern "C" double turns(int position, float inv_freq) { return mi::turns_of<>(position, inv_freq); }
"""
PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    d = tmp_path_factory.mktemp("rope")
    src, so = d / "rope.cpp", str(d / "rope.so")
    src.write_text(DRIVER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-ffp-contract=off", "-shared", "-fPIC", "-I", os.path.join(ROOT, "adreno-llms_amd", "csrc"), "-o", so,
                           str(src)])
    lib = ctypes.CDLL(so)
    lib.turns.restype, lib.turns.argtypes = ctypes.c_double, [ctypes.c_int, ctypes.c_float]
    return lib


def test_turns(rule):
    """2^-54 for the last sum's rounding, another 2^-54 where it comes to a half and over; four roundings of 2^-106 of all turns before it, the second number of
    1 / 2 pi's own among them."""
    rng = random.Random(1)
    positions = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 10 ** 6, 4 * 10 ** 6] + [rng.randint(-2 ** 31, 2 ** 31 - 1) for _ in range(400)]
    freqs = [1.0, 0.7, 1e-6, 65.0, 1e4, 3e9, 2.0 ** -140] + [float(np.float32(10.0 ** rng.uniform(-7, 1))) for _ in range(60)]
    for f in freqs:
        exact_f = Fraction(float(np.float32(f)))
        for p in positions:
            all_of = p * exact_f / (2 * PI)
            got = rule.turns(p, f)
            assert abs(got) <= 0.5
            off = (Fraction(got) - all_of) % 1
            off = min(off, 1 - off)
            assert off <= Fraction(1, 2 ** 53) + abs(all_of) / 2 ** 102, (p, f, float(off))


def test_nothing_and_nan(rule):
    assert rule.turns(0, 1.0) == 0 and rule.turns(0, 3e38) == 0 and rule.turns(77, 0.0) == 0
    assert np.isnan(rule.turns(3, float("inf"))) and np.isnan(rule.turns(3, float("nan")))
