"""The division of a step's number by the steps of one product (term_steps.hpp), compiled for the host."""

import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "causal-tuner_amd", "csrc")
SOURCE = """
#include "term_steps.hpp"
// The first step of `products` products of `one` steps each that is put in the wrong place, or -1.
extern "C" int64_t first_wrong(int one, int products) {
    const ct::TermDivisor by = ct::term_divisor(one);
    for (int64_t t = 0; t < (int64_t)one * products; ++t) {
        const ct::TermStep s = ct::term_step((int)t, one, by);
        if (s.product != t / one || s.at != t % one) return t;
    }
    return -1;
}
"""


@pytest.fixture(scope="module")
def first_wrong(tmp_path_factory):
    place = tmp_path_factory.mktemp("term_steps")
    (place / "steps.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, str(place / "steps.cpp"), "-o",
                    str(place / "steps.so")], check=True)
    call = ctypes.CDLL(str(place / "steps.so")).first_wrong
    call.restype, call.argtypes = ctypes.c_int64, [ctypes.c_int, ctypes.c_int]
    return call


@pytest.mark.parametrize("first,count", [(1, 3000), (26752, 300), (26992, 1), (65535, 2), (262140, 8)])
def test_every_step_is_in_its_product(first, count, first_wrong):
    """26992 steps (1 727 488 rows of 64) are among those where the rounded reciprocal alone is one too large."""
    for one in range(first, first + count):
        assert first_wrong(one, 6) == -1, one
