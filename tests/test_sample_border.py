"""CPU: the borders that csrc/sample_draw.cu asks for (csrc/sample_border.cuh): the float that is returned lies on the near side, the one below it does not, and few floats are looked at, wherever
the border lies -- at and around logit 0 too, where 10^8 floats have the same difference to the maximum."""
import os
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "sample_border.cuh"
static long tests;
template <typename F> struct counted { F f; bool operator()(float v) const { tests++; return f(v); } };
template <typename F> static counted<F> count(F f) { return { f }; }
int main(int argc, char ** argv) {      // maxima, or "min_p", a number and a maximum: for each the most floats looked at for a border, and wrong borders
    if (!strcmp(argv[1], "min_p")) {
        const float min_p = strtof(argv[2], nullptr), mx = strtof(argv[3], nullptr);
        const double p = min_p, log_p = log(p);
        auto in = [=](float l) { return sd_enough(l, mx, p, log_p); };
        const float f = sd_least((float) ((double) mx + log_p), mx, count(in));
        printf("%ld %d\n", tests, f != sd_min_p(min_p, mx) || !in(f) || in(sd_of_rank(sd_rank(f) - 1)));
        return 0;
    }
    for (int i = 1; i < argc; i++) {
        const float mx = strtof(argv[i], nullptr);
        long most = 0, wrong = 0;
        for (int b = 0; b < SD_FINE - 1; b++) {
            auto in = [=](float l) { return sd_fine(l, mx) <= b; };
            tests = 0;
            const float f = sd_least(mx - (float) (b + 1) / SD_PER, mx, count(in));
            if (tests > most) most = tests;
            wrong += f != sd_bin_floor(b, mx) || !in(f) || in(sd_of_rank(sd_rank(f) - 1));
        }
        printf("%ld %ld\n", most, wrong + (sd_bin_floor(SD_FINE - 1, mx) != -FLT_MAX));
    }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("border")
    (d / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "pipeinfer_b200", "csrc"), "-o", str(d / "t"), str(d / "t.cpp")], check=True)
    return str(d / "t")


# maxima behind which a bin's edge is exactly 0 (every bfloat16 number from 0.5 on), lies a few ulps beside it, or nowhere near; the ends of the range
MAXIMA = ["3", "5", "8", "20", "7.5", "10", "12.25", "31.75", "0.5", "0.50390625", "9.00390625", "5.000001", "9.123456", "10.3", "0", "-0.0", "1e-45", "1e-30", "0.001", "-0.001", "-1e-38", "-7.25",
          "65536", "1e30", "3.4028234e38", "-3.4028234e38"]


@pytest.mark.parametrize("mx", MAXIMA)
def test_bins(program, mx):
    most, wrong = (int(v) for v in subprocess.run([program, mx], check=True, capture_output=True, text=True, timeout=60).stdout.split())
    assert wrong == 0 and most <= 64


# 1 behind a maximum of 0 (logits less their maximum, rows of zeros, rows with an infinity): every float down to -5e-17 has e^l = 1; a border that lands at or near 0
@pytest.mark.parametrize("min_p", ["1", "0.99999994", "0.999", "0.5", "0.36787945", "0.1", "1e-20", "1e-38", "1e-45"])
@pytest.mark.parametrize("mx", MAXIMA + ["0.69314718", "1.0", "5.9604645e-08"])
def test_min_p(program, min_p, mx):
    tests, wrong = (int(v) for v in subprocess.run([program, "min_p", min_p, mx], check=True, capture_output=True, text=True, timeout=60).stdout.split())
    assert wrong == 0 and tests <= 64
