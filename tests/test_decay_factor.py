"""CPU test of the factor that a chain of chunks applies to its state (csrc/rpa_decay_factor.h), compiled for the host."""

import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHUNK, CHAIN = 32, 512

SRC = r"""
#include "rpa_decay_factor.h"
extern "C" void chain(float hi, float lo, int n, float* out) {
  rpa::DecayFactor f;
  f.init(hi, lo);
  for (int i = 0; i < n; ++i) out[i] = f.next();
}
"""


@pytest.fixture(scope="module")
def chain(tmp_path_factory):
    at = tmp_path_factory.mktemp("factor")
    (at / "chain.cc").write_text(SRC)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "easydel_amd", "csrc"), str(at / "chain.cc"), "-o",
                    str(at / "chain.so")], check=True)
    lib = ctypes.CDLL(str(at / "chain.so"))
    lib.chain.argtypes = [ctypes.c_float, ctypes.c_float, ctypes.c_int, ctypes.c_void_p]

    def run(g):
        power = np.exp(np.float64(np.float32(g)) * CHUNK)
        hi = np.float32(power)
        out = np.empty(CHAIN, np.float32)
        lib.chain(hi, np.float32(power - np.float64(hi)), CHAIN, out.ctypes.data)
        return power, out

    return run


def test_every_decay_gives_finite_factors(chain):
    """Over all powers that float32 can hold, subnormal ones (log decays of -2.73 to -3.25) and 0 among them: a factor is off by at
    most two roundings, 2^-23 of itself or a step of the subnormals."""
    for g in np.concatenate([np.linspace(-110.0 / CHUNK, 0.0, 1761), [-2.7, -2.72, -2.74, -2.7726, -2.78, -3.0, -3.2, -3.249, -3.26, -100.0, -1e30]]):
        power, out = chain(g)
        assert np.isfinite(out).all(), g
        assert (np.abs(out.astype(np.float64) - power) <= power * 2.0 ** -23 + 2.0 ** -149).all(), g


def test_the_product_of_a_long_chain_stays_at_the_power(chain):
    """Factor k + 1 makes up for what the product of the first k is off, so that only its own rounding remains: 2^-24, and as much
    again for the arithmetic on the correction (terms of 2^-24, each off by a few 2^-24 of that).  The smaller part of a power near
    the subnormals is itself rounded to their grid, by 2^-150 at most: every factor is off by that over the power (2^-24 in all where
    the power is above 2^-117)."""
    for g in np.concatenate([np.linspace(-2.7, -1e-6, 400), [-1e-9, 0.0]]):
        power, out = chain(g)
        product = np.cumsum(np.log(out.astype(np.float64)))
        steps = np.arange(1, CHAIN + 1)
        assert (np.abs(product - steps * np.log(power)) <= 2.0 ** -23 + steps * 2.0 ** -150 / power + 1e-10).all(), g  # (1e-10: 512 logarithms of up to 87 in 64 bits)
