"""Where hyp_verify_batch's filters end (csrc/verify_border.h, compiled here with the host compiler and run a wave's 64 lanes
at a time): over rows whose running sums and weights meet a border to a few roundings, the border is found and is the
definition's, for a running sum to one token."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def border(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("border") / "border.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-ffp-contract=off", "-U_FORTIFY_SOURCE", "-Wall", "-Wextra", "-Werror",
                    "-Wno-unknown-pragmas", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tests", "host_device"),
                    "-I", os.path.join(ROOT, "hyperion_amd", "csrc"), os.path.join(ROOT, "tests", "verify_border_shim.cc"),
                    "-o", so], check=True)
    return ctypes.CDLL(so)


@pytest.mark.parametrize("seed", range(6))
def test_borders_met_to_a_rounding(border, seed):
    message = ctypes.create_string_buffer(400)
    assert not border.check_borders(ctypes.c_uint64(seed), 4000, message, ctypes.c_size_t(400)), message.value.decode()
