"""The 4-bit cache on the CPU: what its kernels check for themselves, compiled for the host, and refusals."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from tests.test_cache4_host import ROOT


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("shim") / "cache4_note_shim.so")
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "ring_attention_b200", "csrc"), os.path.join(ROOT, "tests", "host_shim", "cache4_note_shim.cpp"),
                    "-o", out], check=True, capture_output=True)
    return C.CDLL(out)


def test_parts_are_read_within_the_workspace_whatever_an_item_s_note_holds(shim):
    """A note that was never written (a wait ran out) is followed only where every part it names is one of the launch's."""
    rng = np.random.default_rng(0)
    words = [-(2**31), -1, 0, 1, 7, 147, 148, 295, 296, 2**31 - 1, *rng.integers(-(2**31), 2**31, 200).tolist()]
    for ctas in (1, 148, 296):
        for first in words:
            for last in words:
                assert bool(shim.ra_host_cache_note_holds(first, last, ctas)) == (0 <= first <= last < ctas)
