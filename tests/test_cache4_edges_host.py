"""The 4-bit cache on the CPU: what its kernels check for themselves, compiled for the host, and refusals."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from ring_attention_b200._lib import lib
from tests.test_cache4_host import ROOT, _cache


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


@pytest.mark.parametrize("name", ["k", "v", "k_limits", "v_limits", "positions", "weights", "lengths", "seen"])
def test_an_eviction_into_a_cache_that_shares_an_array_is_refused(name):
    """All arrays of `out` are the cache's own (in place, the same capacity), or none."""
    names = ["k", "v", "k_limits", "v_limits", "positions", "weights", "lengths", "seen"]
    other = {x: 0x100000 + 0x1000 * i for i, x in enumerate(names)}
    assert all(v != getattr(_cache(), x) for x, v in other.items())
    one = C.c_void_p(0x1000)
    shares_one = {**other, name: getattr(_cache(), name)}
    all_but_one = {name: other[name]}
    for arrays in (shares_one, all_but_one):
        assert lib.ra_cache4_evict(C.byref(_cache()), 8, 0, C.byref(_cache(**arrays)), one, 1 << 40, None) == -72
    assert lib.ra_cache4_evict(C.byref(_cache()), 8, 0, C.byref(_cache(capacity=192)), one, 1 << 40, None) == -72
