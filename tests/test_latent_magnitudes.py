"""CPU checks: magnitudes that are not finite, or not as a float32, are refused before a launch."""

import ctypes as ct
import math

import pytest

from ascendflow_amd import _native
from tests.test_latent_abi import P, append, rotary


@pytest.mark.parametrize("magnitude", [1e39, -1e300, math.inf, math.nan])
def test_c_entries(magnitude):
    lib = _native.library()
    p = P(16)
    assert lib.launch_apply_rotary(None, p, p, p, p, ct.byref(rotary(magnitude=magnitude))) == -2
    assert lib.launch_append_paged_kv(None, p, None, None, p, p, p, p, p, None, ct.byref(append(magnitude=magnitude))) == -2
