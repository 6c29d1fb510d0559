"""CPU checks: calls that would need more threads than a launch counts are rejected before it."""

import ctypes as ct

from ascendflow_amd import _native
from tests.test_latent_abi import P, expanded, latent


def test_more_workgroups_than_a_launch_holds():
    lib = _native.library()
    args = [None] + [P(16)] * 7 + [None, P(16), 1 << 40]
    for changes in (dict(B=200000, H=128, Tq=200000, Tk=200000), dict(B=1 << 24, H=1, Tq=1 << 24, Tk=1 << 24)):
        assert lib.launch_latent_attention_expanded(*args, ct.byref(expanded(**changes))) == -2
    for changes in (dict(B=1 << 24, H=1, T=1 << 24), dict(B=10_000_000, H=65, T=10_000_000)):
        assert lib.launch_latent_attention(*args, ct.byref(latent(**changes))) == -2
