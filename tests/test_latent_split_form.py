"""CPU checks of split_form_latent_attention."""

import ctypes as ct

import pytest

from ascendflow_amd import _native
from tests.test_latent_abi import latent


@pytest.mark.parametrize("sizes,form", [
    (dict(T=1, B=1, H=64), [0, 16]),
    (dict(T=64, B=64, H=128, BLOCKS=1000), [1, 1]),    # 147 MB of cache, a tile a request
    (dict(T=64, B=64, H=128, BLOCKS=800), [0, 1]),     # 118 MB
    (dict(T=64, B=1, H=128, BLOCKS=1000), [0, 1]),     # 64 tiles read the same rows
    (dict(T=2000, B=1, H=128, BLOCKS=1000), [0, 0]),   # a tile a workgroup
])
def test_forms(sizes, form):
    got = (ct.c_int64 * 2)()
    lib = _native.library()
    assert lib.split_form_latent_attention(got, ct.byref(latent(**sizes))) == 0 and list(got) == form
    assert lib.split_form_latent_attention(None, ct.byref(latent())) == -1
    assert lib.split_form_latent_attention(got, None) == -1 and lib.split_form_latent_attention(got, ct.byref(latent(L=100))) == -2
