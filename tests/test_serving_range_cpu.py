"""The ends of ranges of the operators around a decoder's cache, refused before anything reaches a GPU (the addresses
are no memory): sizes whose product passes 64 bits, a single rotary pair."""
import pytest

import nnr_amd
from nnr_amd import _lib
from test_decode_cpu import MEM
from test_serving_cpu import rotary, rotary_desc

UNSUPPORTED = _lib.NNRH_ERR_UNSUPPORTED


@pytest.mark.parametrize("axis", ["batch", "token"])
@pytest.mark.parametrize("which", ["q", "qy", "k", "ky"])
@pytest.mark.parametrize("n,step", [((1 << 24) + 1, 1 << 38), ((1 << 16) + 3, 1 << 38), ((1 << 24) + 1, (1 << 30) + 64)])
def test_rotary_extents(axis, which, n, step):
    """2^24 steps of 2^38 fp32 elements are 2^64 bytes, which 64 bits hold as 0: the result's rows would seem to share
    nothing with the table."""
    used, kw = which[0], dict(dtype=_lib.F32, batch=1, seq=1, q_heads=0, k_heads=0, head_dim=64)
    kw.update({f"{used}_heads": 1, "batch" if axis == "batch" else "seq": n, f"{used}_{axis}_stride": 64, f"{used}y_{axis}_stride": 64})
    assert rotary(rotary_desc(**{**kw, f"{which}_{axis}_stride": step}), qy=MEM[2], ky=MEM[3]) == UNSUPPORTED


def test_ntk_of_a_single_pair():
    """Its frequency is 1 whatever the base: nothing could be stretched."""
    with pytest.raises(ValueError, match="single pair"):
        nnr_amd.rotary_frequencies(2, scaling="ntk", factor=4.0)
    with pytest.raises(ValueError, match="single pair"):
        nnr_amd.RotaryEmbedding(64, 100, rotary_dim=2, scaling="ntk", factor=4.0, device="cpu")
    assert nnr_amd.rotary_frequencies(2, scaling="ntk", factor=1.0)[0].tolist() == [1.0]
    assert nnr_amd.rotary_frequencies(0, scaling="ntk", factor=4.0)[0].size == 0
    f, m = nnr_amd.rotary_frequencies(4, 10000.0, "ntk", 4.0)
    assert m == 1 and f[0] == 1 and abs(f[1] * 4 * 100 - 1) < 1e-14
