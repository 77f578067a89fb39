"""Arrays that tierstream_amd.attn refuses as ValueError beside those of test_attn_refusals.py: no GPU is needed."""
import pytest

import tierstream_amd as tsa
from test_attn_refusals import Fake, cache, i32
from tierstream_amd import attn


@pytest.mark.parametrize("k_first", [None, i32(0)])
def test_a_list_of_sequences_has_an_end(k_first):
    q, k = Fake(4, 4, 128), Fake(4, 4, 128)
    with pytest.raises(ValueError, match="first"):
        attn.attend(q, k, k, q, first=i32(0), k_first=k_first)
    with pytest.raises(ValueError, match="first"):
        attn.attend_backward(q, k, k, q, q, Fake(4, 4, dtype="torch.float32"), q, first=i32(0), k_first=k_first)


@pytest.mark.parametrize("bad", [dict(base=5e-324), dict(base=1e-305), dict(factor=1e-305), dict(amplitude=1e39), dict(amplitude=-1e300)])
def test_angles_and_amplitudes_are_numbers(bad):
    """Position 0 times an infinite frequency would be NaN, and an amplitude goes to the products in 32 bits."""
    with pytest.raises(tsa.SsError, match="tsa_rotary_init"):
        attn.Rotary(128, **bad)
    attn.Rotary(128, base=1e-300, amplitude=3e38)


@pytest.mark.parametrize("scale", [1e39, -1e300, float("inf"), float("nan")])
def test_a_scale_beyond_32_bits_is_refused(scale):
    """As a status of the library's, like any other value that it refuses."""
    q, k = Fake(4, 4, 128), Fake(4, 4, 128)
    with pytest.raises(tsa.SsError, match="finite scale"):
        attn.attend(q, k, k, q, scale=scale)
    with pytest.raises(tsa.SsError, match="finite scale"):
        attn.attend_backward(q, k, k, q, q, Fake(4, 4, dtype="torch.float32"), q, scale=scale)
    with pytest.raises(tsa.SsError, match="finite scale"):
        attn.attend_cached(cache(), Fake(4, 8, 128), Fake(4, 8, 128), i32(4, 8), i32(4), i32(5), scale=scale)
