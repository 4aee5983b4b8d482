"""What the paged cache's entry points refuse beside test_paged_cpu.py."""
import pytest

from test_paged_cpu import _args


@pytest.mark.parametrize("scale", [3e38, -3e38, float("inf"), float("nan")])
def test_a_scale_that_is_not_finite_in_base_2_is_refused(scale):
    """Logits are taken times log2(e): the largest 32-bit numbers leave the range there, and 0 times an infinity is no logit."""
    from kch_b200 import _lib
    a = _args(_lib, ws_bytes=1 << 40)
    a.scale = scale
    with pytest.raises(ValueError, match="scale"):
        _lib.check(_lib.load().kch_paged_attend(a, None))
