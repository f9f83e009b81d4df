"""Further refusals of the paged-cache calls and their wrappers, before the device is touched."""
import pytest

from test_paged_cpu import _decode, _prompt, _refused


@pytest.mark.parametrize("call", [_decode, _prompt])
def test_scales_that_overflow_as_powers_of_two(call):
    """3e38 is finite, 3e38 log2(e) is not, and infinity times a score of zero is NaN."""
    for scale in (3e38, -3e38, 2.4e38):
        _refused(call(scale=scale), "log2(e)")
    for scale in (2.3e38, -2.3e38, 0.0, 1e-45):
        _refused(call(scale=scale), "null context")
