"""Limits of the serving operators' C ABI that the host checks, no GPU needed
(include/b2g_serving.h)."""
import pytest

from test_serving_capi_host import _attention, _prompt


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -1e-30])
def test_scales_that_are_no_scale_are_refused(capi, scale):
    assert capi.cache_attention(_attention(capi, scale=scale)) == capi.B2G_ERR_INVALID_ARG
    assert _prompt(capi, scale=scale) == capi.B2G_ERR_INVALID_ARG
