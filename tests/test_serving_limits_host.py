"""Limits of the serving operators' C ABI that the host checks, no GPU needed
(include/b2g_serving.h)."""
import pytest

from test_serving_capi_host import _attention, _prompt


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -1e-30])
def test_scales_that_are_no_scale_are_refused(capi, scale):
    assert capi.cache_attention(_attention(capi, scale=scale)) == capi.B2G_ERR_INVALID_ARG
    assert _prompt(capi, scale=scale) == capi.B2G_ERR_INVALID_ARG


@pytest.mark.parametrize("dim,heads,tile", [(64, 8, 128), (128, 8, 64), (64, 32, 128), (128, 32, 80)])
def test_tiles_of_all_requests_are_counted_in_32_bits(capi, dim, heads, tile):
    """2 kv heads, blocks of 256 tokens: each request's row of the table holds 2^31 - 2^24 tokens."""
    width = (1 << 23) - (1 << 16)
    most = ((1 << 31) - 1) // -(-width * 256 // tile)

    def ask(requests):
        return _attention(capi, requests=requests, dim=dim, heads=heads, block_size=256, table_width=width,
                          table_ld=width)

    assert capi.cache_attention_workspace_bytes(ask(most)) > 0
    assert capi.cache_attention_workspace_bytes(ask(most + 1)) == -1
    assert capi.cache_attention(ask(most + 1)) == capi.B2G_ERR_UNSUPPORTED


@pytest.mark.parametrize("bad", [dict(table_width=1 << 59, table_ld=1 << 59), dict(table_width=1 << 60, table_ld=1 << 60),
                                 dict(num_blocks=1 << 30, heads=0, kv_heads=1 << 60)])
def test_sizes_whose_products_pass_64_bits_are_refused(capi, bad):
    assert capi.cache_attention(_attention(capi, **bad)) == capi.B2G_ERR_UNSUPPORTED
