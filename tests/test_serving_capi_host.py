"""The serving operators' C ABI on the host: struct layouts, argument checks and
workspace sizes (include/b2g_serving.h), no GPU needed."""
import ctypes

import pytest
import torch

ADDR = 1 << 20      # a fake 16-byte-aligned device address: the checks never dereference


def _append(capi, **kw):
    d = capi.CacheAppendDesc(capi.BF16, capi.I8, 4, 2, 64, 8, 16, ADDR, 128, 64, ADDR, 128, 64, ADDR, ADDR,
                             ADDR, ADDR, ADDR)
    for k, v in kw.items():
        setattr(d, k, v)
    return capi.cache_append(d)


def _attention(capi, **kw):
    d = capi.CacheAttentionDesc(capi.F16, capi.E4M3, 3, 8, 2, 64, 10, 16, ADDR, 512, 64, ADDR, ADDR, ADDR, ADDR,
                                ADDR, 5, 5, ADDR, 0.0, ADDR, 0, ADDR, 1 << 30)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _prompt(capi, **kw):
    d = capi.PromptAttentionDesc(capi.F16, 1, 100, 100, 2, 8, 2, 64, ADDR, 512, 64, ADDR, 128, 64, ADDR, 128, 64,
                                 ADDR, 512, 64, ADDR, 0, 0.0, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return capi.prompt_attention(d)


def _tables(capi, **kw):
    a = dict(context_lens=ADDR, new_lens=ADDR, requests=3, block_table=ADDR, table_width=4, table_ld=4,
             free_blocks=ADDR, free_capacity=10, free_count=ADDR, total_tokens=7, block_size=16, slots=ADDR,
             cu_seqlens=ADDR, seq_lens=ADDR, free_count_out=ADDR)
    a.update(kw)
    return capi.block_tables(**a)


def test_struct_layouts_match_the_header(capi):
    assert ctypes.sizeof(capi.CacheAppendDesc) == 8 + 5 * 8 + 2 * 24 + 5 * 8
    assert ctypes.sizeof(capi.CacheAttentionDesc) == 8 + 6 * 8 + 24 + 4 * 8 + 24 + 8 + 8 + 2 * 8 + 16
    assert ctypes.sizeof(capi.PromptAttentionDesc) == 8 + 6 * 8 + 4 * 24 + 2 * 8 + 8 + 8


@pytest.mark.parametrize("bad", [dict(requests=-1), dict(table_ld=3), dict(free_capacity=-1), dict(total_tokens=-1),
                                 dict(block_size=24), dict(free_count=0), dict(slots=0), dict(context_lens=0),
                                 dict(block_table=0), dict(free_blocks=0), dict(cu_seqlens=0)])
def test_tables_refuse(capi, bad):
    assert _tables(capi, **bad) == capi.B2G_ERR_INVALID_ARG


def test_tables_limits(capi):
    assert _tables(capi, requests=capi.MAX_TABLE_REQUESTS + 1) == capi.B2G_ERR_UNSUPPORTED
    assert _tables(capi, total_tokens=1 << 31) == capi.B2G_ERR_UNSUPPORTED


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(dtype=7), dict(codes=3), dict(dim=0), dict(block_size=48),
                                 dict(k=0), dict(slots=0), dict(v_scale=0)])
def test_append_refuses(capi, bad):
    assert _append(capi, **bad) == capi.B2G_ERR_INVALID_ARG


@pytest.mark.parametrize("bad", [dict(dim=72), dict(dim=256), dict(block_size=8), dict(block_size=512),
                                 dict(k_token_stride=129), dict(v_head_stride=4), dict(k=ADDR + 8),
                                 dict(v_cache=ADDR + 4)])
def test_append_limits(capi, bad):
    assert _append(capi, **bad) == capi.B2G_ERR_UNSUPPORTED


@pytest.mark.parametrize("bad", [dict(requests=-1), dict(heads=7), dict(kv_heads=0), dict(dtype=2), dict(codes=-1),
                                 dict(table_ld=4), dict(scale=-1.0), dict(scale=float("nan"))])
def test_attention_refuses(capi, bad):
    d = _attention(capi, **bad)
    assert capi.cache_attention_workspace_bytes(d) == -1
    assert capi.cache_attention(d) == capi.B2G_ERR_INVALID_ARG


@pytest.mark.parametrize("bad", [dict(dim=40), dict(dim=144), dict(block_size=12), dict(block_size=1024),
                                 dict(num_blocks=1 << 31), dict(table_width=1 << 40, table_ld=1 << 40)])
def test_attention_limits(capi, bad):
    assert capi.cache_attention(_attention(capi, **bad)) == capi.B2G_ERR_UNSUPPORTED


def test_attention_workspace(capi):
    d = _attention(capi)
    need = capi.cache_attention_workspace_bytes(d)
    assert 0 < need < 64 << 20
    assert capi.cache_attention_workspace_bytes(_attention(capi, requests=0)) == 0
    assert capi.cache_attention_workspace_bytes(_attention(capi, requests=300, table_width=4000, table_ld=4000)) >= need
    for bad in (dict(q=0), dict(out=0), dict(seq_lens=0), dict(block_table=0), dict(k_cache=0), dict(k_scale=0)):
        assert capi.cache_attention(_attention(capi, **bad)) == capi.B2G_ERR_INVALID_ARG


@pytest.mark.parametrize("bad", [dict(tokens=-1), dict(heads=9), dict(kv_heads=0), dict(dtype=5), dict(scale=-0.5),
                                 dict(q=0), dict(k=0), dict(cu_q=0), dict(tokens_k=50)])
def test_prompt_refuses(capi, bad):
    assert _prompt(capi, **bad) == capi.B2G_ERR_INVALID_ARG


@pytest.mark.parametrize("bad", [dict(dim=136), dict(dim=24), dict(heads=512, kv_heads=2), dict(q_token_stride=513),
                                 dict(out_head_stride=-64), dict(v=ADDR + 2), dict(tokens=1 << 31, tokens_k=1 << 31)])
def test_prompt_limits(capi, bad):
    assert _prompt(capi, **bad) == capi.B2G_ERR_UNSUPPORTED


def test_empty_calls_need_no_device(capi):
    assert _append(capi, tokens=0) == capi.B2G_OK
    assert capi.cache_attention(_attention(capi, requests=0)) == capi.B2G_OK
    assert _prompt(capi, tokens=0, tokens_k=0) == capi.B2G_OK


def test_without_gpu_reports_no_device(capi):
    if torch.cuda.is_available():
        pytest.skip("host-only check")
    assert _tables(capi) == capi.B2G_ERR_NO_DEVICE
    assert _append(capi) == capi.B2G_ERR_NO_DEVICE
    assert capi.cache_attention(_attention(capi)) == capi.B2G_ERR_NO_DEVICE
    assert _prompt(capi) == capi.B2G_ERR_NO_DEVICE
