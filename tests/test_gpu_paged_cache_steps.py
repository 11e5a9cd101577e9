"""Steps of the paged cache (cupilot-kernels_b200/serving.py) in which some
requests, or none, gain tokens, and steps that are taken back."""
import pytest
import torch

from conftest import import_pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serving():
    return import_pkg("serving")


def _qkv(n, heads=2, kv_heads=1, dim=32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, h, dim, generator=g, device="cuda").half() for h in (heads, kv_heads, kv_heads)]


def _cache(serving, **kw):
    return serving.PagedCache(**{**dict(layers=2, requests=3, max_tokens=64, blocks=8, kv_heads=1, dim=32), **kw})


def test_a_step_in_which_no_request_gains_a_token(serving):
    c = _cache(serving)
    c.begin([3, 0, 20])
    c.prefill(0, *_qkv(23))
    step = c.begin([0, 0, 0])
    assert step.slots.numel() == 0 and c.lengths == [3, 0, 20]
    q, k, v = _qkv(0)
    for layer in range(2):
        assert c.decode(layer, q, k, v).shape == (0, 2, 32)
    assert c.prefill(0, q, k, v).shape == (0, 2, 32)
    c.begin([1, 0, 1])
    assert torch.isfinite(c.decode(0, *_qkv(2, seed=1))).all()


def test_the_requests_that_gain_a_token_are_the_ones_attended_for(serving, ops):
    c = _cache(serving)
    for layer in range(2):
        if layer == 0:
            c.begin([17, 5, 30])
        c.prefill(layer, *_qkv(52, seed=layer))
    step = c.begin([1, 0, 1])
    for layer in range(2):
        q, k, v = _qkv(2, seed=5 + layer)
        got = c.decode(layer, q, k, v)
        rows = torch.tensor([0, 2], device="cuda")
        want = ops.cache_attention(q, c.k_cache[layer], c.v_cache[layer], c.k_scale[layer], c.v_scale[layer],
                                   c.block_table[rows], step.seq_lens[rows])
        assert torch.equal(got, want)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_a_step_that_is_taken_back_leaves_no_token(serving, codes):
    """A step that prefill() and decode() refuse, or that is not wanted any more: the cache goes on as
    if it had not been begun."""
    caches = [_cache(serving, codes=codes) for _ in range(2)]
    outs = []
    for c, mixed in zip(caches, (False, True)):
        c.begin([17, 0, 30])
        c.prefill(0, *_qkv(47))
        if mixed:
            before = (c.lengths, c.free, c.lens.tolist(), c.free_count.item())
            c.begin([1, 20, 1])                       # a prompt among running requests
            with pytest.raises(RuntimeError, match="one token a request"):
                c.decode(0, *_qkv(22, seed=3))
            with pytest.raises(RuntimeError, match="held no token"):
                c.prefill(0, *_qkv(22, seed=3))
            c.cancel()
            assert (c.lengths, c.free, c.lens.tolist(), c.free_count.item()) == before
            with pytest.raises(RuntimeError, match="begin"):
                c.decode(0, *_qkv(2))
        c.begin([1, 0, 1])
        outs.append(c.decode(0, *_qkv(2, seed=4)))
        c.begin([0, 20, 0])
        outs.append(c.prefill(0, *_qkv(20, seed=5)))
        c.begin([1, 1, 1])
        outs.append(c.decode(0, *_qkv(3, seed=6)))
        c.release(2)
        assert sorted(c.free_blocks[:c.free].tolist() + c.block_table[0, :2].tolist()
                      + c.block_table[1, :2].tolist()) == list(range(8))
    assert all(torch.equal(a, b) for a, b in zip(outs[:3], outs[3:]))


def test_cancel_wants_a_step(serving):
    c = _cache(serving)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="begin"):
            c.cancel()
        c.begin([1, 0, 0])
        c.cancel()
    c.begin([16, 0, 0])
    c.release(0)
    with pytest.raises(RuntimeError, match="begin"):
        c.cancel()
    assert c.free == 8 and c.free_count.item() == 8
