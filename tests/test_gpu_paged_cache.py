"""The paged cache as a user runs it: prompts, tokens, requests that end and
begin (cupilot-kernels_b200/serving.py, examples/paged_serving.py).

Tolerances.  Prompts are attended to in bf16: 2^-7 as for the operator.  A
generated token reads keys and values in 8 bits: int8 steps are 1/127 of a
block's largest value (about 3.5 standard deviations), an error of 3.5 / 127 /
sqrt(12) = 0.8 % of a value's standard deviation in V, and as much again in
the scores through K, so outputs of averaged values stay below 4 %; e4m3 keeps
3 mantissa bits, a relative error up to 2^-4 (rms 2.6 %): below 12 %.
"""
import importlib
import sys

import pytest
import torch

from conftest import REPO, import_pkg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serving():
    return import_pkg("serving")


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, str(REPO / "examples"))
    try:
        return importlib.import_module("paged_serving")
    finally:
        sys.path.pop(0)


@pytest.mark.parametrize("codes,tol", [("int8", 0.04), ("e4m3", 0.12)])
def test_example(example, ops, codes, tol):
    worst = example.main(codes)
    assert worst["prompt"] <= 2.0 ** -7
    assert worst["token"] <= tol
    torch.cuda.synchronize()
    assert ops.read_device_error(torch.cuda.current_device()) == 0


def test_blocks_are_given_out_once_and_come_back(serving):
    c = serving.PagedCache(layers=1, requests=3, max_tokens=64, blocks=8, kv_heads=1, dim=16)
    c.begin([17, 0, 33])
    assert c.free == 3 and c.free_count.item() == 3
    c.begin([15, 1, 0])
    held = [c.block_table[r, :n].tolist() for r, n in enumerate([2, 1, 3])]
    blocks = sum(held, [])
    assert len(set(blocks)) == 6 and all(0 <= b < 8 for b in blocks)
    c.release(2)
    assert c.free == 5 and c.free_count.item() == 5
    assert set(c.free_blocks[:5].tolist()) == set(range(8)) - set(held[0] + held[1])
    c.begin([0, 0, 64])
    again = sum((c.block_table[r, :n].tolist() for r, n in enumerate([2, 1, 4])), [])
    assert len(set(again)) == 7


def test_refusals(serving):
    c = serving.PagedCache(layers=1, requests=2, max_tokens=64, blocks=3, kv_heads=1, dim=16)
    with pytest.raises(RuntimeError, match="begin"):
        c.append(0, torch.zeros(1, 1, 16, device="cuda").half(), torch.zeros(1, 1, 16, device="cuda").half())
    with pytest.raises(ValueError, match="2 values"):
        c.begin([1])
    with pytest.raises(ValueError, match="negative"):
        c.begin([1, -1])
    with pytest.raises(ValueError, match="allows 64"):
        c.begin([65, 0])
    with pytest.raises(RuntimeError, match="3 are free"):
        c.begin([32, 32])
    x = torch.zeros(3, 1, 16, device="cuda").half()
    c.begin([3, 0])
    with pytest.raises(RuntimeError, match="one token a request"):
        c.decode(0, x, x, x)
    c.begin([3, 0])
    with pytest.raises(RuntimeError, match="held no token"):
        c.prefill(0, x, x, x)
    with pytest.raises(ValueError, match="codes"):
        serving.PagedCache(1, 1, 16, 1, 1, 16, codes="int4")
    with pytest.raises(ValueError, match="dim"):
        serving.PagedCache(1, 1, 16, 1, 1, 20)
    with pytest.raises(ValueError, match="block_size"):
        serving.PagedCache(1, 1, 16, 1, 1, 16, block_size=24)


@pytest.mark.parametrize("request_", [-1, 2])
def test_release_of_a_request_that_is_not_there(serving, request_):
    c = serving.PagedCache(layers=1, requests=2, max_tokens=64, blocks=4, kv_heads=1, dim=16)
    c.begin([16, 16])
    with pytest.raises(IndexError, match="from 0 to 1"):
        c.release(request_)
    assert c.free == 2 and c.lengths == [16, 16] and c.lens.tolist() == [16, 16]
    assert c.free_count.item() == 2


def test_refused_steps_leave_the_cache_as_it_was(serving):
    c = serving.PagedCache(layers=1, requests=2, max_tokens=64, blocks=4, kv_heads=1, dim=16)
    x = torch.ones(3, 1, 16, device="cuda").half()
    for call in (c.prefill, c.decode):
        with pytest.raises(RuntimeError, match="begin"):
            call(0, x, x, x)
    c.begin([3, 0])
    with pytest.raises(RuntimeError, match="one token a request"):
        c.decode(0, x, x, x)
    c.begin([3, 0])
    with pytest.raises(RuntimeError, match="held no token"):
        c.prefill(0, x, x, x)
    assert (c.k_cache.view(torch.uint8) == 0).all() and (c.v_scale == 0).all()
