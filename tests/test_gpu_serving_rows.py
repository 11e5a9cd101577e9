"""Attention of the serving operators element by element, in the shapes where a
CTA's work items hold two tiles and where they hold one.

The bound of an element.  With w the softmax weights in 64 bits and A = sum w |v|:
  - each weight is rounded to 16 bits before the second product, an error of
    u_w w (u_w = 2^-11 in fp16, 2^-8 in bf16; the cache attention's weights are
    fp16 for both types), below 2^-14 of the largest of 2^-25 times the largest
    (the cache attention: 2^-21 and 2^-32, times value scales within a factor of 4);
  - exponentials and scores in 32 bits: 2^-12 w (7.5e-5 at most for the
    polynomial of bf16 prompts, the rest for scores up to 40); int8 scores are
    differences of sums up to 1152 * 128 in 32 bits: 2^-11 w in all;
  - the result is rounded once more to q's type: u |out|.
Together (u_w + slack) A + tail + u |out|, the worst case of each.
"""
import math

import pytest
import torch

from test_gpu_serving import CODES, DTYPES, _codes_of, _dev, _ids, _no_error, _random_cache

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _bounded(q, k, v, scale, seen, u_w, u_out, slack, below):
    """Output in 64 bits and the bound: q (n, heads, d), k, v (m, kv_heads, d), seen (n, m) or None."""
    group = q.shape[1] // k.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for j in range(q.shape[1]):
        z = q[:, j] @ k[:, j // group].T * scale
        if seen is not None:
            z = z.masked_fill(~seen, -math.inf)
        top = z.amax(-1, keepdim=True)
        p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
        l = p.sum(-1, keepdim=True)
        inv = torch.where(l > 0, 1 / l, 0.0)
        vj = v[:, j // group]
        out[:, j] = p @ vj * inv
        there = torch.ones_like(p) if seen is None else seen.double()
        bound[:, j] = ((u_w + slack) * (p @ vj.abs()) + below * (there @ vj.abs())) * inv
    return out, bound + u_out * out.abs()


def _check(got, want, bound):
    over = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all()
    assert over.max() <= 0, f"{over.max().item():.2e} beyond the bound"


def _two_tiles(tokens, sequences, group, kv_heads):
    """Whether work items hold two tiles of 128 / group tokens: one only where that leaves no more items
    than SMs."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return (tokens // (128 // group) + sequences) * kv_heads > sms


def _prompts(ops, lens, h, group, d, dtype, lens_k=None, causal=True, scale=None, q_scale=1.0, two=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    own_k = lens_k is not None
    lens_k = lens_k if own_k else lens
    assert _two_tiles(sum(lens), len(lens), group, h) == two
    q = (torch.randn(sum(lens), h * group, d, generator=g, device="cuda") * q_scale).to(dtype)
    k, v = (torch.randn(sum(lens_k), h, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    cu, cuk = ([sum(x[:i]) for i in range(len(x) + 1)] for x in (lens, lens_k))
    got = ops.prompt_attention(q, k, v, _dev(cu), _dev(cuk) if own_k else None, causal, scale)
    below = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for s, (n, m) in enumerate(zip(lens, lens_k)):
        if n == 0:
            continue
        rows, keys = slice(cu[s], cu[s + 1]), slice(cuk[s], cuk[s + 1])
        if m == 0:
            assert (got[rows] == 0).all()
            continue
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if causal:
            seen = torch.arange(m, device="cuda")[None, :] <= torch.arange(n, device="cuda")[:, None] + m - n
        want, bound = _bounded(q[rows].double(), k[keys].double(), v[keys].double(), scale or d ** -0.5, seen,
                               UNIT[dtype], UNIT[dtype], 2.0 ** -12, below)
        _check(got[rows], want, bound)
    _no_error(ops)
    return q, k, v, got


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("d", [16, 64, 80, 128])
@pytest.mark.parametrize("h,group", [(8, 2), (16, 1), (8, 3), (8, 7), (4, 16)], ids=_ids)
def test_prompt_rows_of_two_tiles(ops, h, group, d, dtype):
    _prompts(ops, [1100, 0, 513, 130, 1], h, group, d, dtype, seed=h + group + d)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("group", [9, 11, 13, 15])
def test_prompt_rows_of_groups_from_9_to_15(ops, group, dtype):
    _prompts(ops, [300, 77, 1], 1, group, 128, dtype, seed=group, two=False)
    _prompts(ops, [300, 77, 1], 8, group, 64, dtype, seed=group)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_prompt_rows_of_one_tile(ops, dtype):
    _prompts(ops, [2500, 1111], 1, 2, 128, dtype, two=False)
    _prompts(ops, [900], 1, 1, 64, dtype, two=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_of_two_tiles_masks(ops, d, dtype):
    # not causal, with keys of their own or not; chunks of longer prompts; rows that see nothing
    _prompts(ops, [3, 900, 257], 8, 4, d, dtype, causal=False, seed=1)
    _prompts(ops, [3, 900, 257], 8, 4, d, dtype, lens_k=[1200, 1, 129], causal=False, seed=2)
    _prompts(ops, [640, 1, 200, 130], 8, 4, d, dtype, lens_k=[1500, 77, 200, 131], seed=3)
    _prompts(ops, [700, 300, 100, 5], 8, 4, d, dtype, lens_k=[300, 10, 0, 5], seed=4)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_prompt_rows_of_two_tiles_peaked(ops, dtype):
    _prompts(ops, [1100, 40], 8, 2, 128, dtype, seed=5, q_scale=8.0)
    _prompts(ops, [1100, 40], 8, 2, 64, dtype, seed=6, scale=1.0)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_of_two_tiles_rising(ops, d):
    """Every key tile brings a new maximum: O is rescaled at each one, in both tiles."""
    n, h = 1100, 24
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k = (torch.zeros(n, h, d, device="cuda").half() for _ in range(2))
    q[:, :, 0] = 1
    k[:, :, 0] = (torch.arange(n, device="cuda") / 32.0)[:, None]
    v = torch.randn(n, h, d, generator=g, device="cuda").half()
    assert _two_tiles(n, 1, 1, h)
    got = ops.prompt_attention(q, k, v, _dev([0, n]), scale=1.0)
    seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    want, bound = _bounded(q.double(), k.double(), v.double(), 1.0, seen, UNIT[torch.float16], UNIT[torch.float16],
                           2.0 ** -12, 2.0 ** -25)
    _check(got, want, bound)
    _no_error(ops)


def test_prompt_two_tiles_neighbours_do_not_leak(ops):
    g = torch.Generator(device="cuda").manual_seed(8)
    n, h = 700, 24
    q, k, v = (torch.randn(n, h, 64, generator=g, device="cuda").half() for _ in range(3))
    cu = _dev([0, 330, 470, n])
    assert _two_tiles(n, 3, 1, h)
    want = ops.prompt_attention(q, k, v, cu)
    for bad in (math.inf, -math.inf, math.nan):
        for there in (slice(330, None), slice(0, 330), slice(330, 470)):
            k2, v2 = k.clone(), v.clone()
            k2[there], v2[there] = bad, bad
            got = ops.prompt_attention(q, k2, v2, cu)
            keep = torch.ones(n, dtype=torch.bool, device="cuda")
            keep[there] = False
            assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype,tol", [(torch.float16, 1.5e-5), (torch.bfloat16, 9e-5)], ids=_ids)
@pytest.mark.parametrize("column", [0, 10, 20, 30, 43, 127])
def test_log_sums_of_one_heavy_key(ops, column, dtype, tol):
    """The log sum is the heavy key's score but for e^-40: its exponential's error shows.  A part of the
    columns goes through a polynomial of relative error 7.5e-5 in bf16 and 2.6e-6 in fp16; beside it
    four roundings of the score, 40 * 2^-24 each."""
    q = torch.zeros(1, 1, 64, device="cuda", dtype=dtype)
    k, v = (torch.zeros(200, 1, 64, device="cuda", dtype=dtype) for _ in range(2))
    q[0, 0, 0], k[column, 0, 0] = 1, 40
    _, lse = ops.prompt_attention(q, k, v, _dev([0, 1]), _dev([0, 200]), scale=1.0, return_lse=True)
    assert abs(lse.item() - 40) <= tol


# ------------------------------------------------------------ one token each
def _tokens(ops, lens, h, group, d, bs, dtype, codes, q=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // bs) for n in lens]
    order = torch.randperm(sum(counts) + 2, generator=g)
    kc, ks = _random_cache(g, len(order), h, bs, d, codes)
    vc, vs = _random_cache(g, len(order), h, bs, d, codes)
    table = torch.full((len(lens), max(counts + [1])), -1, dtype=torch.int32)
    if q is None:
        q = torch.randn(len(lens), h * group, d, generator=g)
    q = q.to(dtype).cuda()
    at = 0
    for r, n in enumerate(counts):
        table[r, :n] = order[at:at + n]
        at += n
    kc, vc, ks, vs, table = (x.cuda() for x in (kc, vc, ks, vs, table))
    got = ops.cache_attention(q, kc, vc, ks, vs, table, _dev(lens))
    slack = 2.0 ** -11 if codes == torch.int8 else 2.0 ** -12
    for r, n in enumerate(lens):
        if n == 0:
            assert (got[r] == 0).all()
            continue
        ids = table[r, :counts[r]].long()
        k, v = ((c.view(torch.uint8)[ids].view(codes).double() * s[ids].double()[:, :, None, None])
                .transpose(1, 2).reshape(-1, h, d)[:n] for c, s in ((kc, ks), (vc, vs)))
        want, bound = _bounded(q[r:r + 1].double(), k, v, d ** -0.5, None, 2.0 ** -11, UNIT[dtype], slack, 2.0 ** -30)
        _check(got[r:r + 1], want, bound)
    _no_error(ops)


@pytest.mark.parametrize("codes", CODES, ids=_ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("h,group,d,bs", [(1, 1, 64, 16), (8, 4, 128, 16), (2, 9, 80, 32), (3, 16, 64, 64),
                                          (2, 13, 128, 128), (1, 40, 112, 256)], ids=_ids)
def test_token_rows(ops, h, group, d, bs, dtype, codes):
    _tokens(ops, [1, 0, 15, 64, 129, 700, 5000], h, group, d, bs, dtype, codes, seed=h + group + d)
    _tokens(ops, [97 * i % 500 for i in range(120)], h, group, d, bs, dtype, codes, seed=h + group)
