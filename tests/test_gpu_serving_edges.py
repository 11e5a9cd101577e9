"""Edges of the serving operators: inputs at which a range, a limit or a mask
decides (include/b2g_serving.h), against plain implementations in 64 bits.
Tolerances as in test_gpu_serving.py where none is stated beside the test.
"""
import math
import subprocess
import sys

import pytest
import torch

from conftest import REPO
from test_gpu_serving import (CODES, DTYPES, LSE_TOL, _attend, _close, _codes_of, _dev, _ids, _no_error, _random_cache,
                              _step, _step_state)

pytestmark = pytest.mark.gpu


# ------------------------------------------- cache attention: value scales
@pytest.mark.parametrize("codes", CODES, ids=_ids)
@pytest.mark.parametrize("gap,power", [(120, 28), (200, 28), (130, 110)])
@pytest.mark.parametrize("d,group", [(64, 2), (128, 2), (64, 12), (128, 12)])
def test_blocks_of_zeros_lead_before_large_value_scales(ops, d, group, gap, power, codes):
    """The first blocks lead by 2^gap and hold zeros only (value scale 0); the later ones, with value
    scales of 2^power, are then all of the output: finite, and in range at (130, 110)."""
    g = torch.Generator().manual_seed(d + group + gap)
    # 700 requests share the blocks, so that one warp meets both kinds.
    n, zeros, blocks, reqs = 333, 10, 21, 700
    lead = (torch.arange(blocks) < zeros).view(blocks, 1)
    sign = torch.where(lead, 1.0, -1.0)[:, :, None, None]
    kc = _codes_of(sign * 64 + torch.randint(-8, 9, (blocks, 1, 16, d), generator=g), codes)
    vc, vs = _random_cache(g, blocks, 1, 16, d, codes)
    ks = torch.full((blocks, 1), 1 / 64.0)
    vs = torch.where(lead, 0.0, vs * 2.0 ** power)
    vc = torch.where(lead[:, :, None, None], 0, vc.view(torch.uint8)).view(codes)
    q = torch.full((1, group, d), gap / 2 * math.log(2.0) / d ** 0.5).bfloat16()
    k, v = (c.double() * s.double()[:, :, None, None] for c, s in ((kc, ks), (vc, vs)))
    k, v = (x.transpose(1, 2).reshape(-1, 1, d)[:n] for x in (k, v))
    want, _ = _attend(q.double(), k, v, d ** -0.5)
    want = want.bfloat16().double()              # (2^-172 at gap 200: 0)
    out = ops.cache_attention(q.cuda().repeat(reqs, 1, 1), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(),
                              _dev([list(range(blocks))] * reqs), _dev([n] * reqs))
    assert torch.isfinite(out).all()
    for j in range(group):
        _close(out[:, j], want[:, j].expand(reqs, d), torch.bfloat16)
    _no_error(ops)


# ---------------------------------------------- prompts: values not yet seen
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("h,d", [(1, 64), (1, 128), (60, 64)])
def test_later_values_near_the_types_end_do_not_reach_earlier_rows(ops, h, d, dtype):
    """A masked weight is 0: the largest finite values behind a row change no bit of it."""
    g = torch.Generator().manual_seed(h + d)
    n = 300
    q, k, v = (torch.randn(n, h, d, generator=g).to(dtype).cuda() for _ in range(3))
    cu = _dev([0, n])
    want, lse = ops.prompt_attention(q, k, v, cu, return_lse=True)
    for row in (1, 9, 10, 21, 31, 127, 128, 200, 299):
        big = v.clone()
        big[row:] = torch.finfo(dtype).max
        got, got_lse = ops.prompt_attention(q, k, big, cu, return_lse=True)
        assert torch.equal(got[:row], want[:row])
        assert torch.equal(got_lse, lse)


# ------------------------------------------------ block tables: their limits
_ONE_TOKEN_EACH = """
import importlib, torch
ops = importlib.import_module("cupilot-kernels_b200.ops")
n = {n}
ctx = torch.arange(n, dtype=torch.int32, device="cuda") % 40
table = torch.arange(3 * n, dtype=torch.int32, device="cuda").view(n, 3)
free = 3 * n + torch.arange(n, dtype=torch.int32, device="cuda")
new = torch.ones(n, dtype=torch.int32, device="cuda")
count = torch.full((1,), n, dtype=torch.int32, device="cuda")
slots, cu, lens, left = ops.block_tables(ctx, new, table, free, count, n, 16)
opens = ctx % 16 == 0
at = n - 1 - (opens.int().cumsum(0) - opens.int())
block = torch.where(opens, free[at], table.gather(1, (ctx // 16).long()[:, None])[:, 0])
assert torch.equal(slots, block.long() * 16 + ctx % 16)
assert torch.equal(cu, torch.arange(n + 1, dtype=torch.int32, device="cuda"))
assert torch.equal(lens, ctx + 1) and left.item() == n - opens.sum().item()
assert ops.read_device_error(0) == 0
"""


@pytest.mark.parametrize("n", [4085, 4086, 4095, 4096, 16384])
def test_tables_of_many_requests(ops, n):
    exec(_ONE_TOKEN_EACH.format(n=n), {})


def test_tables_of_4086_requests_first_in_a_process():
    # 48 KB of shared memory together with the kernel's own 128 bytes; no larger call came before
    code = f"import sys\nsys.path.insert(0, {str(REPO)!r})" + _ONE_TOKEN_EACH.format(n=4086)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_tables_of_lengths_that_sum_past_31_bits(ops):
    """Out of the documented range: wrong slots at most, and no entry from beyond the stack."""
    most = (1 << 31) - 1
    free = torch.arange(100, 108, dtype=torch.int32, device="cuda")
    big = torch.full((4, 9), -7, dtype=torch.int32, device="cuda")
    slots, cu, lens, left = ops.block_tables(_dev([0, 5, 0, 40]), _dev([most] * 4), big[:, :6], free, _dev([8]),
                                             64, 16)
    assert (big[:, 6:] == -7).all()
    entries = big[:, :6]
    assert ((entries == -7) | (entries == -1) | ((entries >= 100) & (entries < 108))).all()
    assert slots.shape == (64,) and ((slots >= -1) & (slots < 108 * 16)).all()
    _no_error(ops)


# -------------------------------------------------------------- refused scales
@pytest.mark.parametrize("scale", [1e-60, 1e60, math.inf, math.nan, 0.0])
def test_scales_that_32_bits_do_not_hold_are_refused(ops, scale):
    q = torch.randn(4, 2, 64, device="cuda").half()
    with pytest.raises(RuntimeError, match="scale must be positive"):
        ops.prompt_attention(q, q, q, _dev([0, 4]), scale=scale)
    kc, ks = torch.zeros(2, 2, 16, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, device="cuda")
    with pytest.raises(RuntimeError, match="scale must be positive"):
        ops.cache_attention(q, kc, kc, ks, ks, _dev([[0]] * 4), _dev([1] * 4), scale)


# --------------------------------------------------- key scales that are NaN
@pytest.mark.parametrize("bits", [0xffffffff, 0x7fffffff, 0x7fc00000])
@pytest.mark.parametrize("d", [64, 128])
def test_a_key_scale_of_nan_is_not_a_missing_block(ops, d, bits):
    g = torch.Generator().manual_seed(d)
    kc, ks = _random_cache(g, 4, 1, 16, d, torch.int8)
    ks[2].view(torch.int32)[:] = bits - (1 << 32) if bits >> 31 else bits
    q = torch.randn(2, 2, d, generator=g).half().cuda()
    args = [x.cuda() for x in (kc, kc, ks, torch.ones_like(ks))]
    out, lse = ops.cache_attention(q, *args, _dev([[0, 1], [2, 3]]), _dev([30, 30]), return_lse=True)
    assert torch.isfinite(out[0]).all() and torch.isfinite(lse[0]).all()
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()


# ---------------------------------------------------------------- gradients
def test_a_backward_pass_that_is_not_there_raises(ops):
    """Forward results are the same where an input wants a gradient, which is not lost silently."""
    q, k = (torch.randn(4, h, 64, device="cuda").half() for h in (4, 2))
    kc, ks = torch.zeros(2, 2, 16, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, device="cuda")
    cu, table, lens = _dev([0, 4]), _dev([[0]] * 4), _dev([1] * 4)
    calls = [lambda q, k, lse: ops.prompt_attention(q, k, k, cu, return_lse=lse),
             lambda q, k, lse: ops.cache_attention(q, kc, kc, ks, ks, table, lens, return_lse=lse)]
    for f in calls:
        want = f(q, k, True)
        assert not want[0].requires_grad
        leaf, other = q.clone().requires_grad_(), k.clone().requires_grad_()
        for part in (0, 1):
            got = f(leaf, other, True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            with pytest.raises(RuntimeError, match="no backward pass"):
                got[part].sum().backward()
        with pytest.raises(RuntimeError, match="no backward pass"):
            (f(leaf * 2, other, False).sum() + leaf.sum()).backward()
        assert leaf.grad is None
        for context in (torch.no_grad, torch.inference_mode):
            with context():
                assert not f(leaf, other, False).requires_grad
    with pytest.raises(RuntimeError, match="no backward pass"):
        ops.prompt_attention(q, other, k, cu).sum().backward()


# ------------------------------------------------------------------- C ABI
def test_the_c_entries_give_what_the_torch_entries_give(ops, capi):
    g = torch.Generator(device="cuda").manual_seed(40)
    h, group, d, bs, n = 2, 4, 80, 32, 70
    stream = torch.cuda.current_stream().cuda_stream
    ctx, new = _dev([5, 0]), _dev([30, 40])
    free, count = torch.arange(6, dtype=torch.int32, device="cuda"), _dev([6])
    tables = [_dev([[7, -1, -1], [-1, -1, -1]]) for _ in range(2)]
    want = ops.block_tables(ctx, new, tables[0], free, count, n, bs)
    got = [torch.empty_like(x) for x in want]
    assert capi.block_tables(ctx.data_ptr(), new.data_ptr(), 2, tables[1].data_ptr(), 3, 3, free.data_ptr(), 6,
                             count.data_ptr(), n, bs, *(x.data_ptr() for x in got), stream=stream) == capi.B2G_OK
    assert torch.equal(*tables) and all(torch.equal(a, b) for a, b in zip(got, want))

    q = torch.randn(n, h * group, d, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(n, h, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    caches = [[torch.zeros(8, h, bs, d, dtype=torch.int8, device="cuda") for _ in range(2)]
              + [torch.zeros(8, h, device="cuda") for _ in range(2)] for _ in range(2)]
    slots, cu, lens, _ = want
    ops.cache_append(k, v, slots, *caches[0])
    desc = capi.CacheAppendDesc(capi.BF16, capi.I8, n, h, d, 8, bs, k.data_ptr(), h * d, d, v.data_ptr(), h * d, d,
                                slots.data_ptr(), *(x.data_ptr() for x in caches[1]))
    assert capi.cache_append(desc, stream) == capi.B2G_OK
    assert all(torch.equal(a, b) for a, b in zip(*caches))

    out, lse = ops.cache_attention(q[:2], *caches[0], tables[0], lens, return_lse=True)
    mine, mine_lse = torch.empty_like(out), torch.empty_like(lse)
    kc, vc, ks, vs = caches[0]
    desc = capi.CacheAttentionDesc(capi.BF16, capi.I8, 2, h * group, h, d, 8, bs, q.data_ptr(), h * group * d, d,
                                   kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), tables[0].data_ptr(),
                                   3, 3, lens.data_ptr(), 0.0, mine.data_ptr(), mine_lse.data_ptr(), None, 0)
    assert capi.cache_attention(desc, stream) == capi.B2G_ERR_WORKSPACE
    space = torch.empty(capi.cache_attention_workspace_bytes(desc), dtype=torch.uint8, device="cuda")
    desc.workspace, desc.workspace_bytes = space.data_ptr(), space.numel()
    assert capi.cache_attention(desc, stream) == capi.B2G_OK
    assert torch.equal(mine, out) and torch.equal(mine_lse, lse)

    out, lse = ops.prompt_attention(q, k, v, cu, return_lse=True)
    mine, mine_lse = torch.empty_like(out), torch.empty_like(lse)
    desc = capi.PromptAttentionDesc(capi.BF16, 1, n, n, 2, h * group, h, d, q.data_ptr(), h * group * d, d,
                                    k.data_ptr(), h * d, d, v.data_ptr(), h * d, d, mine.data_ptr(), h * group * d, d,
                                    cu.data_ptr(), None, 0.0, mine_lse.data_ptr())
    assert capi.prompt_attention(desc, stream) == capi.B2G_OK
    assert torch.equal(mine, out) and torch.equal(mine_lse, lse)
    _no_error(ops)


# ------------------------------------------------ cache attention: queries
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("d", [64, 128])
def test_small_values_beside_a_large_one_in_a_query_keep_their_bits(ops, d, dtype):
    # values 2^-22 of the row's largest, which the keys do not see
    codes = torch.float8_e4m3fn
    g = torch.Generator().manual_seed(d)
    n, blocks = 200, 13
    kc, ks = _random_cache(g, blocks, 2, 16, d, codes)
    vc, vs = _random_cache(g, blocks, 2, 16, d, codes)
    kc = torch.where(torch.arange(d) == 3, 0, kc.view(torch.uint8)).view(codes)
    ks = ks * 2.0 ** 13
    q = (torch.randn(1, 8, d, generator=g) * 2.0 ** -12).to(dtype)
    q[:, :, 3] = 2.0 ** 10
    k, v = ((c.double() * s.double()[:, :, None, None]).transpose(1, 2).reshape(-1, 2, d)[:n]
            for c, s in ((kc, ks), (vc, vs)))
    want, want_lse = _attend(q.double(), k, v, d ** -0.5)
    out, lse = ops.cache_attention(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), _dev([list(range(blocks))]),
                                   _dev([n]), None, True)
    _close(out, want, dtype)
    assert (lse.cpu().double() - want_lse).abs().max() <= LSE_TOL


@pytest.mark.parametrize("codes", CODES, ids=_ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_queries_of_any_size_give_the_same_scores(ops, dtype, codes):
    """Powers of two move between the query and the scale: from the type's least normal value to its largest."""
    g = torch.Generator().manual_seed(50)
    kc, ks = _random_cache(g, 7, 2, 16, 64, codes)
    q = torch.randn(1, 8, 64, generator=g).clamp(-3.9, 3.9).to(dtype)
    q = torch.where(q.abs() < 0.25, 0.25, q)
    args = [x.cuda() for x in (kc, kc, ks, ks)] + [_dev([list(range(7))]), _dev([100])]
    want, want_lse = ops.cache_attention(q.cuda(), *args, 0.125, True)
    for power in (-12, 13) if dtype == torch.float16 else (-115, -60, 60, 110, 122):
        out, lse = ops.cache_attention(q.cuda() * 2.0 ** power, *args, 0.125 * 2.0 ** -power, True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("bias", [3.0, 10.0])
def test_log_sums_of_queries_with_a_common_part(ops, bias, dtype):
    """The products add up bias * (code + offset) dim by dim in 32 bits, of which the offset's share is
    taken out: 8 additions, each cut at 2^-23 of sums up to 128 |q|_1 in units of ks * scale."""
    g = torch.Generator().manual_seed(51)
    n, d, blocks = 1000, 128, 63
    kc, _ = _random_cache(g, blocks, 1, 16, d, torch.int8)
    vc, vs = _random_cache(g, blocks, 1, 16, d, torch.int8)
    ks = torch.full((blocks, 1), 0.03)
    q = (torch.randn(1, 4, d, generator=g) + bias).to(dtype)
    k, v = ((c.double() * s.double()[:, :, None, None]).transpose(1, 2).reshape(-1, 1, d)[:n]
            for c, s in ((kc, ks), (vc, vs)))
    want, want_lse = _attend(q.double(), k, v, d ** -0.5)
    out, lse = ops.cache_attention(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), _dev([list(range(blocks))]),
                                   _dev([n]), None, True)
    _close(out, want, dtype)
    cut = 8 * 2.0 ** -23 * 128 * q.double().abs().sum(-1) * 0.03 * d ** -0.5
    assert ((lse.cpu().double() - want_lse).abs() <= cut + 2e-5).all()


# ------------------------------------------------------------ a captured step
def test_a_captured_step_replayed_while_lengths_grow(ops):
    """The lengths and the stack's count come back as new tensors: copied into the captured inputs between
    replays, they make the same steps as calls do."""
    eager, state = _step_state(60), _step_state(60)
    _step(ops, _step_state(61))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(ops, state)
    for _ in range(20):
        want = _step(ops, eager)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        for s, (_, lens, left, *_) in ((eager, want), (state, got)):
            s["lens"].copy_(lens)
            s["count"].copy_(left)
        for s in (eager, state):
            s["q"].mul_(-1.25).clamp_(-8, 8)
            s["k"].mul_(1.125).clamp_(-8, 8)
    _no_error(ops)
