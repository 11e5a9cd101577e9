"""The serving operators (include/b2g_serving.h) against plain implementations
in 64 bits: block tables and slot map, the quantising cache write, the
attention of one token over the 8-bit cache, causal attention of packed
prompts.

Tolerances.  Integers, codes and scales are defined by fp32 operations that
the oracle repeats: they have to be equal.  Attention outputs: the weights
enter the second product in 16 bits (relative rounding 2^-11 in fp16, 2^-8 in
bf16, at random signs) and the result is rounded once more to q's type, so the
relative Frobenius error stays below 2 * 2^-11 (fp16; the cache attention's
weights are fp16 for both types) and 2 * 2^-8 (bf16).  An output of few values
may sit at the worst case of both roundings, which the same bounds cover.  Log
sums are fp32 sums of exponentials with relative error 2^-20: 1e-4 absolute
(natural logarithm, |z| < 100).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
LSE_TOL = 1e-4
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
DTYPES = [torch.float16, torch.bfloat16]
CODES = [torch.int8, torch.float8_e4m3fn]


def _ids(x):
    return str(x).replace("torch.", "") if not isinstance(x, (list, tuple)) else "x".join(map(str, x))


def _dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _no_error(ops):
    torch.cuda.synchronize()
    assert ops.read_device_error(torch.cuda.current_device()) == 0


def _close(out, ref, dtype):
    assert torch.isfinite(out).all()
    d = (out.double().cpu() - ref).norm() / max(ref.norm().item(), 1e-30)
    assert d <= TOL[dtype], f"relative error {d:.2e}"


# ------------------------------------------------------------ block tables
def _tables_oracle(ctx, new, table, free, count, total, bs):
    table, width = table.copy(), table.shape[1]
    slots, cu, need = [], [0], 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        held, full = min(-(-c // bs), width), min(-(-(c + n) // bs), width)
        for j in range(held, full):
            at = count - 1 - need
            table[r, j] = free[at] if at >= 0 else -1
            need += 1
        for pos in range(c, c + n):
            j = pos // bs
            b = table[r, j] if j < width else -1
            slots.append(int(b) * bs + pos % bs if b >= 0 else -1)
        cu.append(cu[-1] + n)
    slots = (slots + [-1] * total)[:total]
    lens = [max(c, 0) + max(n, 0) for c, n in zip(ctx, new)]
    return table, slots, cu, lens, count - need


def _tables_case(ops, ctx, new, width, bs, count=None, total=None, pitch=0):
    rng = np.random.default_rng(len(ctx) + width)
    held = [min(-(-max(c, 0) // bs), width) for c in ctx]
    need = sum(-(-(max(c, 0) + max(n, 0)) // bs) for c, n in zip(ctx, new))
    order = rng.permutation(sum(held) + need + 5).astype(np.int32)
    table = np.full((len(ctx), width), -7, np.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        at += h
    free = order[at:]
    count = len(free) if count is None else count
    total = sum(max(n, 0) for n in new) if total is None else total
    big = torch.full((len(ctx), width + pitch), -7, dtype=torch.int32, device="cuda")
    t = big[:, :width]
    t.copy_(torch.from_numpy(table))
    ft = torch.from_numpy(free.copy()).cuda()
    slots, cu, lens, left = ops.block_tables(_dev(ctx), _dev(new), t, ft, _dev([count]), total, bs)
    want = _tables_oracle(ctx, new, table, free, count, total, bs)
    assert np.array_equal(t.cpu().numpy(), want[0])
    assert slots.cpu().tolist() == want[1] and slots.dtype == torch.int64
    assert cu.cpu().tolist() == want[2] and lens.cpu().tolist() == want[3]
    assert left.cpu().tolist() == [want[4]]
    assert (big[:, width:] == -7).all()


@pytest.mark.parametrize("bs", [16, 32, 128, 256])
@pytest.mark.parametrize("reqs,hi", [(1, 1), (1, 700), (3, 40), (33, 17), (600, 5), (1500, 3)])
def test_tables(ops, reqs, hi, bs):
    rng = np.random.default_rng(reqs * hi + bs)
    ctx = rng.integers(0, 900, reqs).tolist()
    new = rng.integers(0, hi + 1, reqs).tolist()
    _tables_case(ops, ctx, new, 1700 // bs + 2, bs, pitch=reqs % 3)


def test_tables_one_token_each(ops):
    _tables_case(ops, [0, 15, 16, 17, 31, 32], [1] * 6, 4, 16)


def test_tables_edges(ops):
    _tables_case(ops, [5, 0, 16, 0], [0, 0, 0, 0], 3, 16)            # nothing new
    _tables_case(ops, [0, 0, 7], [0, 33, 0], 4, 16)                  # empty requests around one
    _tables_case(ops, [-3, 4], [5, -2], 3, 16)                       # negative lengths count as 0
    _tables_case(ops, [30, 3], [40, 2], 3, 16)                       # a row too short
    _tables_case(ops, [10, 20, 30], [50, 50, 50], 8, 16, count=5)    # too few free blocks
    _tables_case(ops, [10, 20], [50, 50], 8, 16, count=0)
    _tables_case(ops, [1, 2], [3, 4], 2, 16, total=20)               # padded rows
    _tables_case(ops, [1, 2], [30, 40], 4, 16, total=33)             # fewer rows than tokens


def test_tables_no_requests(ops):
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    slots, cu, lens, left = ops.block_tables(e, e, e.view(0, 4), _dev([1, 2]), _dev([2]), 3, 16)
    assert slots.tolist() == [-1] * 3 and cu.tolist() == [0] and lens.numel() == 0
    assert left.tolist() == [2]


# ------------------------------------------------------------- cache write
def _codes_of(x, dtype):
    """fp32 values in steps of the scale to codes: nearest even, infinities to the ends, NaN to 0
    (int8) or NaN (e4m3)."""
    q = QMAX[dtype]
    if dtype == torch.int8:
        return torch.nan_to_num(x, nan=0.0, posinf=q, neginf=-q).round().clamp(-q, q).to(torch.int8)
    return x.clamp(-q, q).to(dtype)


def _append_oracle(x, slots, cache, scale):
    """Group by group, head by head, in fp32 (CPU tensors, changed in place)."""
    n, h, bs, _ = cache.shape
    q = torch.tensor(QMAX[cache.dtype])
    t = 0
    while t < len(slots):
        s = slots[t]
        if s < 0 or s >= n * bs:
            t += 1
            continue
        e = t + 1
        while e < len(slots) and slots[e] == slots[e - 1] + 1 and slots[e] % bs:
            e += 1
        b, fill = s // bs, s % bs
        for i in range(h):
            v = x[t:e, i].float()
            fine = v[torch.isfinite(v)].abs()
            amax = fine.max() if fine.numel() else torch.tensor(0.0)
            old = scale[b, i].clone() if fill else torch.tensor(0.0)
            now = torch.maximum(old, amax * (1.0 / q))
            steps = (1.0 / now).clamp(max=3.4028234e38) if now > 0 else torch.tensor(0.0)
            if fill and now > old:
                cache[b, i, :fill] = _codes_of(cache[b, i, :fill].float() * (old / now), cache.dtype)
            y = v * steps
            y = torch.where(torch.isinf(v), v, y)
            cache[b, i, fill:fill + e - t] = _codes_of(y, cache.dtype)
            scale[b, i] = now
        t = e


def _bits(t):
    return t.view(torch.uint8).cpu()


def _random_cache(g, n, h, bs, d, dtype):
    x = torch.randn(n, h, bs, d, generator=g) * QMAX[dtype] / 3.5
    return _codes_of(x, dtype), torch.rand(n, h, generator=g) * 0.02 + 0.01


def _append_case(ops, k, v, slots, n, bs, codes, seed=0):
    g = torch.Generator().manual_seed(seed)
    h, d = k.shape[1:]
    state = []
    for x in (k, v):
        cache, scale = _random_cache(g, n, h, bs, d, codes)
        state.append((x, cache, scale, cache.cuda(), scale.cuda()))
    ops.cache_append(k.cuda() if not k.is_cuda else k, v.cuda() if not v.is_cuda else v,
                     _dev(slots, torch.int64), state[0][3], state[1][3], state[0][4], state[1][4])
    torch.cuda.synchronize()
    for x, cache, scale, dc, ds in state:
        _append_oracle(x.cpu(), slots, cache, scale)
        assert torch.equal(ds.cpu(), scale)
        assert torch.equal(_bits(dc), cache.view(torch.uint8))


def _slots(runs, bs):
    """runs of (first slot, count): consecutive slots, the next block of each run the next one."""
    return [s + i for s, c in runs for i in range(c)]


@pytest.mark.parametrize("codes", CODES, ids=_ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("h,d,bs", [(1, 16, 16), (8, 128, 16), (3, 80, 32), (2, 64, 64), (5, 96, 128),
                                    (2, 112, 256)], ids=_ids)
def test_append(ops, h, d, bs, dtype, codes):
    g = torch.Generator().manual_seed(h * d + bs)
    # one token into a partly filled block, a block begun, a run over block ends, skipped tokens
    slots = ([3] + [2 * bs] + [-1, -1] + list(range(4 * bs + bs - 3, 6 * bs + 5)) + [-1]
             + list(range(8 * bs, 9 * bs)) + [10 * bs + bs - 1] + [12 * bs] + [99 * bs])
    k = torch.randn(len(slots), h, d, generator=g).to(dtype)
    v = (torch.randn(len(slots), h, d, generator=g) * 40).to(dtype)   # v's scales grow, k's do not
    _append_case(ops, k, v, slots, 13, bs, codes)


@pytest.mark.parametrize("codes", CODES, ids=_ids)
def test_append_many_tokens_and_single_ones(ops, codes):
    g = torch.Generator().manual_seed(5)
    for slots in (list(range(7, 3000)), [16 * i + (i * 7) % 16 for i in range(300)]):
        k = torch.randn(len(slots), 4, 64, generator=g).bfloat16()
        v = torch.randn(len(slots), 4, 64, generator=g).bfloat16()
        _append_case(ops, k, v, slots, 300, 16, codes)


@pytest.mark.parametrize("codes", CODES, ids=_ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_append_values_that_are_not_numbers(ops, dtype, codes):
    g = torch.Generator().manual_seed(6)
    k = torch.randn(40, 2, 32, generator=g).to(dtype)
    v = torch.randn(40, 2, 32, generator=g).to(dtype)
    k[3, 0, 5], k[4, 0, 7], k[20, 1, 0] = math.inf, -math.inf, math.nan
    v[:, 1] = 0                                  # scale 0
    v[25, 0] = math.nan                          # a whole token
    v[30, 0] = 1e-7                              # (bf16) far below the scale
    _append_case(ops, k, v, list(range(10, 50)), 4, 16, codes)
    k[:], v[:] = math.inf, math.nan              # nothing finite
    _append_case(ops, k, v, list(range(10, 50)), 4, 16, codes)
    if dtype == torch.bfloat16:
        k[:], v[:] = 1e-40, 1e-38                # subnormal scales
        _append_case(ops, k, v, list(range(16, 56)), 4, 16, codes)


def test_append_strides(ops):
    g = torch.Generator().manual_seed(7)
    kv = torch.randn(50, 2, 3, 64, generator=g).half().cuda()
    slots = list(range(50))
    _append_case(ops, kv[:, 0], kv[:, 1], slots, 4, 16, torch.int8)               # slices of one tensor
    t = torch.randn(3, 50, 64, generator=g).half().cuda()
    _append_case(ops, t.transpose(0, 1), t.transpose(0, 1), slots, 4, 16, torch.int8)   # head-major
    w = torch.randn(50, 3, 65, generator=g).half().cuda()
    _append_case(ops, w[:, :, 1:], w[:, :, :64], slots, 4, 16, torch.int8)        # rows off 16 bytes
    e = torch.randn(50, 1, 64, generator=g).half().cuda().expand(50, 3, 64)
    _append_case(ops, e, e, slots, 4, 16, torch.int8)                             # one head for all


def test_append_again_changes_nothing(ops):
    g = torch.Generator().manual_seed(8)
    k = (torch.randn(30, 2, 64, generator=g) * 9).half().cuda()
    c, s = _random_cache(g, 4, 2, 16, 64, torch.int8)
    kc, vc, ks, vs = c.cuda(), c.cuda(), s.cuda(), s.cuda()
    slots = _dev(list(range(9, 39)), torch.int64)
    ops.cache_append(k, k, slots, kc, vc, ks, vs)
    first = kc.clone(), ks.clone()
    ops.cache_append(k, k, slots, kc, vc, ks, vs)
    assert torch.equal(first[0], kc) and torch.equal(first[1], ks)
    assert torch.equal(kc, vc) and torch.equal(ks, vs)


# --------------------------------------------------------- cache attention
def _attend(q, k, v, scale, seen=None):
    """q (n, heads, d), k, v (m, kv_heads, d) in 64 bits; seen (n, m) or None: out, lse."""
    group = q.shape[1] // max(k.shape[1], 1)
    z = torch.einsum("nhd,mhd->hnm", q, k.repeat_interleave(group, 1)) * scale
    if seen is not None:
        z = z.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(z, -1) if z.shape[-1] else torch.full(z.shape[:-1], -math.inf).double()
    w = torch.exp(z - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    vv = v.repeat_interleave(group, 1).transpose(0, 1)
    w = torch.where(w > 0, w, 0.0)
    return torch.einsum("hnm,hmd->nhd", w, vv), lse.T


def _decode_case(ops, lens, h, group, d, bs, dtype, codes, seed=0, scale=None, q_scale=1.0, poison=True,
                 spread=1.0):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // bs) for n in lens]
    width = max(counts + [1]) + 1
    blocks = sum(counts) + 2
    order = torch.randperm(blocks, generator=g)
    kc, ks = _random_cache(g, blocks, h, bs, d, codes)
    vc, vs = _random_cache(g, blocks, h, bs, d, codes)
    vs = vs * spread ** torch.randn(vs.shape, generator=g)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    q = (torch.randn(len(lens), h * group, d, generator=g) * q_scale).to(dtype)
    want = torch.zeros(q.shape, dtype=torch.float64)
    want_lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    at = 0
    for r, n in enumerate(lens):
        ids = order[at:at + counts[r]]
        at += counts[r]
        table[r, :counts[r]] = ids.int()
        if n == 0:
            continue
        kv = []
        for c, s in ((kc, ks), (vc, vs)):
            x = c[ids].double() * s[ids].double()[:, :, None, None]
            kv.append(x.transpose(1, 2).reshape(-1, h, d)[:n])
        o, l = _attend(q[r:r + 1].double(), kv[0], kv[1], scale or d ** -0.5)
        want[r], want_lse[r] = o[0], l[0]
        if poison and n % bs and codes == torch.float8_e4m3fn:
            # what stands behind the last token is nobody's
            kc.view(torch.uint8)[ids[-1], :, n % bs:] = 0x7f
            vc.view(torch.uint8)[ids[-1], :, n % bs:] = 0x7f
    out, lse = ops.cache_attention(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(),
                                   _dev(lens), scale, True)
    assert out.dtype == dtype and out.shape == q.shape
    _close(out, want, dtype)
    fine = want_lse != -math.inf
    assert torch.equal(lse.cpu() == -math.inf, ~fine)
    assert (lse.cpu().double() - want_lse)[fine].abs().max() <= LSE_TOL if fine.any() else True
    for r, n in enumerate(lens):
        if n == 0:
            assert (out[r] == 0).all()
    _no_error(ops)


@pytest.mark.parametrize("codes", CODES, ids=_ids)
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("d", [16, 64, 80, 128])
@pytest.mark.parametrize("h,group,bs", [(1, 1, 16), (2, 5, 32), (3, 8, 16), (2, 12, 64), (1, 16, 128),
                                        (1, 40, 256)], ids=_ids)
def test_decode(ops, h, group, bs, d, dtype, codes):
    _decode_case(ops, [1, 15, 16, 17, 64, 65, 130, 0, 333], h, group, d, bs, dtype, codes,
                 seed=h * group + d)


@pytest.mark.parametrize("codes", CODES, ids=_ids)
def test_decode_one_long_request(ops, codes):
    _decode_case(ops, [20011], 2, 4, 128, 16, torch.float16, codes, seed=1)


def test_decode_many_requests(ops):
    g = np.random.default_rng(3)
    _decode_case(ops, g.integers(0, 200, 300).tolist(), 2, 2, 64, 16, torch.bfloat16, torch.int8, seed=2)


def test_decode_only_empty(ops):
    _decode_case(ops, [0, 0, 0], 2, 2, 64, 16, torch.float16, torch.int8)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_decode_peaked_and_uneven_scales(ops, dtype):
    # scores far apart: the running maximum moves; value scales over four decades
    _decode_case(ops, [700, 33], 2, 4, 128, 16, dtype, torch.int8, seed=4, q_scale=6.0)
    _decode_case(ops, [700, 33], 2, 4, 128, 16, dtype, torch.float8_e4m3fn, seed=5, spread=10.0)
    _decode_case(ops, [700, 33], 2, 4, 128, 16, dtype, torch.int8, seed=6, scale=0.3)


@pytest.mark.parametrize("codes", CODES, ids=_ids)
@pytest.mark.parametrize("power", [24, 40])
@pytest.mark.parametrize("d,group", [(64, 2), (128, 2), (64, 12), (128, 12)])
def test_decode_value_scales_that_some_heads_do_not_see(ops, d, group, power, codes):
    # Half the blocks have value scales 2^power larger; even heads weigh them with exp(-40), odd
    # heads see little else.  The even heads' output keeps its bits, head by head.
    g = torch.Generator().manual_seed(d + group + power)
    # The kinds alternate every four blocks, and 150 requests share them, so that a warp meets both.
    n, blocks, reqs = 333, 21, 150
    sign = torch.tensor([1.0, -1.0]).repeat_interleave(4).repeat(3)[:blocks].view(blocks, 1, 1, 1)
    kc = _codes_of(sign * 64 + torch.randint(-8, 9, (blocks, 1, 16, d), generator=g), codes)
    vc, vs = _random_cache(g, blocks, 1, 16, d, codes)
    ks = torch.full((blocks, 1), 1 / 64.0)
    vs = torch.where(sign[:, :, 0, 0] < 0, vs * 2.0 ** power, vs)
    q = torch.full((1, group, d), 20 / d ** 0.5)
    q[:, 1::2] *= -1
    q = q.bfloat16()
    k, v = (c.double() * s.double()[:, :, None, None] for c, s in ((kc, ks), (vc, vs)))
    k, v = (x.transpose(1, 2).reshape(-1, 1, d)[:n] for x in (k, v))
    want, want_lse = _attend(q.double(), k, v, d ** -0.5)
    out, lse = ops.cache_attention(q.cuda().repeat(reqs, 1, 1), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(),
                                   _dev([list(range(blocks))] * reqs), _dev([n] * reqs), None, True)
    for r in range(reqs):
        for j in range(group):
            _close(out[r, j], want[0, j], torch.bfloat16)
    assert (lse.cpu().double() - want_lse).abs().max() <= LSE_TOL
    _no_error(ops)


def test_decode_large_queries_in_bf16(ops):
    # beyond fp16's range: q is scaled by a power of two for the products
    _decode_case(ops, [100], 1, 4, 64, 16, torch.bfloat16, torch.int8, seed=7, q_scale=1e6, scale=1e-7)
    _decode_case(ops, [100], 1, 4, 64, 16, torch.bfloat16, torch.int8, seed=8, q_scale=1e-6, scale=1e5)


def test_decode_zero_scales_and_missing_blocks(ops):
    g = torch.Generator().manual_seed(9)
    kc, ks = _random_cache(g, 6, 1, 16, 64, torch.int8)
    vc, vs = _random_cache(g, 6, 1, 16, 64, torch.int8)
    vs[:] = 0
    q = torch.randn(2, 2, 64, generator=g).half()
    args = [x.cuda() for x in (kc, vc, ks, vs)]
    table = _dev([[0, 1, 2], [3, 4, 5]])
    assert (ops.cache_attention(q.cuda(), *args, table, _dev([40, 48])) == 0).all()
    # block numbers outside the cache leave their tokens out
    vs = torch.rand(6, 1, generator=g) + 0.5
    args[3] = vs.cuda()
    out = ops.cache_attention(q.cuda(), *args, _dev([[0, 77, 2], [-1, -1, 99]]), _dev([40, 48]))
    k = kc.double() * ks.double()[:, :, None, None]
    v = vc.double() * vs.double()[:, :, None, None]
    k, v = (x.transpose(1, 2)[[0, 2]].reshape(32, 1, 64)[:24] for x in (k, v))
    want, _ = _attend(q[:1].double(), k, v, 0.125)
    _close(out[:1], want, torch.float16)
    assert (out[1] == 0).all()
    # lengths are cut to the table
    cut = ops.cache_attention(q.cuda(), *args, table[:, :2].contiguous(), _dev([1000, -5]))
    assert torch.equal(cut[:1], ops.cache_attention(q.cuda(), *args, table, _dev([32, 0]))[:1])
    assert (cut[1] == 0).all()


def test_decode_strides_and_repeatability(ops):
    g = torch.Generator().manual_seed(10)
    kc, ks = _random_cache(g, 40, 2, 16, 64, torch.int8)
    args = [x.cuda() for x in (kc, kc, ks, ks)]
    table = torch.randperm(40, generator=g).int().view(4, 10).cuda()
    lens = _dev([150, 3, 99, 160])
    qkv = torch.randn(4, 12, 64, generator=g).half().cuda()
    q = qkv[:, 2:10]
    want = ops.cache_attention(q.contiguous(), *args, table, lens)
    assert torch.equal(ops.cache_attention(q, *args, table, lens), want)
    wide = torch.zeros(4, 25, dtype=torch.int32, device="cuda")
    wide[:, 5:15] = table
    assert torch.equal(ops.cache_attention(q, *args, wide[:, 5:15], lens), want)
    odd = torch.randn(4, 8, 65, generator=g).half().cuda()
    odd[:, :, 1:] = q
    assert torch.equal(ops.cache_attention(odd[:, :, 1:], *args, table, lens), want)


# -------------------------------------------------------- prompt attention
def _prompt_case(ops, lens, h, group, d, dtype, lens_k=None, causal=True, seed=0, scale=None, q_scale=1.0,
                 fused=False):
    g = torch.Generator().manual_seed(seed)
    own_k = lens_k is not None
    lens_k = lens_k if own_k else lens
    t, tk = sum(lens), sum(lens_k)
    if fused and not own_k:
        x = torch.randn(t, h * group + 2 * h, d, generator=g).to(dtype).cuda()
        q, k, v = x[:, :h * group], x[:, h * group:h * group + h], x[:, h * group + h:]
    else:
        q = (torch.randn(t, h * group, d, generator=g) * q_scale).to(dtype).cuda()
        k = torch.randn(tk, h, d, generator=g).to(dtype).cuda()
        v = torch.randn(tk, h, d, generator=g).to(dtype).cuda()
    cu, cuk = np.cumsum([0] + lens).tolist(), np.cumsum([0] + lens_k).tolist()
    out, lse = ops.prompt_attention(q, k, v, _dev(cu), _dev(cuk) if own_k else None, causal, scale, True)
    want = torch.zeros(q.shape, dtype=torch.float64)
    want_lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    qc, kc, vc = (x.cpu().double() for x in (q, k, v))
    for s, (n, m) in enumerate(zip(lens, lens_k)):
        seen = torch.ones(n, m, dtype=torch.bool)
        if causal:
            seen = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + m - n
        if n == 0:
            continue
        o, l = _attend(qc[cu[s]:cu[s + 1]], kc[cuk[s]:cuk[s + 1]], vc[cuk[s]:cuk[s + 1]],
                       scale or d ** -0.5, seen)
        want[cu[s]:cu[s + 1]], want_lse[cu[s]:cu[s + 1]] = o, l
    assert out.dtype == dtype and out.shape == q.shape
    _close(out, want, dtype)
    fine = want_lse != -math.inf
    assert torch.equal(lse.cpu() == -math.inf, ~fine)
    assert (out.cpu()[~fine] == 0).all()
    if fine.any():
        assert (lse.cpu().double() - want_lse)[fine].abs().max() <= LSE_TOL
    _no_error(ops)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
@pytest.mark.parametrize("d", [16, 64, 80, 128])
@pytest.mark.parametrize("h,group", [(1, 1), (2, 3), (2, 4), (1, 7), (1, 16), (1, 40)], ids=_ids)
def test_prompt(ops, h, group, d, dtype):
    _prompt_case(ops, [1, 17, 128, 129, 0, 300], h, group, d, dtype, seed=h * group + d, fused=True)


@pytest.mark.parametrize("lens", [[1], [127], [128], [256], [257], [1023], [1, 1, 1, 1], [0, 0, 5, 0],
                                  [31, 1, 511, 64]], ids=_ids)
def test_prompt_lengths(ops, lens):
    _prompt_case(ops, lens, 2, 2, 64, torch.float16, seed=sum(lens))
    _prompt_case(ops, lens, 1, 1, 128, torch.bfloat16, seed=sum(lens))


def test_prompt_many_sequences(ops):
    g = np.random.default_rng(4)
    _prompt_case(ops, g.integers(0, 40, 200).tolist(), 1, 4, 64, torch.float16, seed=1)


def test_prompt_longer(ops):
    _prompt_case(ops, [2500, 1111], 1, 2, 128, torch.bfloat16, seed=2)


def test_prompt_not_causal(ops):
    _prompt_case(ops, [3, 200, 129], 2, 2, 64, torch.float16, causal=False, seed=3)
    _prompt_case(ops, [3, 200, 129], 2, 2, 64, torch.float16, lens_k=[400, 1, 130], causal=False, seed=4)


def test_prompt_keys_of_their_own(ops):
    # chunks of longer prompts; more queries than keys: the first rows see nothing
    _prompt_case(ops, [64, 1, 200, 130], 2, 2, 128, torch.float16, lens_k=[500, 77, 200, 131], seed=5)
    _prompt_case(ops, [300, 100, 5], 1, 2, 64, torch.float16, lens_k=[10, 0, 5], seed=6)
    _prompt_case(ops, [300, 20], 1, 1, 64, torch.bfloat16, lens_k=[0, 0], seed=7)


def test_prompt_peaked_rows(ops):
    # large logits: the running maximum moves by more than the sums may grow
    _prompt_case(ops, [700, 40], 1, 2, 128, torch.float16, seed=8, q_scale=8.0)
    _prompt_case(ops, [700, 40], 1, 2, 64, torch.bfloat16, seed=9, scale=1.5)


def test_prompt_rising_scores(ops):
    # every key tile brings a new maximum: O is rescaled at each one
    n, d = 900, 64
    q = torch.zeros(n, 1, d).half()
    k = torch.zeros(n, 1, d).half()
    q[:, 0, 0] = 1
    k[:, 0, 0] = torch.arange(n) / 4.0
    g = torch.Generator().manual_seed(10)
    v = torch.randn(n, 1, d, generator=g).half()
    out, lse = ops.prompt_attention(q.cuda(), k.cuda(), v.cuda(), _dev([0, n]), scale=1.0, return_lse=True)
    seen = torch.ones(n, n, dtype=torch.bool).tril()
    want, want_lse = _attend(q.double(), k.double(), v.double(), 1.0, seen)
    _close(out, want, torch.float16)
    # |z| reaches 225: fp32 holds z * log2(e) to 2^-16
    assert (lse.cpu().double() - want_lse).abs().max() <= 2 * LSE_TOL


def test_prompt_neighbours_do_not_leak(ops):
    # the sequence behind holds infinities and NaN, in the same key tile
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(300, 2, 64, generator=g).half().cuda() for _ in range(3))
    cu = _dev([0, 50, 170, 300])
    want = ops.prompt_attention(q, k, v, cu)
    for bad in (math.inf, -math.inf, math.nan):
        k2, v2 = k.clone(), v.clone()
        k2[50:], v2[50:] = bad, bad
        got = ops.prompt_attention(q, k2, v2, cu)
        assert torch.equal(got[:50], want[:50])
        k2, v2 = k.clone(), v.clone()
        k2[:50], v2[:50] = bad, bad
        got = ops.prompt_attention(q, k2, v2, cu)
        assert torch.equal(got[50:], want[50:])


def test_prompt_rows_of_no_sequence(ops):
    g = torch.Generator().manual_seed(12)
    q, k, v = (torch.randn(100, 2, 64, generator=g).half().cuda() for _ in range(3))
    out, lse = ops.prompt_attention(q, k, v, _dev([10, 40, 80]), return_lse=True)
    assert (out[:10] == 0).all() and (out[80:] == 0).all()
    assert (lse[:10] == -math.inf).all() and (lse[80:] == -math.inf).all()
    inner = ops.prompt_attention(q[10:80], k[10:80], v[10:80], _dev([0, 30, 70]))
    assert torch.equal(out[10:80], inner)
    none = ops.prompt_attention(q, k, v, _dev([0]))
    assert (none == 0).all()
    # offsets past the tensors are cut to them
    past = ops.prompt_attention(q, k, v, _dev([0, 60, 5000]))
    assert torch.equal(past, ops.prompt_attention(q, k, v, _dev([0, 60, 100])))


def test_prompt_strides(ops):
    g = torch.Generator().manual_seed(13)
    q, k, v = (torch.randn(150, 4, 64, generator=g).bfloat16().cuda() for _ in range(3))
    cu = _dev([0, 33, 150])
    want = ops.prompt_attention(q, k, v, cu)
    t = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]       # head-major
    assert torch.equal(ops.prompt_attention(*t, cu), want)
    w = torch.zeros(150, 4, 65).bfloat16().cuda()
    w[:, :, 1:] = k
    assert torch.equal(ops.prompt_attention(q, w[:, :, 1:], v, cu), want)         # off 16 bytes
    one = k[:, :1]
    assert torch.equal(ops.prompt_attention(q, one.expand(150, 4, 64), v, cu),
                       ops.prompt_attention(q, one.expand(150, 4, 64).contiguous(), v, cu))


def test_prompt_on_another_stream(ops):
    g = torch.Generator().manual_seed(14)
    q, k, v = (torch.randn(500, 4, 64, generator=g).half().cuda() for _ in range(3))
    cu = _dev([0, 200, 500])
    want = ops.prompt_attention(q, k, v, cu)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.prompt_attention(q, k, v, cu)
    s.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------- long caches, streams and graphs
@pytest.mark.parametrize("codes", CODES, ids=_ids)
def test_cache_past_32_bits(ops, codes):
    """Blocks more than 2^32 codes from the cache's start: written, and read again."""
    h, d, bs, n = 8, 128, 16, 280000                 # 4.6 G codes each of K and V
    kc, vc = (torch.empty(n, h, bs, d, dtype=torch.uint8, device="cuda").view(codes) for _ in range(2))
    ks, vs = (torch.zeros(n, h, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(20)
    ids = [n - 1, 3, n - 7, 150000]
    k, v = (torch.randn(60, h, d, generator=g).half() for _ in range(2))
    slots = [ids[t // bs] * bs + t % bs for t in range(60)]
    ops.cache_append(k.cuda(), v.cuda(), _dev(slots, torch.int64), kc, vc, ks, vs)
    kv = []
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        want, scale = torch.zeros(4, h, bs, d, dtype=torch.uint8).view(codes), torch.zeros(4, h)
        _append_oracle(x, list(range(60)), want, scale)
        at = torch.tensor(ids, device="cuda")
        assert torch.equal(s[at].cpu(), scale)
        got = c.view(torch.uint8)[at].cpu().transpose(1, 2).reshape(64, h, d)[:60]
        assert torch.equal(got, want.view(torch.uint8).transpose(1, 2).reshape(64, h, d)[:60])
        kv.append((want.double() * scale.double()[:, :, None, None]).transpose(1, 2).reshape(64, h, d)[:60])
    q = torch.randn(1, 2 * h, d, generator=g).half()
    out = ops.cache_attention(q.cuda(), kc, vc, ks, vs, _dev([ids]), _dev([60]))
    _close(out, _attend(q.double(), *kv, d ** -0.5)[0], torch.float16)
    _no_error(ops)


def test_prompt_past_32_bits(ops):
    """Rows 2^24 elements apart: the last ones begin 3.3 G elements behind the first."""
    n, h, d, pitch = 200, 2, 64, 1 << 24
    buf = torch.empty(n * pitch, dtype=torch.float16, device="cuda")
    q, k, v = (torch.as_strided(buf, (n, h, d), (pitch, d, 1), i * 4096) for i in range(3))
    g = torch.Generator().manual_seed(21)
    for x in (q, k, v):
        x.copy_(torch.randn(n, h, d, generator=g))
    cu = _dev([0, 77, n])
    got = ops.prompt_attention(q, k, v, cu)
    assert torch.equal(got, ops.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu))
    _no_error(ops)


def _step_state(seed):
    g = torch.Generator().manual_seed(seed)
    lens = [40, 0, 17, 100]
    held = [-(-n // 16) for n in lens]
    order = torch.randperm(sum(held) + 6, generator=g).int()
    table = torch.full((4, 10), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    caches = []
    for _ in range(2):
        caches += _random_cache(g, len(order), 2, 16, 64, torch.int8)
    q, k, v = (torch.randn(4, n, 64, generator=g).half() for n in (4, 2, 2))
    kc, ks, vc, vs = (x.cuda() for x in caches)
    return dict(lens=_dev(lens), one=_dev([1] * 4), table=table.cuda(), free=order[at:].clone().cuda(),
                count=_dev([len(order) - at]), kc=kc, ks=ks, vc=vc, vs=vs, q=q.cuda(), k=k.cuda(), v=v.cuda())


def _step(ops, s):
    slots, cu, lens, left = ops.block_tables(s["lens"], s["one"], s["table"], s["free"], s["count"], 4, 16)
    ops.cache_append(s["k"], s["v"], slots, s["kc"], s["vc"], s["ks"], s["vs"])
    out = ops.cache_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], lens)
    own = ops.prompt_attention(s["q"], s["k"], s["v"], cu)
    return slots, lens, left, out, own, s["kc"], s["ks"], s["table"]


def test_step_on_another_stream(ops):
    want = _step(ops, _step_state(30))
    state = _step_state(30)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = _step(ops, state)
    stream.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_step_in_a_graph(ops):
    want = _step(ops, _step_state(31))
    warm, state = _step_state(32), _step_state(31)
    _step(ops, warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(ops, state)
    fresh = _step_state(31)                          # the capture ran nothing
    for name, x in state.items():
        assert torch.equal(x, fresh[name])
    for _ in range(2):                               # a step over the same lengths repeats itself
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)
    _no_error(ops)


def test_prompt_then_one_token_agree(ops):
    """The last row of a prompt's attention is what one token sees over the cache of the others, but
    for the cache's 8 bits (int8: about 1 % of a value's standard deviation, in K and in V)."""
    g = torch.Generator().manual_seed(33)
    n, h, d = 300, 2, 128
    q, k, v = (torch.randn(n, x, d, generator=g).half().cuda() for x in (4 * h, h, h))
    blocks = -(-n // 16)
    kc, vc = (torch.zeros(blocks, h, 16, d, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(blocks, h, device="cuda") for _ in range(2))
    ops.cache_append(k, v, torch.arange(n, device="cuda"), kc, vc, ks, vs)
    table = torch.arange(blocks, dtype=torch.int32, device="cuda")[None]
    token, lse = ops.cache_attention(q[-1:], kc, vc, ks, vs, table, _dev([n]), return_lse=True)
    prompt, plse = ops.prompt_attention(q, k, v, _dev([0, n]), return_lse=True)
    assert ((token - prompt[-1:]).norm() / prompt[-1:].norm()) <= 0.04
    assert (lse - plse[-1:]).abs().max() <= 0.04


# ----------------------------------------------------------------- refusals
def test_refusals(ops):
    q = torch.randn(4, 4, 64, device="cuda").half()
    k = torch.randn(4, 2, 64, device="cuda").half()
    cu = _dev([0, 4])
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        ops.prompt_attention(q.float(), k.float(), k.float(), cu)
    with pytest.raises(RuntimeError, match="one dtype"):
        ops.prompt_attention(q, k.bfloat16(), k.bfloat16(), cu)
    with pytest.raises(RuntimeError, match="multiple of k's"):
        ops.prompt_attention(q[:, :3], k, k, cu)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        ops.prompt_attention(q[:, :, :40], k[:, :, :40], k[:, :, :40], cu)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        ops.prompt_attention(*(torch.zeros(4, 1, 256, device="cuda").half() for _ in range(3)), cu)
    with pytest.raises(RuntimeError, match="cu_seqlens must be"):
        ops.prompt_attention(q, k, k, cu.long())
    with pytest.raises(RuntimeError, match="cu_seqlens_k"):
        ops.prompt_attention(q, k[:3], k[:3], cu)
    with pytest.raises(RuntimeError, match="as many values"):
        ops.prompt_attention(q, k, k, cu, _dev([0, 2, 4]))
    with pytest.raises(RuntimeError, match="scale must be positive"):
        ops.prompt_attention(q, k, k, cu, scale=-1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.prompt_attention(q.cpu(), k, k, cu)
    with pytest.raises(RuntimeError, match="same device"):
        ops.prompt_attention(q, k.cpu(), k.cpu(), cu)

    kc = torch.zeros(3, 2, 16, 64, dtype=torch.int8, device="cuda")
    ks = torch.zeros(3, 2, device="cuda")
    table, lens = _dev([[0, 1]] * 4), _dev([1] * 4)
    with pytest.raises(RuntimeError, match="int8 or float8_e4m3fn"):
        ops.cache_attention(q, kc.half(), kc.half(), ks, ks, table, lens)
    with pytest.raises(RuntimeError, match="one shape"):
        ops.cache_attention(q, kc, kc[:2], ks, ks, table, lens)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.cache_attention(q, kc.transpose(1, 2).contiguous().transpose(1, 2), kc, ks, ks, table, lens)
    with pytest.raises(RuntimeError, match="power of two"):
        ops.cache_attention(q, kc[:, :, :8].contiguous(), kc[:, :, :8].contiguous(), ks, ks, table, lens)
    with pytest.raises(RuntimeError, match="k_scale"):
        ops.cache_attention(q, kc, kc, ks[:, :1].contiguous(), ks, table, lens)
    with pytest.raises(RuntimeError, match="one row for each request"):
        ops.cache_attention(q, kc, kc, ks, ks, table[:3], lens)
    with pytest.raises(RuntimeError, match="seq_lens"):
        ops.cache_attention(q, kc, kc, ks, ks, table, lens.long())
    with pytest.raises(RuntimeError, match="multiple of the cache's"):
        ops.cache_attention(q[:, :3], kc, kc, ks, ks, table, lens)

    slots = _dev([0, 1, 2, 3], torch.int64)
    with pytest.raises(RuntimeError, match="the cache holds"):
        ops.cache_append(q, q, slots, kc, kc.clone(), ks, ks.clone())
    with pytest.raises(RuntimeError, match="slots"):
        ops.cache_append(k, k, slots.int(), kc, kc.clone(), ks, ks.clone())
    with pytest.raises(RuntimeError, match="slots must have"):
        ops.cache_append(k, k, slots[:3].contiguous(), kc, kc.clone(), ks, ks.clone())
    with pytest.raises(RuntimeError, match="one shape, dtype"):
        ops.cache_append(k, k.bfloat16(), slots, kc, kc.clone(), ks, ks.clone())

    i = _dev([1, 2])
    with pytest.raises(RuntimeError, match="one value for each request"):
        ops.block_tables(i, i[:1].contiguous(), _dev([[0], [0]]), i, _dev([2]), 3, 16)
    with pytest.raises(RuntimeError, match="one row for each request"):
        ops.block_tables(i, i, _dev([[0]]), i, _dev([2]), 3, 16)
    with pytest.raises(RuntimeError, match="power of two"):
        ops.block_tables(i, i, _dev([[0], [0]]), i, _dev([2]), 3, 24)
    with pytest.raises(RuntimeError, match="new_lens must be"):
        ops.block_tables(i, i.long(), _dev([[0], [0]]), i, _dev([2]), 3, 16)


def test_empty_calls(ops):
    kc = torch.zeros(3, 2, 16, 64, dtype=torch.int8, device="cuda")
    ks = torch.zeros(3, 2, device="cuda")
    e = torch.empty(0, 2, 64, device="cuda").half()
    ops.cache_append(e, e, _dev([], torch.int64), kc, kc.clone(), ks, ks.clone())
    assert ops.cache_attention(e, kc, kc, ks, ks, _dev([]).view(0, 2), _dev([])).shape == e.shape
    assert ops.prompt_attention(e, e, e, _dev([0, 0])).shape == e.shape
    q = torch.randn(2, 4, 64, device="cuda").half()
    none = torch.zeros(0, 2, 16, 64, dtype=torch.int8, device="cuda")
    out = ops.cache_attention(q, none, none, ks[:0], ks[:0], _dev([[0], [0]]), _dev([3, 0]))
    assert (out == 0).all()


def test_rows_that_begin_off_16_bytes(ops):
    # dense, so that a dense copy is what it is already
    g = torch.Generator().manual_seed(70)

    def odd(*shape):
        n = math.prod(shape)
        return torch.randn(n + 1, generator=g).half().cuda()[1:].view(shape)

    q, k, v = odd(20, 4, 64), odd(20, 2, 64), odd(20, 2, 64)
    cu = _dev([0, 7, 20])
    assert torch.equal(ops.prompt_attention(q, k, v, cu), ops.prompt_attention(q.clone(), k.clone(), v.clone(), cu))
    caches = []
    for a, b in ((k, v), (k.clone(), v.clone())):
        c = [torch.zeros(2, 2, 16, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
        c += [torch.zeros(2, 2, device="cuda") for _ in range(2)]
        ops.cache_append(a, b, torch.arange(20, device="cuda"), *c)
        caches.append(c)
    assert all(torch.equal(x, y) for x, y in zip(*caches))
    table, lens = _dev([[0, 1]]), _dev([20])
    assert torch.equal(ops.cache_attention(q[:1], *caches[0], table, lens),
                       ops.cache_attention(q[:1].clone(), *caches[0], table, lens))
    _no_error(ops)
