"""The serving operators on the GPU against 64-bit restatements of their formulas (tests/serving_ref.py)."""
import math

import numpy as np
import pytest
import torch

from m3_avm_b200 import _lib
from tests import serving_ref as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def status(clear=True):
    import ctypes

    s = ctypes.c_uint32()
    _lib.check(_lib.load().m3g_device_status(0, ctypes.byref(s), 1 if clear else 0))
    return s.value


@pytest.fixture(autouse=True)
def clean_status():
    status()
    yield
    assert status() == 0


def randn(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


# ---------------------------------------------------------------- rope
# c and s come from sincospi of a fraction of a turn rounded to 24 bits: 2^-24 of at most one half turn, pi 2^-24 in
# the angle, and 2^-23 of sincospi and the magnitude's product; a result is two products and a sum, each rounded.
ROPE_TOL = math.pi * 2.0 ** -24 + 2.0 ** -22


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,KH,D,rot", [(1, 32, 8, 128, 128), (37, 5, 1, 64, 32), (3, 64, 8, 128, 64),
                                          (2, 3, 3, 80, 20), (5, 2, 1, 6, 2), (2, 1, 1, 512, 256), (130, 9, 2, 64, 64)])
def test_rope(dtype, inter, T, H, KH, D, rot):
    from m3_avm_b200.attention import Rope

    q, k = randn(1, T, H, D, dtype=dtype), randn(2, T, KH, D, dtype=dtype)
    pos = torch.randint(0, 200000, (T,), dtype=torch.int32, generator=torch.Generator().manual_seed(3)).cuda()
    plan = Rope(D, rot_dim=rot, theta=500000.0, interleaved=inter)
    f, mag = R.frequencies(rot, 500000.0)
    for inverse in (False, True):
        got = plan.apply(pos, q, k, inverse=inverse)
        for x, y in zip((q, k), got):
            want, size, a, b = R.rope(x, pos, rot, inter, f, mag, inverse)
            err = np.abs(y.double().cpu().numpy() - want)
            tol = R.EPS[dtype] * np.abs(want)
            tol[..., a] += ROPE_TOL * size
            tol[..., b] += ROPE_TOL * size
            assert np.all(err <= tol + 1e-7 * (dtype == F16)), float((err / (tol + 1e-30)).max())
            assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("scaling,kw", [("linear", dict(factor=4.0)), ("ntk", dict(factor=2.5)),
                                        ("yarn", dict(factor=8.0, orig_ctx=4096)),
                                        ("yarn", dict(factor=2.0, orig_ctx=64, beta_fast=4.0, beta_slow=2.0)),
                                        ("llama3", dict(factor=8.0, orig_ctx=8192))])
def test_rope_scalings_far_positions_and_both_ends(scaling, kw):
    from m3_avm_b200.attention import Rope

    pos = torch.tensor([0, 1, 2 ** 31 - 1, -1, -2 ** 31, 1000003, 131071], dtype=torch.int32).cuda()
    q = randn(5, 7, 3, 128)
    f, mag = R.frequencies(128, 10000.0, scaling, **kw)
    y, none = Rope(128, scaling=scaling, **kw).apply(pos, q)
    assert none is None
    want, size, a, b = R.rope(q, pos, 128, False, f, mag)
    # f itself is a double: at position 2^31 it moves the angle by 2^31 2^-53
    tol = R.EPS[F32] * np.abs(want)
    tol[..., a] += (ROPE_TOL + 2.0 ** -20) * size * mag
    tol[..., b] += (ROPE_TOL + 2.0 ** -20) * size * mag
    assert np.all(np.abs(y.cpu().numpy() - want) <= tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rope_strides_in_place_and_unaligned(dtype):
    from m3_avm_b200.attention import Rope

    plan = Rope(64, rot_dim=32)
    pos = torch.arange(9, dtype=torch.int32).cuda() * 1000
    joint = randn(6, 9, 7, 64, dtype=dtype)
    want = plan.apply(pos, joint[:, :4].contiguous(), joint[:, 4:6].contiguous())
    got = plan.apply(pos, joint[:, :4], joint[:, 4:6])
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    # heads outermost
    swapped = joint[:, :4].permute(1, 0, 2).contiguous().permute(1, 0, 2)
    out = torch.empty(4, 9, 64, dtype=dtype, device="cuda").permute(1, 0, 2)
    assert torch.equal(plan.apply(pos, swapped, q_out=out)[0], want[0]) and torch.equal(out, want[0])
    # rows that start one value off a 16-byte boundary
    buf = torch.zeros(9 * 4 * 65 + 1, dtype=dtype, device="cuda")
    odd = buf[1:].as_strided((9, 4, 64), (4 * 65, 65, 1))
    odd.copy_(joint[:, :4])
    odd = buf.as_strided((9, 4, 64), (4 * 65, 65, 1), 1)
    assert torch.equal(plan.apply(pos, odd)[0], want[0])
    # in place; what lies between the heads stays
    keep = joint.clone()
    plan.apply(pos, joint[:, :4], joint[:, 4:6], q_out=joint[:, :4], k_out=joint[:, 4:6])
    assert torch.equal(joint[:, :4], want[0]) and torch.equal(joint[:, 4:6], want[1])
    assert torch.equal(joint[:, 6], keep[:, 6])


def test_rope_inverse_is_the_gradient():
    """<R x, g> = <x, R^T g>, and against differences of the forward call."""
    from m3_avm_b200.attention import Rope

    plan = Rope(64, scaling="yarn", factor=4.0, orig_ctx=2048, interleaved=True)
    pos = torch.tensor([5, 77, 4000], dtype=torch.int32).cuda()
    x, g = randn(1, 3, 2, 64), randn(2, 3, 2, 64)
    grad = plan.apply(pos, g, inverse=True)[0].double()
    y = plan.apply(pos, x)[0].double()
    assert abs(float((y * g.double()).sum() - (x.double() * grad).sum())) < 384 * 2.0 ** -18
    d = randn(3, 3, 2, 64)
    # the map is linear: a difference of any step is exact up to rounding
    diff = plan.apply(pos, x + d)[0].double() - y
    assert abs(float((diff * g.double()).sum() - ((x + d).double() - x.double()).mul(grad).sum())) < 384 * 2.0 ** -17


def test_rope_nothing_to_do():
    from m3_avm_b200.attention import Rope

    plan = Rope(64)
    q = torch.empty(0, 4, 64, device="cuda")
    y, _ = plan.apply(torch.empty(0, dtype=torch.int32, device="cuda"), q)
    assert y.shape == q.shape


# ---------------------------------------------------------------- cache
@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,kvh,page,ctx,new", [(64, 2, 16, [0, 5, 31], [1, 17, 40]), (128, 3, 64, [100], [1]),
                                                 (128, 8, 16, [0, 7, 15, 16], [3, 0, 1, 33]), (64, 1, 1024, [0], [1030])])
def test_cache_write_and_read(q8, dtype, hd, kvh, page, ctx, new):
    from m3_avm_b200.attention import KvCache

    batch, pages, _, _ = R.make_batch(ctx, new, page, seed=len(new))
    cache = KvCache(8 if q8 else 2, 3, kvh, hd, page, pages)
    cache.pool.fill_(0xAB)
    before = cache.pool.clone()
    t = sum(new)
    k, v = randn(1, t, kvh, hd, scale=3.0, dtype=dtype), randn(2, t, kvh, hd, scale=0.01, dtype=dtype)
    cache.write(1, k, v, batch)
    per = cache.pool.numel() // 3
    assert torch.equal(cache.pool[:per], before[:per]) and torch.equal(cache.pool[2 * per:], before[2 * per:])
    rows = pages * kvh * page
    # rows of no new token stay as they were: 2 (codes + scales) planes change in t * kvh rows at most
    changed = (cache.pool[per:2 * per] != before[per:2 * per]).sum().item()
    assert changed <= 2 * t * kvh * ((hd if q8 else hd // 2) + hd // 16) and rows > 0
    for out_type in (F32, dtype):
        gk, gv = cache.read(1, batch, dtype=out_type)
        for got, x in ((gk, k), (gv, v)):
            assert torch.equal(got.cpu(), R.quantised(x, q8).to(out_type))


@pytest.mark.parametrize("q8", [True, False])
def test_cache_blocks_are_those_of_the_host_quantiser(q8):
    from m3_avm_b200 import quant
    from m3_avm_b200.attention import KvCache

    batch, pages, table, _ = R.make_batch([0], [16], 16)
    cache = KvCache(8 if q8 else 2, 1, 1, 64, 16, pages)
    x = randn(3, 16, 1, 64, scale=100.0)
    x[3] = 0
    x[4, 0, :32] *= 1e-9
    x[5] = torch.round(x[5])  # halves and whole quotients
    x[6, 0, :32] = torch.arange(32).cuda() - 15.5
    cache.write(0, x, x, batch)
    page = int(table[0, 0])
    cb = 64 if q8 else 32
    codes = cache.pool[page * 16 * cb:(page + 1) * 16 * cb].cpu().numpy().reshape(16, 2, cb // 2)
    at = pages * 16 * cb
    scales = cache.pool[at + page * 64:at + (page + 1) * 64].cpu().numpy().reshape(16, 2, 2)
    for t in range(16):
        for b in range(2):
            dst = bytearray(34 if q8 else 18)
            src = x[t, 0, 32 * b:32 * b + 32].cpu().numpy()
            assert (quant.quantize_q8_0 if q8 else quant.quantize_q4_0)(src, dst)
            want = np.frombuffer(bytes(dst), np.uint8)
            assert np.array_equal(scales[t, b], want[:2])
            if want[0] or want[1]:  # a scale of 0: the codes stand for 0 whatever they are
                assert np.array_equal(codes[t, b], want[2:] + (128 if q8 else 0))


@pytest.mark.parametrize("q8", [True, False])
def test_cache_values_that_are_not_finite_or_too_large(q8):
    from m3_avm_b200.attention import KvCache

    batch, pages, _, _ = R.make_batch([0], [8], 16)
    cache = KvCache(8 if q8 else 2, 1, 1, 64, 16, pages)
    x = randn(3, 8, 1, 64)
    x[0, 0, 3] = float("nan")
    x[1, 0, 40] = float("inf")
    x[2, 0, 31] = float("-inf")
    x[3, 0, 5] = 3e38
    x[4, 0, 5] = 65504.0 * (127 if q8 else 7)  # the largest scale
    x[5, 0, 5] = 1e-45
    x[6] = 1e-40
    cache.write(0, x, -x, batch)
    gk, gv = cache.read(0, batch)
    want = R.quantised(x, q8)
    assert torch.isnan(want).sum() == 32 * 4
    assert torch.equal(torch.isnan(gk.cpu()), torch.isnan(want))
    assert torch.equal(gk.cpu().nan_to_num(), want.nan_to_num())
    assert torch.equal(gv.cpu().nan_to_num(), -want.nan_to_num()) or not q8  # 4 bits: -8 .. 7 is not symmetric


def test_cache_strides_broadcast_and_unaligned():
    from m3_avm_b200.attention import KvCache

    batch, pages, _, _ = R.make_batch([3, 0], [5, 2], 16)
    cache = KvCache(8, 1, 4, 64, 16, pages)
    joint = randn(1, 7, 9, 64, dtype=BF16)
    cache.write(0, joint[:, 1:5], joint[:, 5:], batch)
    k, v = cache.read(0, batch, dtype=BF16)
    assert torch.equal(k.cpu(), R.quantised(joint[:, 1:5], True).to(BF16))
    assert torch.equal(v.cpu(), R.quantised(joint[:, 5:], True).to(BF16))
    one = randn(2, 7, 1, 64)
    cache.write(0, one.expand(7, 4, 64), one.expand(7, 4, 64), batch)  # one head's rows for all
    k, v = cache.read(0, batch)
    assert torch.equal(k.cpu(), R.quantised(one, True).expand(7, 4, 64)) and torch.equal(k, v)
    buf = torch.zeros(7 * 4 * 67 + 3, device="cuda")
    odd = buf.as_strided((7, 4, 64), (4 * 67, 67, 1), 3)
    odd.copy_(one.expand(7, 4, 64))
    cache.pool.zero_()
    cache.write(0, odd, odd, batch)
    out = buf.clone().as_strided((7, 4, 64), (4 * 67, 67, 1), 3).fill_(7.0)
    cache.read(0, batch, k_out=out, v_out=torch.empty_like(k))
    assert torch.equal(out, k)


def test_cache_bad_pages_and_batches():
    """What a batch says wrongly is skipped and reported, and touches nothing else."""
    from m3_avm_b200.attention import KvBatch, KvCache

    batch, pages, table, start = R.make_batch([0, 4, 0], [6, 3, 20], 16)
    cache = KvCache(8, 1, 2, 64, 16, pages)
    x = randn(1, 29, 2, 64)
    want = R.quantised(x, True)
    bad = table.clone()
    bad[1, 0], bad[2, 1] = pages, -7
    b2 = KvBatch(batch.q_start, batch.ctx_len, bad.cuda(), 29, 20, 23)
    cache.write(0, x, x, b2)
    assert status() == 32
    k = torch.full((29, 2, 64), 5.0, device="cuda")
    v = torch.full((29, 2, 64), 5.0, device="cuda")
    cache.read(0, b2, k_out=k, v_out=v)
    assert status() == 32
    skipped = torch.zeros(29, dtype=torch.bool)
    skipped[6:9] = True
    skipped[9 + 16:] = True
    assert torch.equal(k.cpu()[~skipped], want[~skipped]) and bool((k.cpu()[skipped] == 5).all())
    # too long for the call's limits, starts outside the tensors, a negative context
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    for q_start, ctx, most, length in ((i32(0, 6, 9, 29), i32(0, 4, 0), 19, 23), (i32(0, 6, 9, 29), i32(0, 4, 4), 20, 23),
                                       (i32(0, 6, 9, 30), i32(0, 4, 0), 21, 23), (i32(0, 6, 9, 29), i32(0, 4, -1), 20, 23),
                                       (i32(0, 6, 9, 29), i32(0, 4, 2 ** 31 - 1), 20, 23)):
        b3 = KvBatch(q_start, ctx, table.cuda(), 29, most, length)
        cache.pool.zero_()
        cache.write(0, x, x, b3)
        assert status() == 16
        k.fill_(5.0)
        cache.read(0, b3, k_out=k, v_out=v)
        assert status() == 16
        assert torch.equal(k.cpu()[:9], want[:9]) and bool((k.cpu()[9:] == 5).all())


# ---------------------------------------------------------------- attention
def roomy(batch, page):
    """The same batch with limits of 2^18 positions: large trees then take the form for large calls."""
    from m3_avm_b200.attention import KvBatch

    table = torch.full((batch.page_table.shape[0], 2 ** 18 // page), -1, dtype=torch.int32, device="cuda")
    table[:, :batch.page_table.shape[1]] = batch.page_table
    return KvBatch(batch.q_start, batch.ctx_len, table, batch.n_tokens, batch.max_tokens, 2 ** 18)


def attention_case(q8, dtype, heads, kvh, hd, page, ctx, new, tree, seed=0, empty=(), qscale=1.5, strided=False,
                   scale=None, large=False):
    from m3_avm_b200.attention import KvCache, tree_attention

    batch, pages, _, _ = R.make_batch(ctx, new, page, seed=seed)
    if large:
        batch = roomy(batch, page)
    cache = KvCache(8 if q8 else 2, 2, kvh, hd, page, pages)
    cache.pool.fill_(0xFF)  # rows behind the sequences: scales that are NaN
    full = R.whole(batch, ctx, new)
    total = full.n_tokens
    k, v = randn(seed + 1, total, kvh, hd), randn(seed + 2, total, kvh, hd)
    cache.write(1, k, v, full)
    kd, vd = R.quantised(k, q8).double(), R.quantised(v, q8).double()
    cut = [c + n for c, n in zip(ctx, new)]
    ks, vs = torch.split(kd, cut), torch.split(vd, cut)
    t = sum(new)
    q = randn(seed + 3, t, heads, hd, scale=qscale, dtype=dtype)
    if strided:
        big = torch.zeros(heads, t, hd + 8, dtype=dtype, device="cuda")
        big[:, :, :hd] = q.permute(1, 0, 2)
        q = big[:, :, :hd].permute(1, 0, 2)
    mask, bits = None, [np.tril(np.ones((n, n), bool)) for n in new]
    if tree:
        bits = R.tree_bits(new, seed, empty)
        mask = R.pack_bits(bits, -(-max(new) // 32) + (seed % 2))
    got = tree_attention(q, cache, 1, batch, mask=mask, scale=scale)
    want, vmax, smag = R.attention(q, ks, vs, ctx, new, bits, scale or hd ** -0.5)
    return got, want, R.attention_bound(want, vmax, smag, dtype), (q, cache, batch, mask)


def assert_within(got, want, bound):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), f"worst error / bound {float((err / bound).max()):.3g}"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kvh,page,ctx,new,tree", [
    (8, 2, 16, [0], [1], False),                       # one token, nothing before it
    (32, 8, 64, [1023], [1], False),                   # a decode step
    (4, 4, 16, [15, 16, 17, 31, 0], [1, 1, 1, 1, 1], False),
    (12, 4, 16, [40, 0, 129], [7, 13, 1], True),
    (5, 1, 32, [300, 77], [64, 33], True),             # two mask words, groups of five
    (16, 2, 128, [0, 500], [40, 3], False),            # a prompt without a context
    (64, 8, 16, [2100], [9], True),
])
def test_attention(dtype, q8, hd, heads, kvh, page, ctx, new, tree):
    got, want, bound, _ = attention_case(q8, dtype, heads, kvh, hd, page, ctx, new, tree, seed=hd + len(ctx))
    assert_within(got, want, bound)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_long_and_many(dtype):
    got, want, bound, _ = attention_case(True, dtype, 8, 2, 64, 64, [9000, 1, 4000], [2, 5, 1], True, seed=9)
    assert_within(got, want, bound)
    n = 300  # more sequences than a CTA has threads
    r = np.random.default_rng(0)
    ctx, new = [int(x) for x in r.integers(0, 90, n)], [int(x) for x in r.integers(0, 4, n)]
    got, want, bound, _ = attention_case(False, dtype, 4, 2, 64, 16, ctx, new, True, seed=10)
    assert_within(got, want, bound)


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_large_trees(q8, large, hd):
    for dtype, new in ((BF16, [64, 50, 17]), (F16, [64]), (F32, [40, 40]), (BF16, [257]), (F16, [7, 33])):
        got, want, bound, _ = attention_case(q8, dtype, 16, 2, hd, 64, [777, 0, 64][:len(new)], new, True, seed=4,
                                             large=large)
        assert_within(got, want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kvh,page,ctx,new,tree", [
    (64, 8, 16, [0], [9], False), (64, 1, 16, [63], [1], False), (64, 1, 64, [64, 0, 1, 127], [1, 2, 1, 65], True),
    (10, 2, 32, [3000, 100, 5], [30, 1, 12], True), (32, 1, 128, [20000], [3], True),
])
def test_attention_large_form(dtype, heads, kvh, page, ctx, new, tree):
    for q8 in (True, False):
        got, want, bound, (q, cache, batch, mask) = attention_case(q8, dtype, heads, kvh, 128, page, ctx, new, tree,
                                                                   seed=kvh, large=True)
        assert_within(got, want, bound)
        from m3_avm_b200.attention import tree_attention

        for _ in range(3):
            assert torch.equal(tree_attention(q, cache, 1, batch, mask=mask), got)


def test_attention_large_form_growing_scores():
    """Maxima that grow by 2^20 from one chunk to the next: the results so far are rescaled each time."""
    from m3_avm_b200.attention import KvCache, tree_attention

    for dtype in (F16, BF16):
        batch, pages, _, _ = R.make_batch([700], [20], 16)
        cache = KvCache(8, 1, 1, 64, 16, pages)
        full = R.whole(batch, [700], [20])
        k, v = randn(1, 720, 1, 64, scale=0.1), randn(2, 720, 1, 64)
        q = randn(3, 20, 4, 64, dtype=dtype)
        k += (torch.arange(720, device="cuda") // 64 * 0.25).view(-1, 1, 1) * torch.sign(q[3, 1].float())
        cache.write(0, k, v, full)
        got = tree_attention(q, cache, 0, roomy(batch, 16), scale=1.0)
        bits = [np.tril(np.ones((20, 20), bool))]
        want, vmax, smag = R.attention(q, [R.quantised(k, True).double()], [R.quantised(v, True).double()], [700], [20],
                                       bits, 1.0)
        assert_within(got, want, R.attention_bound(want, vmax, smag, dtype))


def test_attention_rows_that_see_nothing():
    got, want, bound, _ = attention_case(True, F32, 8, 2, 64, 16, [0, 5], [4, 3], True, seed=2, empty=(0, 2, 5))
    assert_within(got, want, bound)
    assert bool((got[0] == 0).all()) and bool((got[2] == 0).all()) and bool((got[5] != 0).any())


def test_attention_what_a_row_does_not_see_does_not_reach_it():
    """A drafted token whose K or V is NaN leaves the rows that do not see it as they were."""
    from m3_avm_b200.attention import KvCache, tree_attention

    for hd, dtype, heads, large in ((64, F32, 4, False), (128, BF16, 4, False), (128, BF16, 64, False),
                                    (128, BF16, 64, True), (64, F16, 64, True)):
        batch, pages, _, _ = R.make_batch([20], [6], 16)
        batch = roomy(batch, 16) if large else batch
        cache = KvCache(8, 1, 2, hd, 16, pages)
        full = R.whole(batch, [20], [6])
        k, v = randn(1, 26, 2, hd), randn(2, 26, 2, hd)
        q = randn(3, 6, heads, hd, dtype=dtype)
        bits = [np.tril(np.ones((6, 6), bool))]
        bits[0][3:, 2] = False  # tokens 3 .. 5 do not see token 2
        mask = R.pack_bits(bits, 1)
        cache.write(0, k, v, full)
        clean = tree_attention(q, cache, 0, batch, mask=mask)
        for where in ("k", "v"):
            k2, v2 = k.clone(), v.clone()
            (k2 if where == "k" else v2)[22] = float("nan")
            cache.write(0, k2, v2, full)
            got = tree_attention(q, cache, 0, batch, mask=mask)
            assert torch.equal(got[[0, 1, 3, 4, 5]], clean[[0, 1, 3, 4, 5]])
            assert bool(torch.isnan(got[2]).all())
        # one row's q that is NaN
        cache.write(0, k, v, full)
        q2 = q.clone()
        q2[1, 1, 0] = float("nan")
        got = tree_attention(q2, cache, 0, batch, mask=mask)
        assert bool(torch.isnan(got[1, 1]).all())
        got[1, 1], ref = 0, clean.clone()
        ref[1, 1] = 0
        assert torch.equal(got, ref)


def test_attention_strides_in_place_and_scale():
    from m3_avm_b200.attention import tree_attention

    for dtype, heads, large in ((F32, 8, False), (F16, 8, False), (F16, 32, True), (BF16, 32, True)):
        got, want, bound, (q, cache, batch, mask) = attention_case(True, dtype, heads, 2, 128, 16, [50], [5], True,
                                                                   seed=6, strided=True, scale=0.2, large=large)
        assert_within(got, want, bound)
        buf = torch.zeros(5 * heads * 131 + 1, dtype=dtype, device="cuda")
        odd = buf.as_strided((5, heads, 128), (heads * 131, 131, 1), 1)
        odd.copy_(q)
        assert torch.equal(tree_attention(odd, cache, 1, batch, mask=mask, scale=0.2), got)
        assert tree_attention(odd, cache, 1, batch, mask=mask, scale=0.2, out=odd) is odd
        assert torch.equal(odd, got)


def test_attention_rows_behind_the_last_sequence_stay():
    from m3_avm_b200.attention import KvBatch, tree_attention

    got, want, bound, (q, cache, batch, _) = attention_case(True, BF16, 8, 2, 64, 16, [30, 9], [4, 2], False, seed=1)
    q8 = torch.cat([q, torch.full_like(q[:3], float("nan"))])
    b = KvBatch(batch.q_start, batch.ctx_len, batch.page_table, 9, 8, 200)
    out = torch.full_like(q8, 5.0)
    tree_attention(q8, cache, 1, b, out=out)
    assert torch.equal(out[:6], got) and bool((out[6:] == 5).all())
    # a sequence past the limits is skipped whole
    b = KvBatch(batch.q_start, batch.ctx_len, batch.page_table, 6, 3, 200)
    out = torch.full_like(q, 5.0)
    tree_attention(q, cache, 1, b, out=out)
    assert status() == 16
    assert torch.equal(out[4:], got[4:]) and bool((out[:4] == 5).all())


def test_attention_bad_page_reads_as_zeros():
    from m3_avm_b200.attention import KvBatch, tree_attention

    _, _, _, (q, cache, batch, _) = attention_case(True, F32, 8, 2, 64, 16, [60], [2], False, seed=1)
    table = batch.page_table.clone()
    table[0, 1] = cache.n_pages + 5
    got = tree_attention(q, cache, 1, KvBatch(batch.q_start, batch.ctx_len, table, 2, 2, 62))
    assert status() == 32
    # the same with that page's rows zero
    k, v = cache.read(1, R.whole(batch, [60], [2]))
    k[16:32] = 0
    v[16:32] = 0
    cache.write(1, k, v, R.whole(batch, [60], [2]))
    want = tree_attention(q, cache, 1, batch)
    assert float((got - want).abs().max()) <= 2.0 ** -17 * float(v.abs().max())


def test_attention_of_large_and_tiny_values():
    from m3_avm_b200.attention import KvCache, tree_attention

    for dtype, large in ((F32, False), (BF16, False), (BF16, True)):
        for scale_v in (3e5, 1e-6):
            batch, pages, _, _ = R.make_batch([100], [3], 16)
            heads = 64 if large else 4
            cache = KvCache(8, 1, 1, 64, 16, pages)
            full = R.whole(batch, [100], [3])
            k, v = randn(1, 103, 1, 64, scale=20.0), randn(2, 103, 1, 64, scale=scale_v)
            v[50:] *= 1e-3 if scale_v > 1 else 1.0
            cache.write(0, k, v, full)
            q = randn(3, 3, heads, 64, scale=2.0, dtype=dtype)
            got = tree_attention(q, cache, 0, roomy(batch, 16) if large else batch)
            bits = [np.tril(np.ones((3, 3), bool))]
            want, vmax, smag = R.attention(q, [R.quantised(k, True).double()], [R.quantised(v, True).double()], [100],
                                           [3], bits, 0.125)
            assert_within(got, want, R.attention_bound(want, vmax, smag, dtype))


@pytest.mark.parametrize("heads,large", [(8, False), (64, True)])
def test_attention_repeats_to_the_bit_and_replays_from_a_graph(heads, large):
    from m3_avm_b200.attention import tree_attention

    _, _, _, (q, cache, batch, mask) = attention_case(True, BF16, heads, 2, 128, 16, [3000, 20], [5, 6], True, seed=3,
                                                      large=large)
    first = tree_attention(q, cache, 1, batch, mask=mask)
    for _ in range(3):
        assert torch.equal(tree_attention(q, cache, 1, batch, mask=mask), first)
    out = torch.zeros_like(q)
    ws = torch.empty(cache.attention_workspace(heads, BF16, 6), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tree_attention(q, cache, 1, batch, mask=mask, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tree_attention(q, cache, 1, batch, mask=mask, out=out, workspace=ws)
    out.zero_()
    g.replay()
    assert torch.equal(out, first)
    # the replay reads the lengths of its moment: the last sequence shorter
    batch.ctx_len[1] = 4
    g.replay()
    want = tree_attention(q, cache, 1, batch, mask=mask)
    assert torch.equal(out, want) and not torch.equal(out, first)


def test_attention_two_streams_at_once():
    from m3_avm_b200.attention import tree_attention

    a = attention_case(True, F32, 8, 2, 64, 16, [5000], [3], True, seed=3)
    b = attention_case(False, F16, 64, 4, 128, 16, [7000], [9], True, seed=5, large=True)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s, (got, _, _, (q, cache, batch, mask)) in ((s1, a), (s2, b)):
            with torch.cuda.stream(s):
                outs.append((tree_attention(q, cache, 1, batch, mask=mask), got))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in outs)


def test_attention_of_nothing():
    from m3_avm_b200.attention import KvBatch, KvCache, tree_attention

    cache = KvCache(8, 1, 2, 64, 16, 2)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    b = KvBatch(i32(0, 0), i32(5), i32(0).view(1, 1), 0, 0, 16)
    assert tree_attention(torch.empty(0, 4, 64, device="cuda"), cache, 0, b).shape == (0, 4, 64)
    q = torch.full((2, 4, 64), 3.0, device="cuda")  # tokens of no sequence
    b = KvBatch(i32(0, 0), i32(5), i32(0).view(1, 1), 2, 2, 16)
    out = torch.full_like(q, 4.0)
    tree_attention(q, cache, 0, b, out=out)
    assert bool((out == 4).all())


# ---------------------------------------------------------------- log probabilities
def logprob_reference(x, tokens, k):
    x = x.double().cpu()
    lp = torch.log_softmax(x, -1)
    given = torch.full(tokens.shape, -math.inf, dtype=torch.float64)
    ok = (tokens >= 0) & (tokens < x.shape[1])
    rows = torch.arange(x.shape[0])[:, None].expand_as(tokens)
    given[ok] = lp[rows[ok], tokens[ok].long()]
    p = lp.exp()
    entropy = -(torch.where(p > 0, p * lp, torch.zeros_like(p))).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :k]
    return given, entropy, order, torch.gather(lp, 1, order)


def lp_tolerance(x):
    """Base-2 exponents t = x log2(e) - m are off by 2^-24 (|x| + |m|) each, ex2 by 2^-22, sums of n terms by
    (n / 512 + 32) 2^-24: the relative error of z; a log probability adds two roundings of its own size, the entropy
    sums (t - m) times that."""
    fin = torch.where(x.double().abs() < math.inf, x.double().abs(), torch.zeros(())).amax().item()
    n = x.shape[1]
    z = 2.0 ** -22 + (n / 512 + 32) * 2.0 ** -24 + 2 * 2.0 ** -23 * fin
    return z + 2.0 ** -22 * (2 * fin + math.log(n)), z * (2 + 2 * fin + math.log(n)) + 2.0 ** -22 * (2 * fin + math.log(n))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,n,k", [(1, 128256, 1, 20), (1, 1, 1, 1), (3, 7, 2, 7), (2, 8192, 4, 32), (5, 8193, 1, 5),
                                            (33, 32001, 3, 1), (300, 5000, 1, 0), (700, 1000, 2, 8), (2, 40, 0, 32),
                                            (20, 65536, 1, 3), (80, 20000, 1, 32)])
def test_logprobs(dtype, rows, vocab, n, k):
    from m3_avm_b200.logprobs import token_logprobs

    x = randn(rows + vocab, rows, vocab, scale=4.0, dtype=dtype)
    tokens = torch.randint(-1, vocab + 1, (rows, n), dtype=torch.int32, generator=torch.Generator().manual_seed(1))
    got = token_logprobs(x, tokens.cuda() if n else None, n_top=k, entropy=True)
    given, entropy, ids, tops = logprob_reference(x.cpu(), tokens, k)
    tol, etol = lp_tolerance(x.cpu())
    if n:
        inside = torch.isfinite(given)
        assert torch.equal(torch.isfinite(got.logprob.cpu()), inside)
        assert bool(((got.logprob.double().cpu() - given).abs()[inside] <= tol).all())
        assert bool((got.logprob.cpu()[~inside] == -math.inf).all())
    assert bool(((got.entropy.double().cpu() - entropy).abs() <= etol).all())
    if k:
        assert torch.equal(got.top_ids.cpu().long(), ids)
        assert bool(((got.top_logprobs.double().cpu() - tops).abs() <= tol).all())
    else:
        assert got.top_ids is None and got.top_logprobs is None


@pytest.mark.parametrize("rows,vocab", [(1, 128256), (400, 9001)])
def test_logprobs_ties_masks_and_orders(rows, vocab):
    from m3_avm_b200.logprobs import token_logprobs

    x = torch.zeros(rows, vocab)                      # all equal
    kinds = []
    kinds.append(x.clone())
    y = torch.full((rows, vocab), -math.inf)          # few left
    for j, i in enumerate((vocab - 1, 5, 77, 8195)):
        y[:, i] = j * 0.5
    kinds.append(y)
    kinds.append(torch.arange(vocab).float().expand(rows, vocab).contiguous() / 1000)   # rising
    kinds.append(-torch.arange(vocab).float().expand(rows, vocab).contiguous() / 1000)  # falling
    z = torch.randint(-3, 3, (rows, vocab), generator=torch.Generator().manual_seed(2)).float()
    z[:, ::3] = -0.0                                  # many ties, zeros of both signs
    kinds.append(z)
    kinds.append(torch.full((rows, vocab), torch.finfo(F32).min))  # the type's lowest value
    kinds[-1][:, 9] = 3.0
    w = torch.full((rows, vocab), -1e4)
    w[:, -1] = 1e4
    kinds.append(w)
    for m in kinds:
        tokens = torch.tensor([[0, vocab - 1, 5]], dtype=torch.int32).expand(rows, 3).contiguous()
        got = token_logprobs(m.cuda(), tokens.cuda(), n_top=32, entropy=True)
        given, entropy, ids, tops = logprob_reference(m, tokens, 32)
        tol, etol = lp_tolerance(torch.where(m > -3e38, m, torch.zeros(())))
        assert torch.equal(got.top_ids.cpu().long(), ids)
        for a, b, t in ((got.logprob, given, tol), (got.top_logprobs, tops, tol), (got.entropy[:, None], entropy[:, None], etol)):
            a = a.double().cpu()
            inf = torch.isinf(b) | (b < -1e37)
            assert bool((a[inf] < -1e37).all()) and bool(((a - b).abs()[~inf] <= t).all())


def test_logprobs_rows_without_a_distribution():
    from m3_avm_b200.logprobs import token_logprobs

    x = randn(1, 5, 3000)
    clean = token_logprobs(x, torch.zeros(5, 1, dtype=torch.int32).cuda(), n_top=4, entropy=True)
    y = x.clone()
    y[1, 17] = float("nan")
    y[2] = -math.inf
    y[3, 2999] = math.inf
    got = token_logprobs(y, torch.zeros(5, 1, dtype=torch.int32).cuda(), n_top=4, entropy=True)
    for r in (1, 2, 3):
        assert torch.isnan(got.logprob[r]).all() and torch.isnan(got.entropy[r]) and torch.isnan(got.top_logprobs[r]).all()
        assert bool(((got.top_ids[r] >= 0) & (got.top_ids[r] < 3000)).all())
    for r in (0, 4):
        assert all(torch.equal(a[r], b[r]) for a, b in zip(got, clean))
    assert int(got.top_ids[3, 0]) == 2999


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 60001), (700, 300)])
def test_logprobs_rows_of_extreme_logits(dtype, rows, vocab):
    """Rows with nothing above the type's lowest value, and rows up to its largest: all but the largest logits have
    probability 0 there, so a log probability is -ln(how many), of which log2, the product with ln 2 and its constant
    are rounded.  A largest logit below 1e38 (F16: above -32768) has the term 2^d, d the rounding of its product with
    log2(e): ex2 is off by 2^-22 and their sum by (n / 512 + 32) 2^-24 of itself."""
    from m3_avm_b200.logprobs import token_logprobs

    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    tol = 3 * 2.0 ** -22 * math.log(vocab) + 2.0 ** -22 + (vocab / 512 + 32) * 2.0 ** -24
    some = torch.arange(vocab) % 3 == 1
    for fill, value in ((low, low), (-math.inf, low), (low, 0.75 * low), (0.75 * low, 0.5 * low), (low, high), (0, high),
                        (-math.inf, high), (0.75 * high, high)):
        x = torch.where(some, torch.tensor(value, dtype=dtype), torch.tensor(fill, dtype=dtype)).expand(rows, vocab)
        x = x.contiguous()
        tokens = torch.tensor([[1, 4, 0]], dtype=torch.int32).expand(rows, 3).contiguous()
        got = token_logprobs(x.cuda(), tokens.cuda(), n_top=5, entropy=True)
        given, entropy, ids, tops = logprob_reference(x, tokens, 5)
        assert torch.equal(got.top_ids.cpu().long(), ids)
        for a, b in ((got.logprob, given), (got.top_logprobs, tops), (got.entropy, entropy)):
            a = a.double().cpu()
            far = b < -200.0  # differences of logits: one rounding, or past the type
            assert bool(((a - b).abs()[~far] <= tol).all())
            assert bool(((a[far] <= b[far] * (1 - 2.0 ** -20)) & (a[far] < -200.0)).all())
    y = torch.full((2, vocab), low, dtype=dtype)
    y[0, 7], y[1, vocab - 1] = float("nan"), math.inf
    got = token_logprobs(y.cuda(), torch.zeros(2, 1, dtype=torch.int32).cuda(), n_top=3, entropy=True)
    assert torch.isnan(got.logprob).all() and torch.isnan(got.entropy).all() and torch.isnan(got.top_logprobs).all()


def test_logprobs_strides_and_unaligned_rows():
    from m3_avm_b200.logprobs import token_logprobs

    for dtype in (F32, BF16):
        x = randn(1, 6, 4097, dtype=dtype)  # rows of an odd length: none but the first is aligned
        big = torch.zeros(6, 4104, dtype=dtype, device="cuda")
        big[:, :4097] = x
        tokens = torch.full((6, 2), 4096, dtype=torch.int32).cuda()
        a = token_logprobs(x, tokens, n_top=9, entropy=True)
        b = token_logprobs(big[:, :4097], tokens, n_top=9, entropy=True)
        assert torch.equal(a.top_ids, b.top_ids)
        tol, etol = lp_tolerance(x.cpu())
        assert float((a.logprob - b.logprob).abs().max()) <= 2 * tol
        same = token_logprobs(x[:1].expand(6, 4097), tokens, n_top=9)  # one row six times
        assert bool((same.top_ids == same.top_ids[:1]).all())


def test_logprobs_captured():
    from m3_avm_b200.logprobs import token_logprobs

    x = randn(1, 3, 50000)
    tokens = torch.tensor([[1], [2], [3]], dtype=torch.int32).cuda()
    token_logprobs(x, tokens, n_top=3, entropy=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = token_logprobs(x, tokens, n_top=3, entropy=True)
    x.copy_(randn(2, 3, 50000))
    g.replay()
    want = token_logprobs(x, tokens, n_top=3, entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(out, want))


# ---------------------------------------------------------------- together
def test_a_verify_step():
    """Turn, write, attend, score: a drafted tree against the same tokens fed one after the other along each path."""
    from m3_avm_b200.attention import KvBatch, KvCache, Rope, tree_attention
    from m3_avm_b200.logprobs import token_logprobs

    heads, kvh, hd, ctx = 8, 2, 64, 45
    rope = Rope(hd, theta=500000.0, scaling="llama3", factor=8.0, orig_ctx=8192)
    parents = [-1, 0, 0, 1, 2]
    depth = [0, 1, 1, 2, 2]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    table = torch.randperm(6, generator=torch.Generator().manual_seed(0)).int().cuda().view(1, 6)
    past_k, past_v = randn(1, ctx, kvh, hd), randn(2, ctx, kvh, hd)
    q, k, v = randn(3, 5, heads, hd), randn(4, 5, kvh, hd), randn(5, 5, kvh, hd)
    head = randn(6, heads * hd, 1000, scale=0.05)
    bits = np.zeros((5, 5), bool)
    for j, p in enumerate(parents):
        if p >= 0:
            bits[j] = bits[p]
        bits[j, j] = True

    def cache_with_past():
        c = KvCache(8, 1, kvh, hd, 16, 6)
        c.write(0, past_k, past_v, KvBatch(i32([0, ctx]), i32([0]), table, ctx, ctx, 96))
        return c

    cache = cache_with_past()
    batch = KvBatch(i32([0, 5]), i32([ctx]), table, 5, 5, 96)
    tq, tk = rope.apply(i32([ctx + d for d in depth]), q, k)
    cache.write(0, tk, v, batch)
    out = tree_attention(tq, cache, 0, batch, mask=R.pack_bits([bits], 1))
    lp = token_logprobs(out.reshape(5, -1) @ head, i32([[7]] * 5), n_top=3)
    for path in ([0, 1, 3], [0, 2, 4]):
        step = cache_with_past()
        for d, node in enumerate(path):
            b = KvBatch(i32([0, 1]), i32([ctx + d]), table, 1, 1, 96)
            sq, sk = rope.apply(i32([ctx + d]), q[node:node + 1], k[node:node + 1])
            step.write(0, sk, v[node:node + 1], b)
            one = tree_attention(sq, step, 0, b)
            # the same positions with the same values, in another order and split
            assert float((one[0] - out[node]).abs().max()) <= 2.0 ** -15 * 5
            lp1 = token_logprobs(one.reshape(1, -1) @ head, i32([[7]]), n_top=3)
            assert torch.equal(lp1.top_ids[0], lp.top_ids[node])
            assert abs(float(lp1.logprob[0, 0] - lp.logprob[node, 0])) < 1e-3
    # the accepted path's rows written again behind the context: the cache of the path fed token by token
    acc = i32([0, 2, 4]).long()
    cache.write(0, tk[acc], v[acc], KvBatch(i32([0, 3]), i32([ctx]), table, 3, 3, 96))
    every = KvBatch(i32([0, ctx + 3]), i32([0]), table, ctx + 3, ctx + 3, 96)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(0, every), step.read(0, every)))
