"""Edges of the serving operators on the GPU: other streams, pools of other writers, bounds, captures, layouts."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from m3_avm_b200 import _lib
from tests import serving_ref as R
from tests.test_serving_gpu import assert_within, randn, roomy, status

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def clean_status():
    status()
    yield
    assert status() == 0


# ---------------------------------------------------------------- streams
def stream_of(t):
    """The stream whose memory t is, by the allocator."""
    for seg in torch.cuda.memory_snapshot():
        if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"]:
            return seg["stream"]
    raise AssertionError("not the allocator's memory")


def step_calls(seed=0):
    """Every operator on the same inputs: name -> call(stream)."""
    from m3_avm_b200.attention import KvCache, Rope, tree_attention
    from m3_avm_b200.logprobs import token_logprobs

    batch, pages, _, _ = R.make_batch([70, 9], [3, 2], 16)
    cache = KvCache(8, 1, 2, 64, 16, pages)
    full = R.whole(batch, [70, 9], [3, 2])
    cache.write(0, randn(1, full.n_tokens, 2, 64), randn(2, full.n_tokens, 2, 64), full)
    q, pos = randn(3, 5, 8, 64), torch.arange(5, dtype=torch.int32).cuda()
    x, rope = randn(4, 5, 3000), Rope(64)
    tokens = torch.zeros(5, 1, dtype=torch.int32).cuda()
    ws = torch.empty(cache.attention_workspace(8, F32, 3), dtype=torch.uint8, device="cuda")
    return {
        "rope": lambda s: rope.apply(pos, q, q[:, :2], stream=s),
        "read": lambda s: cache.read(0, full, stream=s),
        "attention": lambda s: (tree_attention(q, cache, 0, batch, stream=s),),
        "attention with a workspace": lambda s: (tree_attention(q, cache, 0, batch, workspace=ws, stream=s),),
        "logprobs": lambda s: tuple(token_logprobs(x, tokens, n_top=20, entropy=True, stream=s)),
    }


@pytest.mark.parametrize("name", ["rope", "read", "attention", "attention with a workspace", "logprobs"])
def test_calls_on_a_stream_of_their_own_beside_a_busy_current_one(name):
    call = step_calls()[name]
    want = call(None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    big = torch.full((4096, 4096), 1.0, device="cuda")
    for _ in range(5):
        for _ in range(4):
            (big @ big).sum()  # pending work on blocks that are free again
        got = call(side.cuda_stream)
        assert all(stream_of(t) == side.cuda_stream for t in got)
        for t in got:
            t.record_stream(side)
        side.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.current_stream().synchronize()
    with torch.cuda.stream(side):  # the default stream by its handle
        got = call(0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and stream_of(a) == 0 for a, b in zip(got, want))


# ---------------------------------------------------------------- captures
CAPTURED = """
import torch
from m3_avm_b200.attention import KvBatch, KvCache, Rope, tree_attention
from m3_avm_b200.logprobs import token_logprobs
i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()
cache = KvCache(8, 1, 2, 64, 16, 4)
batch = KvBatch(i32(0, 3), i32(0), i32(2, 1).view(1, 2), 3, 3, 32)
q, k, v, pos = torch.randn(3, 4, 64).cuda(), torch.randn(3, 2, 64).cuda(), torch.randn(3, 2, 64).cuda(), i32(0, 1, 2)
head, rope = torch.randn(256, 500).cuda(), Rope(64)
def step():
    a, b = rope.apply(pos, q, k)
    cache.write(0, b, v, batch)
    o = tree_attention(a, cache, 0, batch)
    kk, vv = cache.read(0, batch)
    return [a, b, o, kk, vv] + [t for t in token_logprobs(o.view(3, 256), n_top=3, entropy=True) if t is not None]
torch.mm(head.t()[:2], head)  # cuBLAS is not what is tested
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got]
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("captured")
"""


def test_first_calls_of_a_process_can_be_captured():
    done = subprocess.run([sys.executable, "-c", CAPTURED], capture_output=True, text=True, timeout=300,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__))))
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


# ---------------------------------------------------------------- pools of other writers
def planes(cache, layer=0):
    """The layer's planes as the header lays them out: K codes, K scales, V codes, V scales."""
    cb = cache.head_dim if cache.dtype == 8 else cache.head_dim // 2
    nb = cache.head_dim // 32
    rows = cache.n_pages * cache.n_kv_heads * cache.page_size
    at, out = layer * rows * 2 * (cb + 2 * nb), []
    for _ in range(2):
        out.append(cache.pool[at:at + rows * cb].view(cache.n_pages, cache.n_kv_heads, cache.page_size, cb))
        at += rows * cb
        out.append(cache.pool[at:at + rows * 2 * nb].view(F16).view(cache.n_pages, cache.n_kv_heads, cache.page_size, nb))
        at += rows * 2 * nb
    return out


def flip(cache, where):
    """The blocks that `where` picks with the opposite sign of scale and codes: the same values."""
    for codes, scales in (planes(cache)[:2], planes(cache)[2:]):
        pick = where(scales.shape)
        scales.copy_(torch.where(pick, -scales, scales))
        wide = pick.repeat_interleave(codes.shape[-1] // scales.shape[-1], -1)
        if cache.dtype == 8:
            neg = (256 - codes.int()).to(torch.uint8)
        else:
            lo, hi = codes.int() & 15, codes.int() >> 4
            neg = ((16 - lo) % 16 + 16 * ((16 - hi) % 16)).to(torch.uint8)
        codes.copy_(torch.where(wide, neg, codes))


@pytest.mark.parametrize("every", [True, False])
@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,hd,large", [(F32, 64, False), (F16, 128, False), (BF16, 128, False), (BF16, 64, True),
                                            (F16, 128, True)])
def test_attention_scales_below_zero(dtype, hd, large, q8, every):
    from m3_avm_b200.attention import KvCache, tree_attention

    batch, pages, _, _ = R.make_batch([150], [4], 16)
    heads = 64 if large else 4
    for size in (1.0, 3e5 if q8 else 2e4):  # scales of up to 1e4, in f16's range
        cache = KvCache(8 if q8 else 2, 1, 1, hd, 16, pages)
        full = R.whole(batch, [150], [4])
        k, v = randn(1, 154, 1, hd), randn(2, 154, 1, hd, scale=size)
        cache.write(0, k, v, full)
        g = torch.Generator().manual_seed(4)
        flip(cache, lambda s: torch.ones(s, dtype=torch.bool).cuda() if every else
             (torch.rand(s, generator=g) < 0.5).cuda())
        kd, vd = (x.double().cpu() for x in cache.read(0, full))
        assert torch.equal(kd.float(), R.quantised(k, q8)) and torch.equal(vd.float(), R.quantised(v, q8))
        q = randn(3, 4, heads, hd, dtype=dtype)
        got = tree_attention(q, cache, 0, roomy(batch, 16) if large else batch)
        bits = [np.tril(np.ones((4, 4), bool))]
        want, vmax, smag = R.attention(q, [kd], [vd], [150], [4], bits, hd ** -0.5)
        bound = R.attention_bound(want, vmax, smag, dtype)
        past = want.abs() + bound >= torch.finfo(dtype).max  # F16: the nearest value may be infinite
        got = torch.where(past & torch.isinf(got.cpu()) & (torch.sign(got.cpu()) == torch.sign(want)), want, got.double().cpu())
        assert_within(got, want, bound)


# ---------------------------------------------------------------- scores and bounds
@pytest.mark.parametrize("dtype,large", [(F32, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("scale,qscale", [(1e-24, 0.0), (1e-44, 1.0), (1e-30, 1e-20)])
def test_attention_scores_that_underflow(dtype, large, scale, qscale):
    """Scores of (nearly) nothing: the mean of what each row sees."""
    from m3_avm_b200.attention import KvCache, tree_attention

    batch, pages, _, _ = R.make_batch([40], [5], 16)
    cache = KvCache(8, 1, 1, 64, 16, pages)
    full = R.whole(batch, [40], [5])
    k, v = randn(1, 45, 1, 64), randn(2, 45, 1, 64)
    cache.write(0, k, v, full)
    q = randn(3, 5, 64 if large else 4, 64, scale=qscale, dtype=dtype)
    got = tree_attention(q, cache, 0, roomy(batch, 16) if large else batch, scale=scale)
    bits = [np.tril(np.ones((5, 5), bool))]
    want, vmax, smag = R.attention(q, [R.quantised(k, True).double()], [R.quantised(v, True).double()], [40], [5], bits,
                                   scale)
    assert_within(got, want, R.attention_bound(want, vmax, smag, dtype))


def test_batch_of_large_bounds():
    """Bounds that only one sequence could reach refuse no batch whose tokens are few."""
    from m3_avm_b200.attention import KvBatch, KvCache, tree_attention

    n = 300
    ctx, new = [5 + i % 40 for i in range(n)], [1] * n
    new[7] = 30
    batch, pages, table, _ = R.make_batch(ctx, new, 64)
    wide = torch.full((n, 2048), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    cache = KvCache(8, 1, 8, 64, 64, pages)
    full = R.whole(batch, ctx, new)
    cache.write(0, randn(1, full.n_tokens, 8, 64), randn(2, full.n_tokens, 8, 64), full)
    for dtype in (BF16, F32):
        q = randn(3, sum(new), 32, 64, dtype=dtype)
        tight = tree_attention(q, cache, 0, batch)
        got = tree_attention(q, cache, 0, KvBatch(batch.q_start, batch.ctx_len, wide.cuda(), sum(new), 2048, 131072))
        assert float((got.float() - tight.float()).abs().max()) < 0.02


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sequences_that_overlap_past_all_bounds_are_refused_whole(dtype):
    """2^12 starts that go back and forth, so that every second sequence claims the same 2^10 tokens, behind 2^20
    positions each: 2^33 chunks and more, where the bounds allow 2^29."""
    from m3_avm_b200.attention import KvBatch, KvCache, tree_attention

    n, t = 1 << 12, 1 << 10
    starts = torch.zeros(n + 1, dtype=torch.int32)
    starts[1::2] = t
    cache = KvCache(8, 1, 8, 64, 1024, 1)
    table = torch.zeros(n, 1024, dtype=torch.int32).cuda()
    batch = KvBatch(starts.cuda(), torch.full((n,), 2 ** 20 - t, dtype=torch.int32).cuda(), table, t, t, 2 ** 20)
    q = randn(1, t, 32, 64, dtype=dtype)
    out = torch.full_like(q, 5.0)
    tree_attention(q, cache, 0, batch, out=out)
    assert status() == 16
    assert bool((out == 5).all())


# ---------------------------------------------------------------- log probabilities of rows that few threads hold
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab,k", [(700, 3500, 32), (1, 3500, 32), (300, 2100, 32), (300, 1031, 20), (40, 259, 32),
                                          (40, 250, 32), (700, 1800, 32)])
def test_logprobs_of_short_rows_with_many_alternatives(dtype, rows, vocab, k):
    from m3_avm_b200.logprobs import token_logprobs
    from tests.test_serving_gpu import logprob_reference, lp_tolerance

    x = randn(rows + vocab, rows, vocab, scale=4.0, dtype=dtype)
    tokens = torch.randint(0, vocab, (rows, 1), dtype=torch.int32, generator=torch.Generator().manual_seed(1))
    got = token_logprobs(x, tokens.cuda(), n_top=k, entropy=True)
    given, entropy, ids, tops = logprob_reference(x.cpu(), tokens, k)
    tol, etol = lp_tolerance(x.cpu())
    assert torch.equal(got.top_ids.cpu().long(), ids)
    assert bool(((got.top_logprobs.double().cpu() - tops).abs() <= tol).all())
    assert bool(((got.logprob.double().cpu() - given).abs() <= tol).all())
    assert bool(((got.entropy.double().cpu() - entropy).abs() <= etol).all())


# ---------------------------------------------------------------- the pool's layout, byte by byte
def host_blocks(rows, dtype):
    """Codes and scales (as bytes) of rows (..., head_dim) by the library's host quantisers."""
    from m3_avm_b200 import quant

    x = rows.float().cpu().numpy()
    codes, scales = [], []
    for row in x.reshape(-1, x.shape[-1]):
        c, s = b"", b""
        for b in row.reshape(-1, 32):
            dst = bytearray(34 if dtype == 8 else 18)
            assert (quant.quantize_q8_0 if dtype == 8 else quant.quantize_q4_0)(np.ascontiguousarray(b), dst)
            s += bytes(dst[:2])
            body = np.frombuffer(bytes(dst[2:]), np.uint8)
            c += (body + 128).astype(np.uint8).tobytes() if dtype == 8 else body.tobytes()
        codes.append(np.frombuffer(c, np.uint8))
        scales.append(np.frombuffer(s, np.uint8))
    shape = x.shape[:-1] + (-1,)
    return np.stack(codes).reshape(shape), np.stack(scales).reshape(shape)


@pytest.mark.parametrize("dtype", [8, 2])
@pytest.mark.parametrize("kvh,hd,page", [(3, 128, 16), (2, 64, 32), (40, 64, 16)])
def test_pool_bytes_are_those_of_the_documented_layout(dtype, kvh, hd, page):
    """Every byte of a pool of 3 layers: [K codes, K scales, V codes, V scales][page][head][place], others untouched."""
    from m3_avm_b200.attention import KvCache

    ctx, new, layers, layer = [5, 0, page - 1, 40], [7, 1, page + 2, 0], 3, 1
    batch, pages, table, _ = R.make_batch(ctx, new, page, seed=kvh)
    cache = KvCache(dtype, layers, kvh, hd, page, pages)
    g = torch.Generator(device="cuda").manual_seed(2)
    cache.pool.copy_(torch.randint(0, 256, cache.pool.shape, generator=g, device="cuda", dtype=torch.uint8))
    want = cache.pool.cpu().numpy().copy()
    k, v = randn(1, sum(new), kvh, hd, scale=2.0), randn(2, sum(new), kvh, hd, scale=0.1)
    cache.write(layer, k, v, batch)
    cb, sb = (hd if dtype == 8 else hd // 2), hd // 16
    rows = pages * kvh * page
    base = layer * rows * 2 * (cb + sb)
    at = {"kc": base, "ks": base + rows * cb, "vc": base + rows * (cb + sb), "vs": base + rows * (2 * cb + sb)}
    for x, c, s in ((k, "kc", "ks"), (v, "vc", "vs")):
        codes, scales = host_blocks(x, dtype)
        t = 0
        for i, (before, n) in enumerate(zip(ctx, new)):
            for pos in range(before, before + n):
                for h in range(kvh):
                    row = (int(table[i, pos // page]) * kvh + h) * page + pos % page
                    want[at[c] + row * cb:at[c] + (row + 1) * cb] = codes[t, h]
                    want[at[s] + row * sb:at[s] + (row + 1) * sb] = scales[t, h]
                t += 1
    assert np.array_equal(cache.pool.cpu().numpy(), want)


@pytest.mark.parametrize("q8", [True, False])
def test_cache_values_below_zero_that_are_not_finite_or_too_large(q8):
    from m3_avm_b200.attention import KvCache

    batch, pages, _, _ = R.make_batch([0], [8], 16)
    cache = KvCache(8 if q8 else 2, 1, 1, 64, 16, pages)
    x = randn(3, 8, 1, 64)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 31], x[3, 0, 5] = float("nan"), float("inf"), float("-inf"), 3e38
    x[4, 0, 5], x[5, 0, 5], x[6] = 65504.0 * (127 if q8 else 7), 1e-45, 1e-40
    cache.write(0, x, -x, batch)
    for got, given in zip(cache.read(0, batch), (x, -x)):
        want = R.quantised(given, q8)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(got.cpu().nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (F16, 128), (F16, 64), (BF16, 128)])
@pytest.mark.parametrize("ksize,vsize", [(1e5, 1.0), (1.0, 1e4), (1e5, 1e4)])
def test_attention_large_form_of_scales_past_the_f16_range(dtype, hd, q8, ksize, vsize):
    """Some blocks whose scales are past 500 (K's scores with an attention scale that keeps them in range)."""
    from m3_avm_b200.attention import KvCache, tree_attention

    batch, pages, _, _ = R.make_batch([200], [6], 16)
    cache = KvCache(8 if q8 else 2, 1, 1, hd, 16, pages)
    full = R.whole(batch, [200], [6])
    k, v = randn(1, 206, 1, hd), randn(2, 206, 1, hd)
    k[60:100] *= ksize
    v[90:150] *= vsize if q8 else vsize / 2
    cache.write(0, k, v, full)
    q = randn(3, 6, 64, hd, dtype=dtype)
    scale = 0.05 / ksize
    got = tree_attention(q, cache, 0, roomy(batch, 16), scale=scale)
    bits = [np.tril(np.ones((6, 6), bool))]
    want, vmax, smag = R.attention(q, [R.quantised(k, q8).double()], [R.quantised(v, q8).double()], [200], [6], bits,
                                   scale)
    assert_within(got, want, R.attention_bound(want, vmax, smag, dtype))


# ---------------------------------------------------------------- batches that say something wrong
@pytest.mark.parametrize("q_start,ctx", [
    ([0, 6, 3, 9], [0, 0, 0]),    # starts that go back
    ([0, 9, 9, 11], [0, 0, 0]),   # a sequence behind the tensors' rows
    ([0, 4, 4, 9], [0, -1, 0]),   # a context of less than nothing, without new tokens
    ([-2, 0, 5, 9], [0, 0, 0]),   # a start before the first row
])
def test_every_operator_reports_every_bad_sequence(q_start, ctx):
    from m3_avm_b200.attention import KvBatch, KvCache, tree_attention

    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    cache = KvCache(8, 1, 2, 64, 16, 3)
    batch = KvBatch(i32(q_start), i32(ctx), i32([[0], [1], [2]]), 9, 9, 16)
    x = randn(1, 9, 2, 64)
    cache.write(0, x, x, batch)
    assert status() == 16
    k = torch.full_like(x, 7.0)
    cache.read(0, batch, k_out=k, v_out=torch.full_like(x, 7.0))
    assert status() == 16
    tree_attention(randn(2, 9, 4, 64), cache, 0, batch)
    assert status() == 16
    last = slice(q_start[2], min(q_start[3], 9)) if q_start[3] <= 9 else slice(9, 9)
    assert torch.equal(k[last].cpu(), R.quantised(x[last], True))


@pytest.mark.parametrize("n", [300, 1024, 1025, 5000])
def test_cache_of_many_sequences(n):
    """More sequences than a CTA has threads, or starts in shared memory; one bad one anywhere is skipped and reported."""
    from m3_avm_b200.attention import KvBatch, KvCache

    r = np.random.default_rng(n)
    ctx, new = [int(x) for x in r.integers(0, 40, n)], [int(x) for x in r.integers(0, 3, n)]
    new[n - 2] = 2
    batch, pages, table, start = R.make_batch(ctx, new, 16, seed=n)
    cache = KvCache(8, 1, 1, 64, 16, pages)
    x = randn(1, sum(new), 1, 64)
    want = R.quantised(x, True)
    for bad in (None, n - 2, 0):
        cache.pool.zero_()
        b = batch
        if bad is not None:
            wrong = torch.tensor(ctx, dtype=torch.int32)
            wrong[bad] = -5
            b = KvBatch(batch.q_start, wrong.cuda(), batch.page_table, batch.n_tokens, batch.max_tokens, batch.max_len)
        cache.write(0, x, x, b)
        assert status() == (0 if bad is None else 16)
        k = torch.full_like(x, 7.0)
        cache.read(0, b, k_out=k, v_out=torch.empty_like(x))
        assert status() == (0 if bad is None else 16)
        skipped = torch.zeros(sum(new), dtype=torch.bool)
        if bad is not None:
            skipped[int(start[bad]):int(start[bad + 1])] = True
        assert torch.equal(k.cpu()[~skipped], want[~skipped]) and bool((k.cpu()[skipped] == 7).all())


@pytest.mark.parametrize("dtype,heads,large", [(F32, 4, False), (BF16, 4, False), (F16, 4, False), (BF16, 64, True),
                                               (F16, 64, True)])
@pytest.mark.parametrize("at", [3, 41])
@pytest.mark.parametrize("infinite", [False, True])
def test_attention_a_seen_nan_counts_however_small_its_weight(dtype, heads, large, at, infinite):
    """0 * NaN (or, in another writer's pool, an infinite scale): a position whose score is 2000 below the others', in the context and among the new tokens."""
    from m3_avm_b200.attention import KvCache, tree_attention

    batch, pages, _, _ = R.make_batch([40], [5], 16)
    cache = KvCache(8, 1, 1, 64, 16, pages)
    full = R.whole(batch, [40], [5])
    k, v = randn(1, 45, 1, 64, scale=0.1), randn(2, 45, 1, 64)
    q = randn(3, 1, 1, 64).sign().expand(5, heads, 64).to(dtype).contiguous()
    k[at] = -40.0 * q[0, :1].float()
    v[at, 0, 7] = float("nan")
    cache.write(0, k, v, full)
    if infinite:
        scales = planes(cache)[3]
        scales.copy_(torch.where(torch.isnan(scales), torch.tensor(float("inf"), dtype=F16, device="cuda"), scales))
        assert int(torch.isinf(scales).sum()) == 1
    got = tree_attention(q, cache, 0, roomy(batch, 16) if large else batch, scale=1.0)
    seen = [max(at - 40, 0) <= j for j in range(5)]
    for j in range(5):
        assert bool(torch.isnan(got[j, :, :32]).all()) == seen[j]  # the block of 32 values that the NaN took with it
        assert not bool(torch.isnan(got[j, :, 32:]).any())
