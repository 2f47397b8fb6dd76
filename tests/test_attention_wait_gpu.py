"""Waits inside attention's form of 128-row tiles that run out, on one GPU, without a fault.

With a limit of (next to) nothing the waits between the kernel's warps give up wherever they happen to be.  The kernel
has to end by itself, with its copies and products settled, report it, and leave NaN in the rows that it did not work
out: never a number from a tile that was not there.  The limit is a host setting; nothing hangs, traps or faults.
"""
import pytest
import torch

from m3_avm_b200 import matvec_quant as MQ
from tests.test_serving_gpu import attention_case, status

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture()
def limit():
    status()
    yield lambda us: MQ.set_tuning("attn_wait_us", us)
    MQ.set_tuning("attn_wait_us", 2000000)
    torch.cuda.synchronize()
    status()


@pytest.mark.parametrize("dtype,q8,hd", [(BF16, True, 128), (F16, True, 128), (BF16, False, 64), (F16, False, 64)])
def test_waits_that_run_out(limit, dtype, q8, hd):
    from m3_avm_b200.attention import tree_attention

    # pieces cut over many CTAs, whole ones, and CTAs with several pieces
    got, _, _, (q, cache, batch, mask) = attention_case(q8, dtype, 64, 2, hd, 16, [5000, 3, 70, 600], [9, 1, 40, 64], True,
                                                        seed=8, large=True)
    assert status() == 0
    given_up = 0
    for us in (0, 1, 2, 5, 0):
        limit(us)
        for _ in range(4):
            out = tree_attention(q, cache, 1, batch, mask=mask)
            torch.cuda.synchronize()
            nan = torch.isnan(out)
            assert bool((nan | (out == got)).all())
            assert bool(nan.any()) <= (status() != 0)
            given_up += int(nan.any())
        if us == 0:
            assert given_up
            limit(0)
            tree_attention(q, cache, 1, batch, mask=mask)
            assert status() == 64
        limit(2000000)
        for _ in range(2):
            assert torch.equal(tree_attention(q, cache, 1, batch, mask=mask), got)
        assert status() == 0


def test_other_calls_neither_report_nor_clear_what_the_serving_operators_met(limit):
    import numpy as np

    from m3_avm_b200 import model
    from m3_avm_b200.attention import KvBatch, tree_attention
    from m3_avm_b200.decoder import GpuDecoder

    _, _, _, (q, cache, batch, mask) = attention_case(True, BF16, 64, 2, 128, 16, [5000, 3], [9, 1], True, seed=8, large=True)
    dec = GpuDecoder.synthetic(model.LlamaShape(n_layers=1, hidden=2048, ffn=2048, n_heads=32, n_kv_heads=8, vocab=4096,
                                                rope_theta=500000.0, embd_dtype=12, attn_dtype=2, gate_up_dtype=8,
                                                down_dtype=14, head_dtype=14), 3, max_pos=16)
    want = dec.prefill_logits(np.arange(4))
    dec.clear_kv_cache()
    limit(0)
    tree_attention(q, cache, 1, batch, mask=mask)  # waits that run out
    few = KvBatch(batch.q_start, batch.ctx_len, batch.page_table, batch.n_tokens, 3, batch.max_len)
    tree_attention(q, cache, 1, few)               # a sequence past the call's limits
    torch.cuda.synchronize()
    assert np.array_equal(dec.prefill_logits(np.arange(4)), want)  # not "a weight copy did not complete"
    dec.close()
    assert status() == 64 | 16
    assert status() == 0


def test_limits_out_of_range_are_refused():
    from m3_avm_b200 import _lib

    for bad in (-1, 60000001):
        with pytest.raises(_lib.M3GError):
            MQ.set_tuning("attn_wait_us", bad)
