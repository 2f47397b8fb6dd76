"""m3g_decoder_score: a prompt's log probabilities against those of the logits that forward_one returns, in 64 bits."""
import math

import numpy as np
import pytest

from m3_avm_b200 import model

pytestmark = pytest.mark.gpu

SHAPE = model.LlamaShape(n_layers=2, hidden=2048, ffn=2048, n_heads=32, n_kv_heads=8, vocab=4096,
                         rope_theta=500000.0, embd_dtype=12, attn_dtype=2, gate_up_dtype=8, down_dtype=14,
                         head_dtype=14)


@pytest.fixture(scope="module")
def dec():
    from m3_avm_b200.decoder import GpuDecoder

    d = GpuDecoder.synthetic(SHAPE, 3, max_pos=48)
    yield d
    d.close()


def log_softmax(rows):
    x = np.asarray(rows, np.float64)
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def tolerances(x):
    """The terms 2^t, t = x log2(e) - m: t off by 2^-24 (|x| + |m|), ex2 by 2^-22, their sum by (n / 512 + 32) 2^-24;
    a log probability adds roundings of its own size, the entropy sums (t - m) times that."""
    fin, n = float(np.abs(x).max()), x.shape[-1]
    z = 2.0 ** -22 + (n / 512 + 32) * 2.0 ** -24 + 2 * 2.0 ** -23 * fin
    own = 2.0 ** -22 * (2 * fin + math.log(n))
    return z + own, z * (2 + 2 * fin + math.log(n)) + own


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("before,n,k", [(0, 1, 1), (0, 7, 5), (9, 30, 32), (47, 1, 0), (0, 48, 3)])
def test_score_is_the_log_softmax_of_each_steps_logits(dec, graph, before, n, k):
    rng = np.random.default_rng(n)
    past, tokens = rng.integers(0, SHAPE.vocab, before), rng.integers(0, SHAPE.vocab, n)
    dec.set_graph(graph)
    dec.clear_kv_cache()
    if before:
        dec.prefill_logits(past)
    got = dec.score(tokens, n_top=k)
    assert dec.pos == before + n
    pick = int(dec.tokens(before + n, 1)[0])
    dec.clear_kv_cache()
    if before:
        dec.prefill_logits(past)
    x = np.stack([dec.forward_one(int(t)) for t in tokens])
    assert pick == int(np.argmax(x[-1]))
    lp = log_softmax(x)
    tol, etol = tolerances(x)
    follows = np.append(tokens[1:], pick)
    assert np.abs(got.logprob - lp[np.arange(n), follows]).max() <= tol
    assert np.abs(got.entropy + (np.exp(lp) * lp).sum(-1)).max() <= etol
    if k:
        order = np.argsort(-x, axis=-1, kind="stable")[:, :k]
        assert np.array_equal(got.top_ids, order)
        assert np.abs(got.top_logprobs - np.take_along_axis(lp, order, -1)).max() <= tol
    else:
        assert got.top_ids is None and got.top_logprobs is None


def test_score_leaves_the_decoder_as_prefill_does(dec):
    prompt = np.random.default_rng(1).integers(0, SHAPE.vocab, 12)
    dec.set_graph(True)
    dec.clear_kv_cache()
    want = dec.generate(prompt, 10)
    dec.clear_kv_cache()
    dec.score(prompt[:5])
    twice = dec.score(prompt[5:], n_top=2)
    got = dec.generate([], 10)
    assert np.array_equal(got, want) and int(twice.top_ids[-1, 0]) == int(want[0])
    assert float(twice.logprob[-1]) == float(twice.top_logprobs[-1, 0])


def test_score_refuses(dec):
    from m3_avm_b200._lib import M3GError

    dec.clear_kv_cache()
    for tokens, k in (([SHAPE.vocab], 0), ([1] * 49, 0), ([1], 33), ([1], -1)):
        with pytest.raises(M3GError):
            dec.score(tokens, n_top=k)
        assert dec.pos == 0
    empty = dec.score([], n_top=2)
    assert empty.logprob.shape == (0,) and empty.top_ids.shape == (0, 2) and dec.pos == 0
