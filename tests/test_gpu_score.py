"""asr_score (Engine.score, Model.score): log p of every target, the entropy and the alternatives of the teacher-forced decoder against the float64 oracle
(decoder_impl, model.py:492-557) and against asr_loss, whose sum it is (model.py:350-360).

Bounds: with logits off by at most d, log p moves by at most 2 d, the entropy by at most 2 d H to first order.  d: 1e-4 of the largest logit, the
bar of the loss tests."""
import math

import numpy as np
import pytest

from oracle import asr_oracle as O
from tests.helpers import product_config, tiny_config, tiny_inputs

pytestmark = pytest.mark.gpu


def _targets(n, ty, vocab, seed):
    rng = np.random.default_rng(seed)
    Y = rng.integers(4, vocab, (n, ty)).astype(np.int32)
    for i in range(n):
        ln = int(rng.integers(1, ty + 1))
        Y[i, ln - 1] = 3
        Y[i, ln:] = 0
    return Y


def _oracle(X, Y, W, ocfg):
    Wc = O.cast_weights(W, np.float64)
    enc, _ = O.encoder(np.asarray(X, np.float64), Wc, ocfg)
    logits = O.output_logits(O.decoder(O.shift_right(Y), enc, Wc, ocfg), Wc, ocfg)
    return logits, O.log_softmax(logits)


def _check(got, X, Y, W, ocfg, top):
    logprob, entropy, tops, tokens = got
    logits, z = _oracle(X, Y, W, ocfg)
    d = 1e-4 * np.abs(logits).max()
    V = ocfg.dst_vocab_size
    picked = np.take_along_axis(z, np.clip(Y, 0, V - 1)[..., None], -1)[..., 0]
    assert np.abs(logprob - np.where(Y != 0, picked, 0.0)).max() <= 2 * d
    H = -(np.exp(z) * z).sum(-1)
    assert (np.abs(entropy - H) <= 2 * d * (1 + H)).all()
    assert tops.shape == tokens.shape == Y.shape + (top,)
    if top:
        want = -np.sort(-z, -1)[..., :top]
        assert np.abs(tops - want).max() <= 2 * d
        assert np.abs(np.take_along_axis(z, tokens.astype(np.int64), -1) - want).max() <= 4 * d     # (a swap only among nearly equal ones)
        assert all(len(set(r)) == top for r in tokens.reshape(-1, top).tolist())


@pytest.mark.parametrize('precision', [None, 'f32', 'f32_bf16x6'])
@pytest.mark.parametrize('cfg,lens,ty,top', [
    (dict(), (60, 90, 75), 7, 5), (dict(tie_embedding_and_softmax=True, ff_activation='relu'), (100, 40), 1, 32), (dict(), (50,), 20, 0),
    (dict(hidden_units=256, num_heads=4, num_blocks=3, dst_vocab_size=300), (150, 200, 120, 90, 201), 60, 10)])
def test_score_matches_the_oracle_and_adds_up_to_the_loss(cfg, lens, ty, top, precision):
    from asr_amd.model import Engine
    ocfg = tiny_config(**cfg)
    W = O.random_weights(ocfg, seed=61, bias_scale=0.1)
    X, Y = tiny_inputs(lens, seed=62), _targets(len(lens), ty, ocfg.dst_vocab_size, 63)
    eng = Engine(product_config(ocfg, precision=precision), 0)
    eng.load_weights(W)
    try:
        got = eng.score(X, Y, top)
        _check(got, X, Y, W, ocfg, top)
        loss = eng.loss(X, Y)
        # row by row both are float32 evaluations of the same logits: (3 ln V + 40) 2^-24 and the value's own half step, on each side
        rows = int((Y != 0).sum())
        assert abs(-got[0].astype(np.float64).sum() - loss) <= rows * 2 * 2.0 ** -24 * (3 * math.log(ocfg.dst_vocab_size) + 40 + 2 * np.abs(got[0]).max())
        for a, b in zip(eng.score(X, Y, top), got):
            assert np.array_equal(a, b)
    finally:
        eng.close()


def test_score_of_padding_and_tokens_outside_the_vocabulary():
    from asr_amd.model import Engine
    ocfg = tiny_config()
    W = O.random_weights(ocfg, seed=61, bias_scale=0.1)
    X = tiny_inputs((60, 90), seed=62)
    Y = np.array([[5, 50, -4, 3, 0], [0, 0, 0, 0, 0]], np.int32)
    eng = Engine(product_config(ocfg), 0)
    eng.load_weights(W)
    try:
        lp, h, tops, tokens = eng.score(X, Y, 2)
        assert math.isnan(lp[0, 1]) and lp[0, 2] == 0.0 and lp[0, 4] == 0.0 and lp[0, 0] < 0.0 and lp[0, 3] < 0.0 and (lp[1] == 0.0).all()
        assert np.isfinite(h).all() and np.isfinite(tops).all() and ((tokens >= 0) & (tokens < 50)).all()
        empty = eng.score(X[:0], Y[:0], 2)
        assert [a.shape for a in empty] == [(0, 5), (0, 5), (0, 5, 2), (0, 5, 2)]
    finally:
        eng.close()


def test_score_over_towers():
    from asr_amd.model import Transformer
    ocfg = tiny_config()
    W = O.random_weights(ocfg, seed=64, bias_scale=0.1)
    X, Y = tiny_inputs((60, 90, 75, 33, 80), seed=65), _targets(5, 9, ocfg.dst_vocab_size, 66)
    m = Transformer(product_config(ocfg, 2), 2, devices=[0])
    m.build_test_model()
    m.restore(W)
    try:
        got = m.score(X, Y, 3)
        for (a, b) in O.expand_shards(5, 2):
            _check([x[a:b] for x in got], X[a:b], Y[a:b], W, ocfg, 3)
    finally:
        m.close()


def test_score_refuses():
    from asr_amd._lib import AsrError
    from asr_amd.model import Engine
    ocfg = tiny_config()
    eng = Engine(product_config(ocfg), 0)
    X, Y = tiny_inputs((60, 90), seed=62), _targets(2, 4, 50, 1)
    try:
        with pytest.raises(AsrError):
            eng.score(X, Y)                                      # no weights yet
        eng.load_weights(O.random_weights(ocfg, seed=61, bias_scale=0.1))
        for bad in (lambda: eng.score(X, Y, 33), lambda: eng.score(X, Y, -1), lambda: eng.score(X[..., :16], Y), lambda: eng.score(X, Y[:, :0])):
            with pytest.raises(AsrError):
                bad()
        with pytest.raises(ValueError):
            eng.score(X, Y[:1])
        assert eng.score(X, Y)[0].shape == (2, 4)
    finally:
        eng.close()
