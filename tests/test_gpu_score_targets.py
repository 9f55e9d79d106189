"""asr_score and asr_loss on targets outside the vocabulary: 0 in the sum (the one-hot row of such a label is all zeros, model.py:350-360), NaN token by token."""
import math

import numpy as np
import pytest

from oracle import asr_oracle as O
from tests.helpers import product_config, tiny_config, tiny_inputs

pytestmark = pytest.mark.gpu


def test_targets_outside_the_vocabulary_in_score_and_loss():
    from asr_amd.model import Engine
    ocfg = tiny_config()
    V = ocfg.dst_vocab_size
    X = tiny_inputs((60, 90, 75), seed=62)
    Y = np.array([[5, V, -4, 7, 3], [V - 1, 3, 0, 0, 0], [1 << 30, -(1 << 31), 0, 9, V + 3]], np.int32)
    eng = Engine(product_config(ocfg), 0)
    eng.load_weights(O.random_weights(ocfg, seed=61, bias_scale=0.1))
    try:
        lp = eng.score(X, Y)[0].astype(np.float64)
        assert np.array_equal(np.isnan(lp), Y >= V)
        assert (lp[(Y <= 0)] == 0.0).all() and (lp[(Y > 0) & (Y < V)] < 0.0).all()
        loss = eng.loss(X, Y)
        counted = (Y > 0) & (Y < V)
        rows = int(counted.sum())
        # row by row both are float32 evaluations of the same logits: (3 ln V + 40) 2^-24 and the value's own half step, on each side
        assert abs(-lp[counted].sum() - loss) <= rows * 2 * 2.0 ** -24 * (3 * math.log(V) + 40 + 2 * np.abs(lp[counted]).max())
    finally:
        eng.close()
