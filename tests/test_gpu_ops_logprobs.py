"""token_logprobs where its kernel changes its width - one wave, four, sixteen - against 64 bits, within a bound for the width that is taken."""
import math

import pytest
import torch

from tests import ops_reference as R
from tests.test_gpu_ops import TYPES, _close, _gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


def _threads(rows, vocab, dtype):
    chunks = vocab // (4 if dtype == 'f32' else 8)                 # 16-byte loads of a row
    return 1024 if rows <= 256 and chunks >= 2048 else 64 if chunks <= (1024 if rows >= 1024 else 256) else 256


def _bound(x, threads):
    """Of log p, absolute, and of the entropy times 1 + H.  Every e^(x-m) is off by (3 |x - m| + 4) u of itself (the difference, log2 e, the product,
    exp2), weighted by p at most (3 (ln V + 1) + 4) u.  A thread adds V / threads + 2 of them one after the other, a wave 6 more, a workgroup 4; a term is scaled at most once for
    each group of four loads and in both joins, each time by a factor off by 5 u besides 3 u for each unit of the maxima's difference, which add up to at most the span of the
    row.  ln S is rounded twice, x - m and the last subtraction once each."""
    x = x.double()
    vocab = x.shape[-1]
    finite = torch.isfinite(x)
    span = torch.where(finite, x, torch.full_like(x, -math.inf)).max(-1).values - torch.where(finite, x, torch.full_like(x, math.inf)).min(-1).values
    span = torch.where(torch.isfinite(span), span, torch.zeros_like(span))
    strip = vocab / threads + 2
    return R.U * (3 * (math.log(vocab) + 1) + 4 + strip + 10 + 5 * (strip / 16 + 3) + 5 * span + 4 * math.log(vocab))


CASES = [(3, 1023, 'f32'), (3, 1028, 'f32'), (3, 2047, 'bf16'), (3, 2056, 'f16'), (1023, 4096, 'f32'), (1024, 4096, 'f32'), (1024, 4100, 'f32'),
         (1024, 8191, 'bf16'), (1024, 8200, 'f16'), (1023, 8191, 'f16'), (256, 8191, 'f32'), (256, 8192, 'f32'), (257, 8192, 'f32'), (256, 16384, 'bf16'),
         (257, 16384, 'bf16'), (2, 16383, 'f16')]


@pytest.mark.parametrize('rows,vocab,dtype', CASES)
def test_token_logprobs_at_the_borders_of_its_widths(ops, rows, vocab, dtype):
    g = _gen(rows + vocab)
    x = torch.randn(rows, vocab, generator=g) * 3
    x[1].masked_fill_(torch.rand(vocab, generator=g) < 0.5, -math.inf)
    x = x.to(TYPES[dtype])
    tokens = torch.randint(-1, vocab, (rows,), generator=g)
    lp, h, tops, at = ops.token_logprobs(x.cuda(), tokens.cuda(), top=6)
    want_lp, want_h, want_tops, want_at = R.token_logprobs(x, tokens, 6)
    bound = _bound(x, _threads(rows, vocab, dtype))
    _close(lp, want_lp, bound, 'log p')
    _close(h, want_h, bound * (1 + want_h), 'entropy')
    _close(tops, want_tops, bound[:, None], 'alternatives')
    assert torch.equal(at.cpu().long(), want_at)
