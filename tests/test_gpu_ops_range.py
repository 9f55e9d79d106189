"""Numbers at the end of float32's range."""
import math

import pytest
import torch

from asr_amd._lib import AsrError
from tests import ops_reference as R
from tests.test_gpu_ops import TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('held', [0, 3])
def test_the_largest_finite_values_stay_finite_in_the_cache(ops, dtype, held):
    """A type's lowest value, as masks have it, and its neighbours: under a scale of 2^120 the nearest code, 256, is 2^128; they take the one below, 240."""
    t = TYPES[dtype]
    top = torch.finfo(t).max
    d = 16
    k = torch.zeros(1, 2, 1, d)
    k[0, 0, 0, :8] = torch.tensor([top, -top, 3.25e38, 3.31e38, -3.31e38, 3.0e38, 1.0e38, 1.5e36])
    k[0, 1, 0, 0] = math.inf
    k = k.to(t)
    cache = ops.kv8_cache(1, 1, 64, d)
    if held:
        ops.kv8_append(k[:, :1].expand(-1, held, -1, -1).cuda() * 2.0 ** -30, k[:, :1].expand(-1, held, -1, -1).cuda(), *cache, torch.zeros(1, dtype=torch.int32).cuda())
    ops.kv8_append(k.cuda(), k.cuda(), *cache, torch.full((1,), held, dtype=torch.int32).cuda())
    for code, scale in (cache[::2], cache[1::2]):
        assert float(scale[0, 0, 0]) == 2.0 ** 120
        got = R.values_of(code)[0, 0, held:held + 2]
        x = k[0, :, 0].double()
        want = R.to_code((x * 2.0 ** -120))
        want = torch.where(x.abs() * 2.0 ** -120 > 240, torch.copysign(torch.full_like(x, 240.0), x), want)
        assert torch.equal(got, want)
        assert bool(torch.isfinite(code.float()[0, 0, :, :] * scale[0, 0, 0]).all())
    if not held:                                                 # (sums over several such values pass float32 before they are divided)
        q = torch.zeros(1, 1, 1, d, dtype=t, device='cuda')
        out = ops.kv8_attention(q, *cache, torch.ones(1, dtype=torch.int32).cuda())
        assert bool(torch.isfinite(out).all())


def test_scales_beyond_float32_are_refused(ops):
    q = torch.zeros(1, 2, 1, 64, device='cuda')
    cache = ops.kv8_cache(1, 1, 64, 64)
    lens = torch.ones(1, dtype=torch.int32, device='cuda')
    for scale in (1e39, -1e300, math.inf, math.nan):
        for call in (lambda: ops.cross_attention(q, q, q, scale=scale), lambda: ops.kv8_attention(q, *cache, lens, scale=scale)):
            with pytest.raises((AsrError, ValueError), match='finite'):
                call()
    assert ops.cross_attention(q, q, q, scale=torch.tensor(0.5)).shape == q.shape
    assert ops.cross_attention(q, q, q, scale=2).shape == q.shape
