"""Scores beyond the float32 resolution of a soft-max's exponent: the largest key takes all, ties share, whatever the number of rows."""
import pytest
import torch

from tests import ops_reference as R
from tests.test_gpu_ops import TYPES, _gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


def _case(tq, tk, d, size, dtype):
    """Integer scores times `size`: products and sums are exact, differences of at least size / sqrt(d) leave one key (or equal ones) its row."""
    t = TYPES[dtype]
    q = torch.randint(-3, 4, (1, tq, 1, d), generator=_gen(tq)).float()
    q[..., 0] = 1.0
    k = torch.randint(-3, 4, (1, tk, 1, d), generator=_gen(tk)).float()
    v = torch.randn(1, tk, 1, d, generator=_gen(d)).to(t)
    root = 2.0 ** (size // 2)
    return (q * root).to(t), (k * 2.0 ** (size - size // 2)).to(t), v


def _want(q, k, v, tk):
    s = torch.einsum('qd,kd->qk', q[0, :, 0].double(), k[0, :, 0].double())
    best = (s == s.max(-1, keepdim=True).values).double()
    return (best / best.sum(-1, keepdim=True)) @ v[0, :, 0].double()


@pytest.mark.parametrize('dtype,size', [('f16', 16), ('f16', 22), ('bf16', 24), ('bf16', 40), ('bf16', 90), ('f32', 30), ('f32', 90)])
@pytest.mark.parametrize('tq,tk,d', [(3, 200, 64), (64, 500, 128), (70, 500, 128), (300, 130, 64), (100, 4000, 128), (130, 200, 80)])
def test_huge_scores(ops, tq, tk, d, dtype, size):
    q, k, v = _case(tq, tk, d, size, dtype)
    want = _want(q, k, v, tk)
    for scale in (1.0, -1.0):
        got = ops.cross_attention(q.cuda(), (k * scale).cuda(), v.cuda(), scale=scale).cpu().double()[0, :, 0]
        assert bool(torch.isfinite(got).all())
        # equal probabilities of at most tk keys: a half step of the result and (tk / 8 + 64) u twice
        bound = R.HALF_STEP[q.dtype] * want.abs() + 2 * ((tk / 8 + 64) * R.U + 2.0 ** -16) * 4.5
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())


@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
@pytest.mark.parametrize('tq', [3, 40, 100, 300])
def test_huge_scores_over_the_cache(ops, tq, dtype):
    d, tk = 64, 320
    cache = ops.kv8_cache(1, 1, tk, d)
    g = _gen(tq)
    q = torch.randint(-3, 4, (1, tq, 1, d), generator=g).float()
    k = torch.randint(-3, 4, (1, 1, tk, d), generator=g).float()
    v = torch.randint(-7, 8, (1, 1, tk, d), generator=g).float()
    cache[0].copy_(k.to(torch.float8_e4m3fn))
    cache[1].copy_(v.to(torch.float8_e4m3fn))
    cache[2].fill_(2.0 ** 40)
    t = TYPES[dtype]
    q = (q * 8).to(t)
    lens = torch.tensor([tk], dtype=torch.int32).cuda()
    want = _want(q, k.transpose(1, 2), v.transpose(1, 2), tk)
    got = ops.kv8_attention(q.cuda(), *cache, lens, scale=1.0).cpu().double()[0, :, 0]
    assert bool(torch.isfinite(got).all())
    bound = R.HALF_STEP[t] * want.abs() + 2 * ((tk / 8 + 64) * R.U + 2.0 ** -16) * 7
    assert bool(((got - want).abs() <= bound).all())
