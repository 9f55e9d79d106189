"""Infinities in admitted values of cross_attention: with a positive weight, however small, they reach the result as what they are."""
import math

import pytest
import torch

from tests import ops_reference as R
from tests.test_gpu_ops import TYPES, _close, _cross_case, _gen
from tests.test_gpu_ops_precision import _tail_bound, _two_terms

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


def _check(ops, q, k, v, admitted, scale=None, **kw):
    """What the finite values give, and in a column with admitted infinities these: NaN where both signs or a NaN meet."""
    n, tq, heads, d = q.shape
    tk, kv_heads = k.shape[1:3]
    got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), scale=scale, **kw)
    x = v.double().transpose(1, 2)                                                     # [n, Hkv, tk, d]
    fine = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    want, weight, size = R.attention(q, k.double().transpose(1, 2), fine, admitted[:, None].expand(n, tq, tk), d ** -0.5 if scale is None else scale)
    vmax = float(fine.abs().max())
    bound = _tail_bound(want, weight, size, d, tk, vmax) if q.dtype == torch.float16 else _two_terms(want, weight, size, d, tk, q.dtype, False)
    seen = lambda what: (what & admitted[:, None, :, None]).any(2).repeat_interleave(heads // kv_heads, 1)[:, None].expand(n, tq, heads, d)  # noqa: E731
    up, down, nan = seen(x == math.inf), seen(x == -math.inf), seen(x.isnan())
    want = torch.where(up, math.inf, want)
    want = torch.where(down, -math.inf, want)
    want = torch.where(nan | (up & down), math.nan, want)
    _close(got, want, bound, 'out')


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('n,tq,tk,heads,kv_heads,d', [(1, 1, 1, 1, 1, 64), (2, 1, 47, 4, 2, 64), (2, 10, 334, 4, 4, 128), (3, 20, 75, 2, 1, 40), (2, 70, 130, 4, 2, 64),
                                                      (1, 3, 2600, 2, 2, 64), (1, 200, 2100, 2, 1, 128), (2, 130, 90, 1, 1, 80), (64, 256, 70, 8, 8, 64)])
def test_admitted_infinities(ops, n, tq, tk, heads, kv_heads, d, dtype):
    if dtype == 'f32':
        n = min(n, 4)
    q, kv = _cross_case(n + tq + tk, n, tq, tk, heads, kv_heads, d, dtype)
    k, v = kv[:, :, 0], kv[:, :, 1].clone()
    lens = torch.randint((tk + 1) // 2, tk + 1, (n,), generator=_gen(tk), dtype=torch.int32)
    pad = torch.rand(n, tk, generator=_gen(n)) < 0.1
    pad[:, 0] = False
    for b in range(n):
        last = int(lens[b]) - 1
        v[b, 0, 0, 1] = math.inf                                                       # (also where one key is all there is)
        v[b, last // 2, -1, 3] = -math.inf
        v[b, 0, :, 5] = math.inf
        v[b, last, :, 5] = math.inf
        v[b, 0, :, 6] = math.inf
        v[b, last, 0, 6] = -math.inf
        v[b, last // 3, 0, d - 1] = math.nan
        v[b, last, 0, d - 2] = -math.inf
    admitted = (torch.arange(tk) < lens[:, None]) & ~pad
    _check(ops, q, k, v, admitted, lens=lens.cuda(), pad=pad.cuda())
    _check(ops, q, k, v, torch.arange(tk).expand(n, tk) < lens[:, None], lens=lens.cuda())


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tq,tk', [(1, 200), (33, 200), (100, 200), (2, 3000), (100, 3000)])
def test_infinities_of_little_weight(ops, tq, tk, dtype):
    """A key far below and far above the others in scores, first or last, so that sums of infinities are scaled and joined."""
    d = 64
    for at, score in ((0, -300.0), (tk - 1, -300.0), (0, -30.0), (tk // 2, 40.0), (0, 0.0)):
        q = torch.zeros(1, tq, 1, d)
        q[..., 0] = 1.0
        k = torch.zeros(1, tk, 1, d)
        k[0, :, 0, 0] = torch.arange(tk) % 5 / 4
        k[0, at, 0, 0] = score
        v = torch.randn(1, tk, 1, d, generator=_gen(tq))
        v[0, at, 0, 9] = math.inf
        v[0, at, 0, 11] = -math.inf
        t = TYPES[dtype]
        _check(ops, q.to(t), k.to(t), v.to(t), torch.ones(1, tk, dtype=torch.bool), scale=1.0)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tq', [3, 90])
def test_rows_of_nan_beside_infinities(ops, tq, dtype):
    """A query row of NaN is NaN, its neighbours have their infinities."""
    q, kv = _cross_case(tq, 1, tq, 100, 2, 2, 64, dtype)
    kv[0, 7, 1, 0, 2] = math.inf
    q[0, 1] = math.nan
    got = ops.cross_attention(q.cuda(), kv[:, :, 0].cuda(), kv[:, :, 1].cuda()).cpu()
    assert bool(got[0, 1].isnan().all())
    rest = got[0, [i for i in range(tq) if i != 1]]
    assert bool((rest[:, 0, 2] == math.inf).all()) and bool(torch.isfinite(rest[:, 1]).all()) and int(torch.isinf(rest).sum()) == tq - 1
