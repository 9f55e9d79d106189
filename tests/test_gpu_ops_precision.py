"""Attention of asr_amd.ops against 64 bits within bounds that know in how many terms each path holds its probabilities: losing one of them is seen."""
import pytest
import torch

from tests import ops_reference as R
from tests.test_gpu_ops import TYPES, _close, _cross_case, _gen, _loud_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


def _two_terms(out, weight, size, d, tk, dtype, codes):
    """R.attention_bound without its half step of a 16-bit probability: one held as the sum of two terms, each rounded to the nearest, is off by the
    square of a half step (bf16, and every type over codes: 2^-16; float16: 2^-22), a float32 one over three terms by nothing that counts.  What is left
    is the scores' error, the exponential's, the sums' and the result's own rounding."""
    p = 2 * (d + 8) * R.U * size + 2.0 ** -22 + (tk / 8 + 64) * R.U
    if dtype != torch.float32:
        p = p + R.HALF_STEP[torch.bfloat16 if codes else dtype] ** 2
    return 2 * p * weight + R.HALF_STEP[dtype] * out.abs() + 1e-30


def _check_cross(ops, q, k, v, lens, pad):
    n, tq, _, d = q.shape
    tk = k.shape[1]
    admitted = (torch.arange(tk) < lens[:, None]) & ~pad
    got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), lens=lens.cuda(), pad=pad.cuda())
    want, weight, size = R.attention(q, k.double().transpose(1, 2), v.double().transpose(1, 2), admitted[:, None].expand(n, tq, tk), d ** -0.5)
    _close(got, want, _two_terms(want, weight, size, d, tk, q.dtype, False), 'out')


def _check_kv8(ops, q, cache, lens, causal):
    n, tq, _, d = q.shape
    tk = cache[0].shape[2]
    got = ops.kv8_attention(q.cuda(), *cache, lens.cuda(), causal=causal)
    k, v = (R.values_of(c) * s.cpu().double().repeat_interleave(64, -1)[..., None] for c, s in (cache[::2], cache[1::2]))
    last = lens.long()[:, None].expand(n, tq)
    if causal:
        last = last - tq + 1 + torch.arange(tq)
    want, weight, size = R.attention(q, k, v, torch.arange(tk) < last[..., None], d ** -0.5)
    _close(got, want, _two_terms(want, weight, size, d, tk, q.dtype, True), 'out')


CROSS = [(2, 1, 47, 2, 2, 64), (2, 10, 334, 4, 2, 64), (1, 40, 300, 2, 2, 128), (1, 41, 300, 2, 2, 128), (2, 61, 300, 4, 2, 64), (2, 64, 300, 2, 2, 64), (2, 65, 300, 2, 2, 64), (1, 200, 1100, 2, 1, 80),
         (1, 4, 4000, 2, 1, 64), (64, 256, 70, 8, 8, 64)]


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('shape', CROSS, ids=str)
def test_cross_attention_holds_two_terms_of_a_probability(ops, shape, dtype):
    n, _, tk = shape[:3]
    if dtype == 'f32' and n == 64:
        n, shape = 4, (4,) + shape[1:]                      # (float32 has no kernel of its own for many rows)
    q, kv = _cross_case(sum(shape) + 1, *shape, dtype)
    lens = torch.randint((tk + 1) // 2, tk + 1, (n,), generator=_gen(tk), dtype=torch.int32)
    pad = torch.rand(n, tk, generator=_gen(n)) < 0.1
    _check_cross(ops, q, kv[:, :, 0], kv[:, :, 1], lens, pad)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('n,tq,heads,kv_heads,capacity,d', [(2, 1, 4, 2, 192, 64), (2, 10, 4, 2, 320, 128), (2, 20, 4, 2, 320, 64), (2, 21, 4, 2, 320, 64), (2, 33, 4, 2, 320, 64),
                                                            (2, 100, 4, 2, 320, 128), (1, 300, 2, 2, 1088, 80), (1, 2, 8, 1, 4096, 128),
                                                            (64, 128, 16, 8, 192, 64)])
def test_kv8_attention_holds_two_terms_of_a_probability(ops, n, tq, heads, kv_heads, capacity, d, causal, dtype):
    g = _gen(n + tq + capacity)
    if dtype != 'bf16' and n == 64:
        n = 4
    cache = _loud_cache(ops, g, n, kv_heads, capacity, d)
    q = torch.randn(n, tq, heads, d, generator=g).to(TYPES[dtype])
    lens = torch.randint(max(tq, capacity // 2), capacity + 1, (n,), generator=g, dtype=torch.int32)
    _check_kv8(ops, q, cache, lens, causal)


# ---- float16: the soft-max's tail --------------------------------------------------------------------------------------------
def _tail_bound(out, weight, size, d, tk, vmax):
    """_two_terms for float16 K and V, whose terms have a smallest step of 2^-24: the largest probability of a row enters as at least 2^7, so each is off by
    at most 2^-25 / 2^7 = 2^-32 of it besides what is relative, in the sum over V and, where the row sum has the unrounded ones, once more in the weights."""
    return _two_terms(out, weight, size, d, tk, torch.float16, False) + 2 * tk * 2.0 ** -32 * vmax


@pytest.mark.parametrize('nats', [10.0, 14.0, 15.0, 16.0, 17.5, 19.0])
@pytest.mark.parametrize('tq,tk,d', [(1, 4097, 64), (16, 300, 64), (40, 4097, 128), (70, 4097, 64), (200, 1000, 128), (130, 900, 80)])
def test_float16_attention_keeps_far_keys(ops, tq, tk, d, nats):
    """One key far above thousands of others with a V of its own: their share is small, but not lost (1.0e-4 of 4096 keys at 17.5 nats)."""
    q = torch.zeros(1, tq, 1, d)
    q[..., 0] = 0.5
    k = torch.zeros(1, tk, 1, d)
    k[0, 1:, 0, 0] = -nats / 4                               # (times 0.5, times a scale of 8: exact)
    k[0, :, 0, 1:] = torch.randn(tk, d - 1, generator=_gen(tk))
    v = torch.zeros(1, tk, 1, d)
    v[0, 1:, 0] = 1024 + 256 * torch.randint(0, 3, (tk - 1, d), generator=_gen(d))         # (no result below float16's normal ones)
    q, k, v = q.half(), k.half(), v.half()
    got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), scale=8.0)
    want, weight, size = R.attention(q, k.double().transpose(1, 2), v.double().transpose(1, 2), torch.ones(1, tq, tk, dtype=torch.bool), 8.0)
    _close(got, want, _tail_bound(want, weight, size, d, tk, 1536.0), 'out')


@pytest.mark.parametrize('shape', CROSS, ids=str)
def test_cross_attention_of_float16_holds_two_terms_of_a_probability(ops, shape):
    n, tq, tk, _, _, d = shape
    q, kv = _cross_case(sum(shape) + 1, *shape, 'f16')
    lens = torch.randint((tk + 1) // 2, tk + 1, (n,), generator=_gen(tk), dtype=torch.int32)
    got = ops.cross_attention(q.cuda(), kv[:, :, 0].cuda(), kv[:, :, 1].cuda(), lens=lens.cuda())
    k, v = (kv[:, :, i].double().transpose(1, 2) for i in (0, 1))
    want, weight, size = R.attention(q, k, v, (torch.arange(tk) < lens[:, None])[:, None].expand(n, tq, tk), d ** -0.5)
    _close(got, want, _tail_bound(want, weight, size, d, tk, float(v.abs().max())), 'out')


def test_float16_attention_of_growing_scores(ops):
    """Scores that grow by less and by more than the slack of the running maximum from tile to tile: probabilities stay finite."""
    tk, d = 2000, 64
    for step in (0.001, 0.02, 0.3):
        q = torch.zeros(1, 70, 1, d)
        q[..., 0] = 1.0
        k = torch.zeros(1, tk, 1, d)
        k[0, :, 0, 0] = torch.arange(tk) * step
        v = torch.randn(1, tk, 1, d, generator=_gen(1))
        q, k, v = q.half(), k.half(), v.half()
        for rows in (1, 20, 70):
            got = ops.cross_attention(q[:, :rows].cuda(), k.cuda(), v.cuda(), scale=1.0)
            want, weight, size = R.attention(q[:, :rows], k.double().transpose(1, 2), v.double().transpose(1, 2), torch.ones(1, rows, tk, dtype=torch.bool), 1.0)
            _close(got, want, _tail_bound(want, weight, size, d, tk, float(v.abs().max())), 'out')
