"""Decode steps of sequences with different numbers of new tokens: kv8_append and causal kv8_attention with the same counts."""
import math

import pytest
import torch

from tests import ops_reference as R
from tests.test_gpu_ops import TYPES, _check_append, _close, _gen, _loud_cache
from tests.test_gpu_ops_precision import _two_terms

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


def _check(ops, q, cache, lens, counts, causal, **kw):
    n, tq, heads, d = q.shape
    tk = cache[0].shape[2]
    got = ops.kv8_attention(q.cuda(), *cache, lens.cuda(), causal=causal, counts=counts.cuda(), **kw)
    k, v = (R.values_of(c) * s.cpu().double().repeat_interleave(64, -1)[..., None] for c, s in (cache[::2], cache[1::2]))
    own = counts.long().clamp(0, tq)[:, None]
    i = torch.arange(tq)
    length = lens.long().clamp(0, tk)[:, None]
    last = torch.where(i < own, length - own + i + 1 if causal else length.expand(n, tq), 0)
    fine = torch.where((i < own)[..., None, None], q.double(), 0.0)                    # (what stands behind the queries does not matter)
    want, weight, size = R.attention(fine, k, v, torch.arange(tk) < last[..., None], d ** -0.5)
    _close(got, want, _two_terms(want, weight, size, d, tk, q.dtype, True), 'out')
    assert float(got.cpu()[~(i < own)].abs().sum()) == 0.0
    return got


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tq,heads,kv_heads,capacity,d', [(1, 2, 2, 128, 64), (5, 4, 2, 256, 64), (12, 4, 4, 320, 80), (40, 4, 2, 192, 128), (90, 2, 1, 448, 64),
                                                          (150, 2, 2, 320, 128), (4, 2, 1, 4096, 64), (200, 1, 1, 4096, 128)])
def test_ragged_new_tokens_and_their_queries(ops, tq, heads, kv_heads, capacity, d, dtype):
    g = _gen(tq + d)
    n, t = 9, TYPES[dtype]
    cache = _loud_cache(ops, g, n, kv_heads, capacity, d)
    counts = torch.tensor([tq, 1, 0, tq // 2, -7, tq + 100, max(1, tq - 1), tq // 3, 2], dtype=torch.int32)
    held = torch.randint(0, capacity - tq + 1, (n,), generator=g, dtype=torch.int32)
    held[1] = held[3] = 0                                                              # nothing before the first query
    held[0] = capacity - tq
    k, v = (torch.randn(n, tq, kv_heads, d, generator=g).to(t) for _ in range(2))
    _check_append(ops, k.cuda(), v.cuda(), cache, held.cuda(), counts.cuda())
    q = torch.randn(n, tq, heads, d, generator=g).to(t)
    own = counts.long().clamp(0, tq)
    for b in range(n):
        q[b, int(own[b]):] = math.nan if b % 2 else math.inf
    lens = held + own.int()
    for causal in (True, False):
        _check(ops, q, cache, lens, counts, causal)
    out = torch.full((n, tq, heads, 2 * d), 5.0, dtype=t, device='cuda')
    _check(ops, q, cache, lens, counts, True, out=out[..., d:])
    assert bool((out[..., :d] == 5.0).all())


def test_two_row_tiles_a_wave_with_counts(ops):
    """64 sequences of 8 key heads and 256 rows each."""
    g = _gen(4)
    cache = _loud_cache(ops, g, 64, 8, 256, 64)
    q = torch.randn(64, 128, 16, 64, generator=g).bfloat16()
    counts = torch.randint(0, 129, (64,), generator=g, dtype=torch.int32)
    lens = counts + torch.randint(0, 129, (64,), generator=g, dtype=torch.int32)
    _check(ops, q, cache, lens, counts, True)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tq,kv_heads', [(6, 2), (120, 2)])
def test_all_counts_are_no_counts(ops, tq, kv_heads, dtype):
    g = _gen(tq)
    cache = _loud_cache(ops, g, 3, kv_heads, 320, 64)
    q = torch.randn(3, tq, 4, 64, generator=g).to(TYPES[dtype]).cuda()
    lens = torch.tensor([320, 7, 200], dtype=torch.int32).cuda()
    for causal in (True, False):
        a = ops.kv8_attention(q, *cache, lens, causal=causal)
        b = ops.kv8_attention(q, *cache, lens, causal=causal, counts=torch.full((3,), tq, dtype=torch.int32).cuda())
        assert torch.equal(a, b)


def test_nan_in_later_tokens_with_counts(ops):
    """NaN in a token reaches its own query and later ones alone, also where a sequence has fewer queries than rows."""
    for tq in (8, 150):
        g = _gen(tq)
        cache = _loud_cache(ops, g, 2, 1, 256, 64)
        counts = torch.tensor([tq // 2, tq], dtype=torch.int32)
        lens = torch.tensor([200, 256], dtype=torch.int32)
        for b in range(2):
            cache[1].view(torch.uint8)[b, 0, int(lens[b]) - 2, 3] = 0x7f
        q = torch.randn(2, tq, 2, 64, generator=g).bfloat16().cuda()
        got = ops.kv8_attention(q, *cache, lens.cuda(), causal=True, counts=counts.cuda()).cpu()
        for b in range(2):
            c = int(counts[b])
            lost = torch.zeros(tq, 2, 64, dtype=torch.bool)
            lost[c - 2:c, :, 3] = True
            assert torch.equal(got[b].isnan(), lost)
            assert float(got[b, c:].abs().sum()) == 0.0


def test_counts_are_checked(ops):
    cache = ops.kv8_cache(2, 1, 64, 64)
    q = torch.zeros(2, 3, 1, 64, device='cuda')
    lens = torch.ones(2, dtype=torch.int32, device='cuda')
    for bad in (lens.long(), lens[:1], lens.cpu(), lens.float()):
        with pytest.raises(ValueError):
            ops.kv8_attention(q, *cache, lens, counts=bad)
