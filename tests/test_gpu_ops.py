"""asr_amd.ops on the GPU against tests/ops_reference.py (64 bits on the CPU) within its derived bounds: sizes from one to many tiles, odd ones,
strides, masks that leave rows empty, values that must not matter, other streams, captured graphs, and a run of the operators together."""
import math

import pytest
import torch

from tests import ops_reference as R

pytestmark = pytest.mark.gpu
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _close(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ': NaN in other places'
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what + ': infinities'
    fine = torch.isfinite(want)
    assert bool(torch.isfinite(got[fine]).all()), what + ': not finite'
    d = (got - want).abs()[fine]
    b = bound.expand(want.shape)[fine]
    worst = float((d / b).max()) if d.numel() else 0.0
    assert worst <= 1.0, '%s: %.3g times its bound' % (what, worst)


# ---- token_logprobs ----------------------------------------------------------------------------------------------------
def _check_logprobs(ops, logits, tokens, top, ordered=True):
    lp, h, tops, at = ops.token_logprobs(logits, tokens, top=top)
    assert lp.dtype == h.dtype == tops.dtype == torch.float32 and at.dtype == torch.int32
    want_lp, want_h, want_tops, want_at = R.token_logprobs(logits.reshape(-1, logits.shape[-1]), tokens.reshape(-1).cpu(), top)
    bound = R.logprob_bound(logits.reshape(-1, logits.shape[-1]))
    _close(lp.reshape(-1), want_lp, bound, 'log p')
    _close(h.reshape(-1), want_h, bound * (1 + want_h.nan_to_num()), 'entropy')
    _close(tops.reshape(want_tops.shape), want_tops, bound[:, None], 'alternatives')
    if ordered:
        assert torch.equal(at.reshape(want_at.shape).cpu().long(), want_at)
    return lp, h, tops, at


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('rows,vocab,top', [(1, 1, 1), (1, 1, 0), (3, 2, 2), (5, 7, 5), (4, 64, 32), (7, 255, 10), (3, 1023, 32), (10, 3900, 10), (33, 3205, 13),
                                            (2, 28444, 5), (600, 1388, 3), (1, 70001, 32), (2, 131072, 10)])
def test_token_logprobs(ops, dtype, rows, vocab, top):
    g = _gen(rows * 1000 + vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(TYPES[dtype]).cuda()
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    _check_logprobs(ops, x, tokens.cuda(), top)
    _check_logprobs(ops, x, tokens.int().cuda(), top)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('start,vocab,pitch', [(1, 777, 801), (3, 5, 11), (5, 1024, 1030), (0, 333, 333), (7, 3, 3001), (2, 4097, 4100)])
def test_token_logprobs_of_rows_that_start_anywhere(ops, dtype, start, vocab, pitch):
    """Columns of a wider matrix: rows start at every alignment, what lies beside them does not count."""
    g = _gen(start + vocab)
    wide = (torch.randn(9, pitch, generator=g) * 2).to(TYPES[dtype])
    wide[:, :start] = math.nan
    wide[:, start + vocab:] = math.nan
    x = wide.cuda()[:, start:start + vocab]
    _check_logprobs(ops, x, torch.randint(0, vocab, (9,), generator=g).cuda(), min(4, vocab))


def test_token_logprobs_keeps_leading_dimensions(ops):
    g = _gen(4)
    x = torch.randn(3, 4, 50, generator=g).cuda()
    t = torch.randint(0, 50, (3, 4), generator=g).cuda()
    out = _check_logprobs(ops, x, t, 2)
    assert [tuple(y.shape) for y in out] == [(3, 4), (3, 4), (3, 4, 2), (3, 4, 2)]
    one = ops.token_logprobs(x[0, 0], t[0, 0], top=2)
    assert [tuple(y.shape) for y in one] == [(), (), (2,), (2,)]
    none = ops.token_logprobs(x[:0], t[:0], top=2)
    assert [tuple(y.shape) for y in none] == [(0, 4), (0, 4), (0, 4, 2), (0, 4, 2)]
    turned = x.transpose(0, 1)                                     # rows of no single stride: taken through a copy
    _check_logprobs(ops, turned, t.T, 2)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('vocab', [40, 3900, 28444])
def test_token_logprobs_masks_and_extremes(ops, dtype, vocab):
    t = TYPES[dtype]
    low = torch.finfo(t).min
    g = _gen(vocab)
    x = (torch.randn(10, vocab, generator=g) * 3).to(t)
    x[0] = -math.inf                                               # nothing admitted
    x[1] = -math.inf
    x[1, vocab // 2] = 1.5                                         # one token admitted
    x[2, ::2] = -math.inf
    x[3] = low                                                     # uniform
    x[4, 1:] = low
    x[5] = 7.0                                                     # uniform: alternatives in token order
    x[6, ::3] = low
    x[7] = 0.0
    x[7, 5::2] = -0.0                                              # -0 and +0 are one value
    x[8, : vocab - 3] = -math.inf                                  # fewer admitted than alternatives
    x[9] = torch.arange(vocab).to(t) / vocab * 8                   # the largest ones together at the end
    tokens = torch.tensor([3, vocab // 2, 1, 2, 0, 9, 1, 5, vocab - 1, vocab - 1])
    _check_logprobs(ops, x.cuda(), tokens.cuda(), 10)
    _check_logprobs(ops, x.cuda(), torch.zeros_like(tokens).cuda(), 32)


@pytest.mark.parametrize('dtype,vocab', [('f32', 2003), ('bf16', 5003), ('f16', 8191)])
def test_token_logprobs_of_many_longer_rows(ops, dtype, vocab):
    """A thousand rows: ordinary ones, a third masked, equal logits throughout, all masked but a few, all masked."""
    g = _gen(vocab)
    x = torch.randn(1030, vocab, generator=g) * 3
    x[200:400].masked_fill_(torch.rand(200, vocab, generator=g) < 1 / 3, -math.inf)
    x[400:410] = 1.5
    x[410:420] = -math.inf
    x[410:415, 7:13] = torch.randn(5, 6, generator=g)
    tokens = torch.randint(-1, vocab, (1030,), generator=g)
    _check_logprobs(ops, x.to(TYPES[dtype]).cuda(), tokens.cuda(), 9)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_token_logprobs_tokens_outside_the_vocabulary(ops, dtype):
    g = _gen(9)
    x = torch.randn(6, 77, generator=g).to(TYPES[dtype]).cuda()
    tokens = torch.tensor([-1, 77, 5, -(1 << 31), (1 << 31) - 1, 76])
    lp = _check_logprobs(ops, x, tokens.int().cuda(), 1)[0]
    assert float(lp[0]) == 0.0 and math.isnan(float(lp[1]))
    _check_logprobs(ops, x, torch.tensor([-(1 << 40), 1 << 40, 3, 0, (1 << 32) + 5, 1]).cuda(), 1)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_token_logprobs_of_rows_with_nan_or_infinity(ops, dtype):
    g = _gen(10)
    x = torch.randn(6, 3000, generator=g).to(TYPES[dtype])
    x[0, 17] = math.nan
    x[1, 2999] = math.inf
    x[2] = math.nan
    x[3] = -math.inf
    x[3, 5] = math.nan
    x[4, 100] = math.nan
    x[4, 101] = math.inf
    lp, h, tops, at = ops.token_logprobs(x.cuda(), torch.zeros(6, dtype=torch.int64).cuda(), top=7)
    assert bool(torch.isnan(lp[:5]).all()) and bool(torch.isnan(h[:5]).all()) and bool(torch.isnan(tops[:5]).all())
    assert bool(torch.isfinite(lp[5])) and bool(torch.isfinite(h[5])) and bool(torch.isfinite(tops[5]).all())
    assert bool(((at >= 0) & (at < 3000)).all())


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('vocab', [28444, 200003])
def test_token_logprobs_alternatives_that_lie_together(ops, dtype, vocab):
    """The likeliest tokens all in few threads' strips (one 16-byte chunk of every 256 and of every 1024), beyond any list of candidates."""
    per = 4 if dtype == 'f32' else 8
    g = _gen(vocab)
    x = torch.randn(2, vocab, generator=g)
    for r, width in enumerate((256, 1024)):
        at = torch.arange(vocab)
        x[r, (at // per) % width == 3] += 20.0
    x = x.to(TYPES[dtype])
    _check_logprobs(ops, x.cuda(), torch.tensor([13, 14]).cuda(), 32)


# ---- attention ---------------------------------------------------------------------------------------------------------
SHAPES = [  # n, tq, tk, heads, kv_heads, d
    (1, 1, 1, 1, 1, 64), (2, 1, 31, 4, 4, 64), (2, 3, 32, 4, 2, 64), (3, 2, 33, 2, 1, 128), (2, 5, 65, 6, 2, 80), (1, 10, 334, 16, 16, 64),
    (2, 16, 100, 4, 4, 32), (2, 17, 129, 2, 2, 128), (1, 33, 257, 4, 1, 64), (2, 40, 190, 8, 2, 128), (1, 130, 300, 2, 1, 96), (3, 61, 77, 3, 3, 48),
    (1, 1, 4001, 8, 1, 128), (1, 4, 2500, 2, 2, 64), (2, 200, 511, 4, 4, 16)]


def _cross_case(seed, n, tq, tk, heads, kv_heads, d, dtype):
    g = _gen(seed)
    t = TYPES[dtype]
    q = torch.randn(n, tq, heads, d, generator=g).to(t)
    kv = torch.randn(n, tk, 2, kv_heads, d, generator=g).to(t)
    return q, kv


def _check_cross(ops, q, k, v, lens=None, pad=None, scale=None, out=None):
    n, tq, heads, d = q.shape
    tk = k.shape[1]
    got = ops.cross_attention(q, k, v, lens=lens, pad=pad, scale=scale, out=out)
    assert got.dtype == q.dtype
    admitted = torch.ones(n, tk, dtype=torch.bool)
    if lens is not None:
        admitted &= torch.arange(tk) < lens.cpu()[:, None]
    if pad is not None:
        admitted &= ~pad.cpu().bool()
    kk, vv = k.cpu().double().transpose(1, 2), v.cpu().double().transpose(1, 2)
    want, weight, size = R.attention(q, kk, vv, admitted[:, None].expand(n, tq, tk), d ** -0.5 if scale is None else scale)
    vmax = float(torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0).abs().max()) if vv.numel() else 0.0
    _close(got, want, R.attention_bound(want, weight, size, d, tk, q.dtype, vmax), 'out')
    return got


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_cross_attention(ops, shape, dtype):
    q, kv = _cross_case(sum(shape), *shape, dtype)
    kv = kv.cuda()
    _check_cross(ops, q.cuda(), kv[:, :, 0], kv[:, :, 1])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tq', [1, 20, 70])
@pytest.mark.parametrize('d', [8, 24, 40, 64, 72, 104, 120, 128])
def test_cross_attention_head_sizes(ops, d, tq, dtype):
    q, kv = _cross_case(d + tq, 2, tq, 75, 2, 1, d, dtype)
    k, v = kv[:, :, 0].contiguous().cuda(), kv[:, :, 1].contiguous().cuda()
    _check_cross(ops, q.cuda(), k, v, scale=0.3)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tq,heads,kv_heads,d', [(1, 4, 4, 64), (10, 4, 2, 64), (40, 4, 1, 128), (150, 2, 2, 64), (9, 2, 2, 40)])
def test_cross_attention_masks(ops, tq, heads, kv_heads, d, dtype):
    """Lengths of zero, one, all, and beyond both ends; flags that leave a sequence empty; NaN and infinities wherever nothing is admitted."""
    n, tk = 8, 130
    q, kv = _cross_case(tq + d, n, tq, tk, heads, kv_heads, d, dtype)
    lens = torch.tensor([0, 1, tk, 64, 33, -5, tk + 1000, 100], dtype=torch.int32)
    pad = torch.rand(n, tk, generator=_gen(3)) < 0.3
    pad[3] = True
    pad[2, 32:64] = True                                          # a whole tile
    pad[7] = False
    admitted = (torch.arange(tk) < lens[:, None]) & ~pad
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(TYPES[dtype]).min):
        x = kv.clone()
        x[~admitted] = bad
        x = x.cuda()
        got = _check_cross(ops, q.cuda(), x[:, :, 0], x[:, :, 1], lens=lens.cuda(), pad=pad.cuda())
        assert float(got[[0, 3, 5]].abs().max()) == 0.0
        as_bytes = ops.cross_attention(q.cuda(), x[:, :, 0], x[:, :, 1], lens=lens.cuda(), pad=(pad.to(torch.uint8) * 200).cuda())
        assert torch.equal(as_bytes, got)
    x = kv.cuda()
    _check_cross(ops, q.cuda(), x[:, :, 0], x[:, :, 1], lens=lens.cuda())
    _check_cross(ops, q.cuda(), x[:, :, 0], x[:, :, 1], pad=pad.cuda())


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tq', [2, 50])
def test_cross_attention_strides(ops, tq, dtype):
    """Head-major queries and states, one set of states for all sequences, flags cut from a wider tensor, an output with gaps; nothing else is
    written."""
    n, tk, heads, d = 3, 90, 4, 64
    g = _gen(tq)
    t = TYPES[dtype]
    q = torch.randn(n, heads, tq, d, generator=g).to(t).cuda().transpose(1, 2)
    k = torch.randn(1, heads, tk, d, generator=g).to(t).cuda().transpose(1, 2).expand(n, -1, -1, -1)
    v = torch.randn(n, heads, tk, d + 8, generator=g).to(t).cuda().transpose(1, 2)[..., 8:]
    pad = (torch.rand(n, tk + 7, generator=g) < 0.2).cuda()[:, 3:tk + 3]
    wide = torch.full((n, tq + 2, heads, 2 * d), 5.0, dtype=t, device='cuda')
    out = wide[:, 1:tq + 1, :, d:]
    got = _check_cross(ops, q, k, v, pad=pad, out=out)
    assert got.data_ptr() == out.data_ptr()
    wide[:, 1:tq + 1, :, d:] = 5.0
    assert bool((wide == 5.0).all())


@pytest.mark.parametrize('n,tq,kv_heads', [(2, 3, 4), (20, 1, 1), (64, 2, 2), (65, 1, 2), (7, 45, 8), (64, 60, 1)])
def test_cross_attention_of_many_lengths(ops, n, tq, kv_heads):
    """Equal, zero and negative lengths and some beyond the end among those of up to 65 sequences, taken in whatever order."""
    q, kv = _cross_case(n + tq, n, tq, 1100, kv_heads, kv_heads, 64, 'bf16')
    kv = kv.cuda()
    lens = torch.randint(-100, 1300, (n,), generator=_gen(n), dtype=torch.int32)
    lens[n // 2:] = lens[:n - n // 2].flip(0)
    _check_cross(ops, q.cuda(), kv[:, :, 0], kv[:, :, 1], lens=lens.cuda())


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('n,tq,tk,heads,kv_heads', [(64, 200, 130, 8, 8), (4, 520, 65, 256, 128), (64, 129, 64, 8, 8), (3, 1030, 90, 64, 64)])
def test_cross_attention_of_many_rows_and_sequences(ops, n, tq, tk, heads, kv_heads, dtype):
    q, kv = _cross_case(n + tq, n, tq, tk, heads, kv_heads, 64, dtype)
    lens = torch.randint(0, tk + 1, (n,), generator=_gen(n), dtype=torch.int32)
    pad = torch.rand(n, tk, generator=_gen(tq)) < 0.2
    kv = kv.cuda()
    _check_cross(ops, q.cuda(), kv[:, :, 0], kv[:, :, 1], lens=lens.cuda(), pad=pad.cuda())


@pytest.mark.parametrize('causal', [False, True])
def test_kv8_attention_of_many_rows_and_sequences(ops, causal):
    g = _gen(9)
    cache = _loud_cache(ops, g, 64, 8, 256, 64)
    q = torch.randn(64, 130, 16, 64, generator=g).bfloat16().cuda()
    lens = torch.randint(100, 257, (64,), generator=g, dtype=torch.int32)
    _check_kv8(ops, q, cache, lens.cuda(), causal=causal)


def test_cross_attention_without_states_or_queries(ops):
    q = torch.randn(2, 3, 4, 64, device='cuda')
    none = torch.empty(2, 0, 4, 64, device='cuda')
    out = torch.full_like(q, 7.0)
    assert float(ops.cross_attention(q, none, none, out=out).abs().max()) == 0.0
    assert ops.cross_attention(q[:, :0], q, q).shape == (2, 0, 4, 64)
    assert ops.cross_attention(q[:0], q[:0], q[:0]).shape == (0, 3, 4, 64)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_cross_attention_of_large_scores(ops, dtype):
    """Scores of hundreds: one state takes all; a negative scale and a scale of zero."""
    q, kv = _cross_case(5, 2, 6, 200, 4, 2, 64, dtype)
    q, kv = (q * 8).cuda(), (kv * 8).cuda()
    for scale in (1.0, -1.0, 0.0):
        _check_cross(ops, q, kv[:, :, 0], kv[:, :, 1], scale=scale)


def test_ops_refuse(ops):
    q = torch.randn(2, 3, 4, 64, device='cuda')
    k = torch.randn(2, 9, 2, 64, device='cuda')
    from asr_amd._lib import AsrError
    ok = torch.tensor([1, 2], dtype=torch.int32, device='cuda')
    bad = [lambda: ops.cross_attention(q.double(), k.double(), k.double()), lambda: ops.cross_attention(q, k.half(), k.half()),
           lambda: ops.cross_attention(q, k, k[:, :8]), lambda: ops.cross_attention(q, k[:1], k[:1]), lambda: ops.cross_attention(q, k, k.cpu()),
           lambda: ops.cross_attention(q, k, k, lens=ok.long()), lambda: ops.cross_attention(q, k, k, lens=ok[:1]),
           lambda: ops.cross_attention(q, k, k, lens=ok.cpu()), lambda: ops.cross_attention(q, k, k, pad=torch.zeros(2, 8, device='cuda') > 0),
           lambda: ops.cross_attention(q, k, k, pad=torch.zeros(2, 9, device='cuda')), lambda: ops.cross_attention(q, k, k, out=q.half()),
           lambda: ops.cross_attention(q, k, k, out=q[:1, :1, :1].expand_as(q)), lambda: ops.cross_attention(q.requires_grad_(), k, k),
           lambda: ops.cross_attention(q.detach().transpose(1, 3).contiguous().transpose(1, 3), k, k),
           lambda: ops.token_logprobs(torch.zeros(2, 5, device='cuda'), ok[:1]), lambda: ops.token_logprobs(torch.zeros(2, 5, device='cuda'), ok.float()),
           lambda: ops.token_logprobs(torch.zeros(2, 5, device='cuda'), ok, top=6), lambda: ops.token_logprobs(torch.zeros(2, 5, device='cuda').double(), ok),
           lambda: ops.token_logprobs(torch.zeros(5, 2, device='cuda').T, ok), lambda: ops.token_logprobs(torch.zeros(2, 0, device='cuda'), ok)]
    k8, v8, ks, vs = ops.kv8_cache(2, 2, 128, 64)
    bad += [lambda: ops.kv8_attention(q.detach(), k8, v8[:, :, :64], ks, vs, ok), lambda: ops.kv8_attention(q.detach(), k8, v8, ks[:, :, :1], vs, ok),
            lambda: ops.kv8_attention(q.detach(), k8.view(torch.uint8), v8, ks, vs, ok), lambda: ops.kv8_attention(q.detach()[:1], k8, v8, ks, vs, ok),
            lambda: ops.kv8_attention(q.detach(), k8, v8, ks, vs, ok.long()), lambda: ops.kv8_append(k, k.half(), k8, v8, ks, vs, ok),
            lambda: ops.kv8_append(k, k, k8, v8, ks.double(), vs, ok), lambda: ops.kv8_append(k[:, :, :1], k, k8, v8, ks, vs, ok),
            lambda: ops.kv8_append(k, k, k8[:1].expand(2, -1, -1, -1), v8[:1].expand(2, -1, -1, -1), ks, vs, ok),
            lambda: ops.kv8_append(k, k, k8, v8, ks, vs, ok, counts=ok[:1])]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print('call %d was not refused' % i)
    refused = [lambda: ops.cross_attention(q.detach()[:, :, :3], k, k), lambda: ops.cross_attention(q.detach()[..., :60], k[..., :60], k[..., :60]),
               lambda: ops.cross_attention(torch.zeros(1, 1, 1, 65, device='cuda')[..., 1:], k[:1, :, :1], k[:1, :, :1]),
               lambda: ops.cross_attention(q.detach(), k, k, scale=math.nan)]
    for call in refused:
        with pytest.raises(AsrError):
            call()


# ---- the 8-bit cache ---------------------------------------------------------------------------------------------------
def _random_cache(ops, g, n, kv_heads, capacity, d):
    """Codes of every kind but NaN under scales of several sizes."""
    k8, v8, ks, vs = ops.kv8_cache(n, kv_heads, capacity, d)
    for c in (k8, v8):
        code = torch.randint(0, 256, c.shape, generator=g, dtype=torch.uint8)
        code[(code & 127) == 127] = 0x55
        c.view(torch.uint8).copy_(code)
    for s in (ks, vs):
        s.copy_(2.0 ** torch.randint(-10, -6, s.shape, generator=g).float())
    return k8, v8, ks, vs


def _check_append(ops, k, v, cache, lens, counts=None):
    k8, v8, ks, vs = cache
    before = [R.values_of(k8), R.values_of(v8), ks.cpu().double(), vs.cpu().double()]
    ops.kv8_append(k, v, k8, v8, ks, vs, lens, counts=counts)
    for x, code, scale, was_code, was_scale, name in ((k, k8, ks, before[0], before[2], 'k'), (v, v8, vs, before[1], before[3], 'v')):
        want, want_scale = R.append(x, was_code, was_scale, lens.cpu(), None if counts is None else counts.cpu())
        assert torch.equal(scale.cpu().double(), want_scale), name + ' scale'
        got = R.values_of(code)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), name + ' NaN'
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)), name + ' codes'


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('n,new,kv_heads,capacity,d', [(1, 1, 1, 64, 64), (3, 1, 4, 192, 64), (6, 1, 2, 128, 128), (2, 64, 2, 128, 32), (3, 65, 1, 256, 80),
                                                       (4, 200, 2, 256, 64), (2, 256, 3, 256, 16), (5, 7, 2, 128, 112), (2, 300, 1, 256, 48)])
def test_kv8_append(ops, dtype, n, new, kv_heads, capacity, d):
    g = _gen(n * new + d)
    cache = _random_cache(ops, g, n, kv_heads, capacity, d)
    k = (torch.randn(n, new, kv_heads, d, generator=g) * 3).to(TYPES[dtype])
    v = torch.randn(n, new, kv_heads, d, generator=g).to(TYPES[dtype]) * 100                  # scales grow
    lens = torch.randint(0, capacity + 1, (n,), generator=g, dtype=torch.int32)
    lens[0] = 0
    _check_append(ops, k.cuda(), v.cuda(), cache, lens.cuda())
    counts = torch.randint(0, new + 1, (n,), generator=g, dtype=torch.int32)
    _check_append(ops, v.cuda(), k.cuda(), cache, lens.cuda(), counts.cuda())


def test_kv8_append_lengths_and_counts_outside_their_range(ops):
    g = _gen(1)
    lens = torch.tensor([-1, -(1 << 31), 128, (1 << 31) - 1, 120, 0, 60, 64], dtype=torch.int32).cuda()
    counts = torch.tensor([9, 9, 9, 9, 1000, -3, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32).cuda()
    cache = _random_cache(ops, g, 8, 2, 128, 64)
    k, v = torch.randn(8, 20, 2, 64, generator=g).cuda(), torch.randn(8, 20, 2, 64, generator=g).cuda()
    _check_append(ops, k, v, cache, lens, counts)
    _check_append(ops, k, v, cache, lens)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_kv8_append_token_by_token_keeps_every_scale_minimal(ops, dtype):
    g = _gen(2)
    cache = ops.kv8_cache(2, 1, 128, 32)
    for i in range(70):
        loud = 2.0 ** float(torch.randint(-6, 7, (1,), generator=g))
        k = (torch.randn(2, 1, 1, 32, generator=g) * loud).to(TYPES[dtype]).cuda()
        _check_append(ops, k, -k, cache, torch.tensor([i, i + 3], dtype=torch.int32).cuda())


def test_kv8_append_extremes(ops):
    """Zeros, subnormals, the largest float32, infinities and NaN; halfway values; NaN and infinities count for no scale."""
    n, d = 8, 16
    k = torch.zeros(n, 3, 1, d)
    k[1] = 2.0 ** -140
    k[2, 0, 0, 0] = 3.0e38
    k[2, 1] = 1.0
    k[3, 0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 5.0])
    k[4] = math.inf
    k[5] = math.nan
    k[6, 0, 0] = torch.tensor([448.0, 232.0, 248.0, -232.0, 17.0, 19.0, 0.0009765625, 0.0029296875, 0.00146484375, -0.0, 464.0, 1.0, 1.0625, 1.1875, 2.0, 3.0])
    k[7] = torch.linspace(-448, 448, 3 * d).reshape(3, 1, d)
    for lens in (0, 5):
        cache = ops.kv8_cache(n, 1, 64, d)
        cache[2].fill_(2.0 ** -9)
        cache[3].fill_(2.0 ** -9)
        cache[0].view(torch.uint8).fill_(0x7e)
        _check_append(ops, k.cuda(), -k.cuda(), cache, torch.full((n,), lens, dtype=torch.int32).cuda())


def test_kv8_append_of_more_new_tokens_than_fit(ops):
    """2^25 new tokens of 128 (their product passes 32 bits), the same memory for each, into a cache of 128: what fits is written."""
    g = _gen(77)
    cache = _random_cache(ops, g, 1, 1, 128, 128)
    row = torch.randn(1, 1, 1, 128, generator=g).to(torch.bfloat16).cuda()
    lens = torch.tensor([3], dtype=torch.int32).cuda()
    other = [c.clone() for c in cache]
    many = row.expand(1, 1 << 25, 1, 128)
    ops.kv8_append(many, many, *cache, lens)
    few = row.expand(1, 125, 1, 128)
    ops.kv8_append(few, few, *other, lens)
    for a, b in zip(cache, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_kv8_append_strides_and_views(ops):
    """Keys and values as halves of one projection, caches as part of larger ones: nothing beside them is written."""
    g = _gen(3)
    kv = torch.randn(2, 40, 2, 3, 64, generator=g).cuda()
    big = _random_cache(ops, g, 4, 3, 128, 64)
    whole = [x.clone() for x in big]
    _check_append(ops, kv[:, :, 0], kv[:, :, 1], [x[1:3] for x in big], torch.tensor([30, 100], dtype=torch.int32).cuda())
    for x, y in zip(big, whole):
        assert torch.equal(x[[0, 3]].view(torch.uint8), y[[0, 3]].view(torch.uint8))


def _check_kv8(ops, q, cache, lens, causal=False, scale=None, out=None):
    n, tq, heads, d = q.shape
    k8, v8, ks, vs = cache
    got = ops.kv8_attention(q, k8, v8, ks, vs, lens, causal=causal, scale=scale, out=out)
    assert got.dtype == q.dtype
    tk = k8.shape[2]
    k = R.values_of(k8) * ks.cpu().double().repeat_interleave(64, -1)[..., None]
    v = R.values_of(v8) * vs.cpu().double().repeat_interleave(64, -1)[..., None]
    last = lens.cpu().long().clamp(0, tk)[:, None].expand(n, tq)
    if causal:
        last = last - tq + 1 + torch.arange(tq)
    admitted = torch.arange(tk) < last[..., None]
    want, weight, size = R.attention(q, k, v, admitted, d ** -0.5 if scale is None else scale)
    _close(got, want, R.attention_bound(want, weight, size, d, tk, q.dtype, float(torch.nan_to_num(v).abs().max()) if v.numel() else 0.0), 'out')
    return got


def _loud_cache(ops, g, n, kv_heads, capacity, d):
    """A cache of normal values whose blocks differ in loudness."""
    k8, v8, ks, vs = ops.kv8_cache(n, kv_heads, capacity, d)
    for c, s in ((k8, ks), (v8, vs)):
        x = torch.randn(c.shape, generator=g, dtype=torch.float64)
        e = torch.randint(-3, 2, s.shape, generator=g)
        c.copy_((x * 100).float().clamp(-448, 448).to(torch.float8_e4m3fn))
        s.copy_(2.0 ** (e.float() - 7))
    return k8, v8, ks, vs


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('n,tq,heads,kv_heads,capacity,d', [
    (1, 1, 1, 1, 64, 64), (3, 1, 4, 4, 128, 64), (2, 1, 8, 2, 192, 128), (2, 10, 4, 4, 320, 64), (2, 20, 2, 1, 128, 80), (1, 1, 8, 1, 4096, 128),
    (2, 40, 4, 2, 192, 128), (1, 150, 2, 1, 256, 64), (2, 64, 3, 3, 64, 16), (2, 33, 4, 1, 128, 112), (1, 260, 4, 2, 512, 128)])
def test_kv8_attention(ops, n, tq, heads, kv_heads, capacity, d, causal, dtype):
    g = _gen(n + tq + capacity + d)
    cache = _loud_cache(ops, g, n, kv_heads, capacity, d)
    q = torch.randn(n, tq, heads, d, generator=g).to(TYPES[dtype]).cuda()
    lens = torch.randint(min(tq, capacity), capacity + 1, (n,), generator=g, dtype=torch.int32)
    lens[0] = capacity
    _check_kv8(ops, q, cache, lens.cuda(), causal=causal)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('tq,heads,kv_heads,d', [(1, 4, 4, 64), (8, 4, 2, 128), (40, 4, 1, 64), (90, 2, 2, 128)])
def test_kv8_attention_lengths(ops, tq, heads, kv_heads, d, causal, dtype):
    """Lengths of zero, one, inside a tile and a block, all, beyond both ends; causal calls with fewer tokens than queries; behind the length codes
    of NaN under scales of infinity."""
    g = _gen(tq + d)
    n, capacity = 9, 192
    cache = _loud_cache(ops, g, n, kv_heads, capacity, d)
    lens = torch.tensor([0, 1, capacity, 64, 33, -5, capacity + 1000, 100, 65], dtype=torch.int32)
    for b in range(n):
        length = max(0, min(capacity, int(lens[b])))
        for c in cache[:2]:
            c.view(torch.uint8)[b, :, length:] = 0x7f
        for s in cache[2:]:
            s[b, :, (length + 63) // 64:] = math.inf
    q = torch.randn(n, tq, heads, d, generator=g).to(TYPES[dtype]).cuda()
    _check_kv8(ops, q, cache, lens.cuda(), causal=causal, scale=0.2)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tq,heads,kv_heads,capacity,d', [(1, 2, 2, 128, 64), (9, 4, 2, 192, 128), (24, 2, 1, 128, 80), (8, 2, 2, 2048, 64), (90, 2, 2, 192, 128),
                                                          (150, 4, 2, 320, 64), (70, 2, 1, 128, 48), (200, 1, 1, 2048, 128),
                                                          (140, 172, 172, 192, 64)])
def test_kv8_attention_nan_in_later_tokens(ops, tq, heads, kv_heads, capacity, d, dtype):
    """A causal query is not touched by NaN in tokens behind its own; one that sees a NaN value has NaN in that value's column alone, one that sees a
    NaN key everywhere."""
    g = _gen(tq + capacity)
    n = 3
    cache = _loud_cache(ops, g, n, kv_heads, capacity, d)
    lens = torch.tensor([capacity, capacity - 37, max(tq, 67)], dtype=torch.int32)
    for b in range(n):
        last = int(lens[b]) - 1
        for h in range(kv_heads):
            for back, column in ((1, (3 + h) % d), (tq // 3, d - 1), (tq // 2, 17)):
                if last - back >= 0:
                    cache[1].view(torch.uint8)[b, h, last - back, column] = 0x7f if h % 2 else 0xff
            cache[0].view(torch.uint8)[b, h, last, 5] = 0x7f
    q = torch.randn(n, tq, heads, d, generator=g).to(TYPES[dtype]).cuda()
    got = ops.kv8_attention(q, *cache, lens.cuda(), causal=True).cpu().double()
    k, v = (R.values_of(c) * s.cpu().double().repeat_interleave(64, -1)[..., None] for c, s in (cache[::2], cache[1::2]))
    admitted = torch.arange(capacity) < (lens.long()[:, None] - tq + 1 + torch.arange(tq))[..., None]
    want, weight, size = R.attention(q, k, v, admitted, d ** -0.5)
    bound = R.attention_bound(want, weight, size, d, capacity, q.dtype, float(torch.nan_to_num(v).abs().max()))
    group = heads // kv_heads
    sees_value = torch.einsum('nik,nhkd->nihd', admitted.double(), v.isnan().double()).repeat_interleave(group, 2) > 0
    sees_key = torch.einsum('nik,nhk->nih', admitted.double(), k.isnan().any(-1).double()).repeat_interleave(group, 2) > 0
    lost = sees_value | sees_key[..., None]
    assert bool(lost.any()) and (tq == 1 or not bool(lost.all()))
    assert torch.equal(got.isnan(), lost)
    _close(got.masked_fill(lost, 0), want.masked_fill(lost, 0), bound, 'out')


def test_kv8_attention_with_scales_far_apart(ops):
    """Blocks whose value scales differ by 2^60 and keys of tiny and large scales."""
    g = _gen(8)
    for dtype in ('f32', 'bf16', 'f16'):
        cache = _loud_cache(ops, g, 2, 2, 256, 64)
        cache[3][:, :, 1] = 2.0 ** -60
        cache[2][:, :, 2] = 2.0 ** -40
        q = torch.randn(2, 3, 4, 64, generator=g).to(TYPES[dtype]).cuda()
        _check_kv8(ops, q, cache, torch.tensor([256, 130], dtype=torch.int32).cuda())


def test_kv8_attention_strides(ops):
    g = _gen(6)
    big = _loud_cache(ops, g, 4, 2, 128, 64)
    cache = [x[1:3] for x in big]
    q = torch.randn(2, 4, 5, 64, generator=g).cuda().transpose(1, 2)
    wide = torch.full((2, 5, 4, 128), 5.0, device='cuda')
    _check_kv8(ops, q, cache, torch.tensor([128, 77], dtype=torch.int32).cuda(), out=wide[..., 64:])
    assert bool((wide[..., :64] == 5.0).all())
    assert ops.kv8_attention(q[:, :0], *cache, torch.tensor([1, 1], dtype=torch.int32).cuda()).shape == (2, 0, 4, 64)


# ---- streams, graphs, together -------------------------------------------------------------------------------------------
def _step(ops, s):
    """Keys and values of new tokens into the cache, attention over it and over encoder states, a projection to logits, their log probabilities."""
    ops.kv8_append(s['k'], s['v'], *s['cache'], s['lens'])
    a = ops.kv8_attention(s['q'], *s['cache'], s['after'], causal=True)
    c = ops.cross_attention(a, s['ek'], s['ev'], lens=s['elens'], pad=s['epad'])
    logits = torch.matmul(c.reshape(-1, c.shape[2] * c.shape[3]).float(), s['w'])
    return (a, c) + tuple(ops.token_logprobs(logits, s['tokens'], top=4))


def _together(ops, seed, dtype=torch.bfloat16, n=3, tq=2, heads=4, kv_heads=2, d=64, capacity=128, tk=70, vocab=333):
    g = _gen(seed)
    r = lambda *shape: torch.randn(*shape, generator=g).to(dtype).cuda()  # noqa: E731
    lens = torch.tensor([0, 63, 100][:n], dtype=torch.int32)
    return {'cache': _loud_cache(ops, g, n, kv_heads, capacity, d), 'k': r(n, tq, kv_heads, d), 'v': r(n, tq, kv_heads, d), 'q': r(n, tq, heads, d),
            'lens': lens.cuda(), 'after': (lens + tq).cuda(), 'ek': r(n, tk, kv_heads, d), 'ev': r(n, tk, kv_heads, d),
            'elens': torch.tensor([70, 1, 40], dtype=torch.int32).cuda(), 'epad': (torch.rand(n, tk, generator=g) < 0.2).cuda(),
            'w': torch.randn(heads * d, vocab, generator=g).cuda() * 0.05, 'tokens': torch.randint(0, vocab, (n * tq,), generator=g).cuda()}


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_the_operators_together(ops, dtype):
    """A step of a scored decoder, each operator against its reference on what the one before it left."""
    s = _together(ops, 11, TYPES[dtype])
    _check_append(ops, s['k'], s['v'], s['cache'], s['lens'])
    a = _check_kv8(ops, s['q'], s['cache'], s['after'], causal=True)
    c = _check_cross(ops, a, s['ek'], s['ev'], lens=s['elens'], pad=s['epad'])
    logits = torch.matmul(c.reshape(6, -1).float(), s['w'])
    _check_logprobs(ops, logits, s['tokens'], 4)


def test_on_another_stream(ops):
    want = _step(ops, _together(ops, 12))
    side = torch.cuda.Stream()
    s = _together(ops, 12)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize('tk', [70, 6000])
def test_captured_and_replayed(ops, tk):
    """Two graphs of the same step on different inputs (long keys: with a workspace each), replayed in turn with eager work in between."""
    states = [_together(ops, 20 + i, tk=tk) for i in range(2)]
    for s in states:
        s['elens'] = torch.tensor([tk, 1, tk - 7], dtype=torch.int32).cuda()
    start = [[x.clone() for x in s['cache']] for s in states]
    want = []
    for s, c in zip(states, start):
        want.append([x.clone() for x in _step(ops, s)])
        for x, y in zip(s['cache'], c):
            x.copy_(y)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(ops, s))
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1) if turn % 2 else (1, 0):
            for x, y in zip(states[i]['cache'], start[i]):
                x.copy_(y)
            graphs[i].replay()
            eager = _step(ops, _together(ops, 30 + turn, tk=tk))
            if turn == 2:
                torch.cuda.synchronize()
            for x, y in zip(outs[i], want[i]):
                assert torch.equal(x, y)
            assert bool(torch.isfinite(eager[2]).all())


def test_calls_on_two_streams_at_once(ops):
    """Long keys (a workspace each) and many rows, queued on two streams in turn: each gives what it gives alone."""
    states = [_together(ops, 50 + i, tk=7000) for i in range(2)]
    for s in states:
        s['elens'] = torch.tensor([7000, 6999, 3000], dtype=torch.int32).cuda()
    many = [torch.randn(2, 300, 8, 64, generator=_gen(60 + i)).bfloat16().cuda() for i in range(2)]
    long = [torch.randn(2, 1500, 2, 8, 64, generator=_gen(70 + i)).bfloat16().cuda() for i in range(2)]

    def run(i):
        ctx = ops.cross_attention(many[i], long[i][:, :, 0], long[i][:, :, 1])
        return [ctx] + list(_step(ops, dict(states[i], cache=[c.clone() for c in states[i]['cache']])))
    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append((i, run(i)))
    torch.cuda.synchronize()
    for i, out in got:
        for x, y in zip(out, want[i]):
            assert torch.equal(x, y)


def test_lengths_and_counts_at_the_ends_of_int32(ops):
    g = _gen(80)
    low, high = -2 ** 31, 2 ** 31 - 1
    lens = torch.tensor([low, high, 5, 0], dtype=torch.int32)
    q, kv = _cross_case(80, 4, 3, 130, 2, 2, 64, 'bf16')
    kv = kv.cuda()
    _check_cross(ops, q.cuda(), kv[:, :, 0], kv[:, :, 1], lens=lens.cuda())
    cache = _loud_cache(ops, g, 4, 2, 128, 64)
    for causal in (False, True):
        _check_kv8(ops, q.cuda(), cache, lens.cuda(), causal=causal)
    k, v = (torch.randn(4, 3, 2, 64, generator=g).cuda() for _ in range(2))
    cache = _random_cache(ops, g, 4, 2, 128, 64)
    _check_append(ops, k, v, cache, torch.tensor([low, high, 5, 0], dtype=torch.int32).cuda(), torch.tensor([3, 3, high, low], dtype=torch.int32).cuda())


def test_more_rows_and_sequences_than_one_grid_dimension(ops):
    rows = (1 << 20) + 9
    logits = torch.randn(rows, 5, generator=_gen(90)).half().cuda()
    tokens = torch.randint(-1, 5, (rows,), generator=_gen(91)).cuda()
    logp, entropy, top_logp, top_tokens = ops.token_logprobs(logits, tokens, top=2)
    some = torch.cat([torch.arange(50), torch.arange(rows - 50, rows)]).cuda()
    # (against 64 bits, not against a call on these rows alone: where a row starts within 16 bytes groups its sums)
    want_lp, want_h, want_tops, want_at = R.token_logprobs(logits[some], tokens[some].cpu(), 2)
    bound = R.logprob_bound(logits[some])
    _close(logp[some], want_lp, bound, 'log p')
    _close(entropy[some], want_h, bound * (1 + want_h), 'entropy')
    _close(top_logp[some], want_tops, bound[:, None], 'alternatives')
    assert torch.equal(top_tokens[some].cpu().long(), want_at)
    n = 70001
    q, kv = torch.randn(n, 1, 1, 8, generator=_gen(92)).cuda(), torch.randn(n, 3, 2, 1, 8, generator=_gen(93)).cuda()
    lens = torch.randint(0, 4, (n,), generator=_gen(94), dtype=torch.int32).cuda()
    out = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1], lens=lens)
    some = torch.cat([torch.arange(50), torch.arange(n - 50, n)]).cuda()
    part = kv[some]
    assert torch.equal(_check_cross(ops, q[some], part[:, :, 0], part[:, :, 1], lens=lens[some]), out[some])


def test_repeated_calls_give_the_same_bits(ops):
    s = _together(ops, 40, tk=5000)
    s['elens'] = torch.tensor([5000, 4999, 3000], dtype=torch.int32).cuda()
    first = _step(ops, s)
    for _ in range(3):
        for x, y in zip(_step(ops, s), first):
            assert torch.equal(x, y)


def test_offsets_beyond_32_bits(ops):
    """States whose rows lie gigabytes apart: one projection of 2.2 GB a sequence, read at its far end."""
    n, tk, d = 2, 9, 64
    pitch = (1 << 28) // 8 * 8
    flat = torch.empty(2 * tk * pitch // 2, dtype=torch.bfloat16, device='cuda')
    k = flat.as_strided((n, tk, 1, d), (tk * pitch // 2, pitch // 2, d, 1))
    v = flat.as_strided((n, tk, 1, d), (tk * pitch // 2, pitch // 2, d, 1), 512)
    g = _gen(7)
    k.copy_(torch.randn(n, tk, 1, d, generator=g))
    v.copy_(torch.randn(n, tk, 1, d, generator=g))
    q = torch.randn(n, 3, 2, d, generator=g).to(torch.bfloat16).cuda()
    _check_cross(ops, q, k, v)


def test_a_long_cache(ops):
    """A cache of over 4 GiB: appending to and reading its last head."""
    n, kv_heads, capacity, d = 1, 5, 64 * 114688, 128
    k8, v8, ks, vs = ops.kv8_cache(n, kv_heads, capacity, d)
    assert k8.numel() > 1 << 32
    g = _gen(5)
    k = torch.randn(n, 70, kv_heads, d, generator=g).cuda()
    lens = torch.tensor([capacity - 100], dtype=torch.int32).cuda()
    ops.kv8_append(k, -k, k8, v8, ks, vs, lens)
    tail = [x[:, :, -128:].clone() if x.dim() == 4 else x[:, :, -2:].clone() for x in (k8, v8, ks, vs)]
    fresh = ops.kv8_cache(n, kv_heads, 128, d)
    ops.kv8_append(k, -k, *fresh, torch.tensor([28], dtype=torch.int32).cuda())
    for x, y in zip(tail, fresh):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # zeros everywhere but the last tokens: their share among capacity - 30 equal scores of zero
    q = torch.zeros(n, 1, kv_heads, d).cuda()
    got = ops.kv8_attention(q, k8, v8, ks, vs, torch.tensor([capacity - 30], dtype=torch.int32).cuda()).double().cpu()
    values = R.values_of(tail[1])[0] * tail[3].cpu().double()[0].repeat_interleave(64, -1)[..., None] / (capacity - 30)
    # every probability is the same; 64 splits of four waves sum them in steps of 32 keys
    bound = 2 * ((capacity / (64 * 4 * 32) + 64) * R.U + 2.0 ** -22) * values.abs().sum(1) + R.U * values.sum(1).abs()
    assert bool(((got[0, 0] - values.sum(1)).abs() <= bound).all())
