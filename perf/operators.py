"""The cases that the framework's scoring and 8-bit cache operators (`asr_amd.ops`) are timed on.

A case names an operator and its sizes; `prepare` makes its inputs on the GPU, `run` makes one pass - with `own` the calls
a user makes of `asr_amd.ops`, without it the same operator in elementary torch operations in 32 bits - and `exact` gives
the outputs in 64 bits, written from the definitions alone.

Operators
  logprobs   log p(token), the entropy and the most likely alternatives of every row of logits [rows, vocab].
  cross      attention of tq query rows per sequence over tk encoder states, `lens` of them valid; H query heads share
             Hkv key heads; optionally single states flagged as padding.
  append     new keys and values written behind what a cache in 8 bits holds: e4m3 codes with one power-of-two scale for
             each block of 64 tokens and head, the smallest scale that keeps the block's largest magnitude within 448.
  attend     attention of tq query rows per sequence over such a cache, optionally causal in the newest tq tokens.
"""
import torch

own = False

BLOCK = 64                                     # tokens that share a scale in the 8-bit cache
MIN_EXP = -100                                 # smallest exponent of a scale
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}


# ---- cases -----------------------------------------------------------------------------------------------------------
def _logprobs(rows, vocab, top, dtype, masked):
    return {'op': 'logprobs', 'rows': rows, 'vocab': vocab, 'top': top, 'dtype': dtype, 'masked': masked}


def _cross(n, tq, tk, heads, kv_heads, d, dtype, pad):
    return {'op': 'cross', 'n': n, 'tq': tq, 'tk': tk, 'heads': heads, 'kv_heads': kv_heads, 'd': d, 'dtype': dtype, 'pad': pad}


def _append(n, held, new, capacity, kv_heads, d, dtype):
    return {'op': 'append', 'n': n, 'held': held, 'new': new, 'capacity': capacity, 'kv_heads': kv_heads, 'd': d, 'dtype': dtype}


def _attend(n, tq, capacity, heads, kv_heads, d, dtype, causal):
    return {'op': 'attend', 'n': n, 'tq': tq, 'capacity': capacity, 'heads': heads, 'kv_heads': kv_heads, 'd': d, 'dtype': dtype,
            'causal': causal}


def listed():
    return [
        # confidence of one utterance's ten beams at one decode step, the char vocabulary: latency
        dict(_logprobs(10, 3900, 10, 'f32', False), name='logprobs_one_step'),
        # 64 hypotheses of 64 tokens rescored with the word vocabulary, part of it masked out
        dict(_logprobs(4096, 28444, 5, 'bf16', True), name='logprobs_rescoring'),
        # one utterance of under two seconds, one token: latency
        dict(_cross(1, 1, 47, 16, 16, 64, 'bf16', False), name='cross_one_token'),
        # a decode step of the headline batch: 64 utterances of up to 334 stacked frames, ten beams each
        dict(_cross(64, 10, 334, 16, 16, 64, 'bf16', False), name='cross_beams'),
        # 50 hypotheses of 61 tokens scored against 30 s utterances in the reference's float32, padding by flags
        dict(_cross(50, 61, 1000, 16, 16, 64, 'f32', True), name='cross_scoring_f32'),
        # long transcripts against long recordings, grouped heads: bound by the matrix pipe
        dict(_cross(8, 768, 4001, 32, 8, 128, 'bf16', False), name='cross_long'),
        # one decoded token of each of 64 sequences joins its history: latency
        dict(_append(64, 200, 1, 256, 16, 64, 'f32'), name='append_one_token'),
        # the encoder's keys and values of 64 utterances of up to 30 s packed once
        dict(_append(64, 0, 1000, 1024, 16, 64, 'bf16'), name='append_encoder_states'),
        # a decode step of 16 sequences over histories of up to 200 tokens in the reference's float32: latency
        dict(_attend(16, 1, 256, 16, 16, 64, 'f32', False), name='attend_one_token'),
        # ten beams of 64 utterances over the packed encoder states
        dict(_attend(64, 10, 1024, 16, 16, 64, 'bf16', False), name='attend_beams'),
        # a prompt of 512 tokens read in behind what the cache holds, grouped heads, causal
        dict(_attend(4, 512, 4096, 32, 8, 128, 'bf16', True), name='attend_chunk'),
        # one token each of 8 sequences over histories of up to 32768 tokens: bound by the cache's bytes
        dict(_attend(8, 1, 32768, 32, 8, 128, 'bf16', False), name='attend_long'),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    def cost(c):
        # float32 products run at a sixteenth of the 16-bit matrix rate; narrow heads have more scores for the same products
        w = work(c)
        if 'd' not in c:
            return (w['bytes'],)
        return w['bytes'], w['flops'] * (16 if c['dtype'] == 'f32' else 1), w['flops'] / c['d']

    op = rng.choice(('logprobs', 'cross', 'append', 'attend'))
    while True:
        if op == 'logprobs':
            c = _logprobs(_spread(rng, 1, 8192), _spread(rng, 100, 70000), rng.choice((0, 1, 3, 5, 10, 13, 32)),
                          rng.choice(('f32', 'bf16', 'f16')), rng.random() < 0.3)
        else:
            heads, kv_heads = rng.choice(((16, 16), (16, 4), (8, 8), (8, 1), (32, 8), (12, 4), (5, 5)))
            d, dtype = rng.choice((64, 64, 128, 128, 80, 32)), rng.choice(('f32', 'bf16', 'bf16', 'f16'))
            if op == 'cross':
                c = _cross(_spread(rng, 1, 128), _spread(rng, 1, 1024), _spread(rng, 1, 5000), heads, kv_heads, d, dtype, rng.random() < 0.4)
            elif op == 'append':
                capacity = BLOCK * _spread(rng, 1, 64)
                new = _spread(rng, 1, capacity)
                c = _append(_spread(rng, 1, 128), rng.choice((0, capacity - new)), new, capacity, kv_heads, d, dtype)
            else:
                capacity = BLOCK * _spread(rng, 1, 512)
                c = _attend(_spread(rng, 1, 128), _spread(rng, 1, min(512, capacity)), capacity, heads, kv_heads, d, dtype, rng.random() < 0.5)
        most = zip(*(cost(x) for x in listed() if x['op'] == op))
        if all(x <= max(m) for x, m in zip(cost(c), most)):
            return c


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(shape, generator=g, device='cuda', dtype=torch.float32)


def _lengths(g, n, low, high):
    """Ragged lengths in low..high as int32; the first sequence is as long as they come."""
    x = torch.randint(low, high + 1, (n,), generator=g, device='cuda', dtype=torch.int32)
    x[0] = high
    return x


def _scale_of(amax):
    """The smallest power of two that keeps `amax` within e4m3's 448."""
    m, p = torch.frexp(amax)                   # amax = m 2^p, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, p - 9, p - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), e)


def _filled_cache(g, n, kv_heads, capacity, d):
    """A cache as a program has it after earlier steps: heads of different loudness, blocks with scales of their own."""
    loud = torch.exp(0.5 * _normal(g, n, kv_heads, 1, 1, 1))
    x = _normal(g, n, kv_heads, capacity // BLOCK, BLOCK, d) * loud
    scale = _scale_of(x.abs().amax((-1, -2)))
    code = (x / scale[..., None, None]).to(torch.float8_e4m3fn)
    return code.reshape(n, kv_heads, capacity, d), scale


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed))
    s = dict(case)
    if case['op'] == 'logprobs':
        rows, vocab, dtype = case['rows'], case['vocab'], TYPES[case['dtype']]
        x = _normal(g, rows, vocab) * 2.0
        token = torch.randint(0, vocab, (rows,), generator=g, device='cuda')
        sure = 4.0 + 6.0 * torch.rand((rows, 1), generator=g, device='cuda')      # a decoder is mostly sure of its token
        x.scatter_add_(1, token[:, None], sure)
        if case['masked']:                     # a third of the vocabulary is not admitted; the tokens are
            out = torch.rand((rows, vocab), generator=g, device='cuda') < 1 / 3
            out.scatter_(1, token[:, None], False)
            x.masked_fill_(out, float('-inf'))
        s['logits'], s['tokens'] = x.to(dtype), token.to(torch.int32)
    elif case['op'] == 'cross':
        n, tq, tk, d, dtype = case['n'], case['tq'], case['tk'], case['d'], TYPES[case['dtype']]
        s['q'] = _normal(g, n, tq, case['heads'], d).to(dtype)
        kv = _normal(g, n, tk, 2, case['kv_heads'], d).to(dtype)                  # one projection gives keys | values
        s['k'], s['v'] = kv[:, :, 0], kv[:, :, 1]
        s['lens'] = _lengths(g, n, (tk + 1) // 2, tk)
        s['pad_flags'] = torch.rand((n, tk), generator=g, device='cuda') < 0.05 if case['pad'] else None
    elif case['op'] == 'append':
        n, new, cap, hkv, d, dtype = (case[k] for k in ('n', 'new', 'capacity', 'kv_heads', 'd', 'dtype'))
        s['k_cache'], s['k_scale'] = _filled_cache(g, n, hkv, cap, d)
        s['v_cache'], s['v_scale'] = _filled_cache(g, n, hkv, cap, d)
        s['k'] = (_normal(g, n, new, hkv, d) * 1.5).to(TYPES[dtype])
        s['v'] = (_normal(g, n, new, hkv, d) * 1.5).to(TYPES[dtype])
        s['lens'] = _lengths(g, n, 0, case['held'])
        s['counts'] = _lengths(g, n, (new + 1) // 2, new)
    else:
        n, tq, cap, hkv, d = (case[k] for k in ('n', 'tq', 'capacity', 'kv_heads', 'd'))
        s['k_cache'], s['k_scale'] = _filled_cache(g, n, hkv, cap, d)
        s['v_cache'], s['v_scale'] = _filled_cache(g, n, hkv, cap, d)
        s['q'] = _normal(g, n, tq, case['heads'], d).to(TYPES[case['dtype']])
        s['lens'] = _lengths(g, n, max(tq, cap // 2), cap)
    return s


# ---- the operators in plain form -------------------------------------------------------------------------------------
def _plain_logprobs(logits, tokens, top):
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    none = m == float('-inf')                  # every token is masked out: log p = -inf, entropy 0
    d = x - m.masked_fill(none, 0.0)
    e = d.exp()
    s = e.sum(-1, keepdim=True)
    log_s = s.log()
    h = log_s - (e * d.clamp(min=-1e30)).sum(-1, keepdim=True) / s
    picked = d.gather(-1, tokens.long()[:, None]) - log_s
    lp = picked.masked_fill(none, float('-inf'))[:, 0]
    h = h.masked_fill(none, 0.0)[:, 0]
    # alternatives in the order of (logit, lowest index first): both in one 64-bit key
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7fffffff)).long() << 32
    key = order + (x.shape[-1] - 1 - torch.arange(x.shape[-1], device=x.device))
    best = key.topk(top, -1).values
    at = x.shape[-1] - 1 - (best & 0xffffffff)
    tops = (d.gather(-1, at) - log_s).masked_fill(none, float('-inf'))
    return lp, h, tops, at.to(torch.int32)


def _plain_attention(q, k, v, valid):
    """q [n, tq, H, d]; k, v [n, Hkv, tk, d] in 32 bits; valid [n, 1, tq or 1, tk]: rows with no valid key give 0."""
    n, tq, heads, d = q.shape
    hkv = k.shape[1]
    x = q.float().reshape(n, tq, hkv, heads // hkv, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)       # rows: tq x group
    s = torch.matmul(x, k.transpose(-1, -2)) * d ** -0.5
    rows = valid.expand(-1, -1, tq, -1).repeat_interleave(heads // hkv, 2)
    s = s.masked_fill(~rows, float('-inf'))
    m = s.amax(-1, keepdim=True).clamp(min=-3.0e38)
    p = (s - m).exp()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / l
    o = o.masked_fill(l == 0, 0.0)
    return o.reshape(n, hkv, tq, heads // hkv, d).permute(0, 2, 1, 3, 4).reshape(n, tq, heads, d).to(q.dtype)


def _plain_cross(q, k, v, lens, pad):
    valid = torch.arange(k.shape[1], device=q.device) < lens[:, None]
    if pad is not None:
        valid = valid & ~pad
    return _plain_attention(q, k.float().transpose(1, 2), v.float().transpose(1, 2), valid[:, None, None, :])


def _plain_attend(q, k_cache, v_cache, k_scale, v_scale, lens, causal):
    k = k_cache.float() * k_scale.repeat_interleave(BLOCK, -1)[..., None]
    v = v_cache.float() * v_scale.repeat_interleave(BLOCK, -1)[..., None]
    tq, at = q.shape[1], torch.arange(k.shape[2], device=q.device)
    last = lens[:, None].long().expand(-1, tq)
    if causal:                                 # query i is the sequence's token lens - tq + i
        last = last - (tq - 1) + torch.arange(tq, device=q.device)
    return _plain_attention(q, k, v, (at < last[..., None])[:, None])


def _plain_append(x, cache, scale, lens, counts):
    n, new, hkv, d = x.shape
    code = cache.view(torch.uint8).view(n, hkv, -1, BLOCK, d)
    touched = min((new + BLOCK - 2) // BLOCK + 1, code.shape[2])
    first = (lens.long() // BLOCK).clamp(max=code.shape[2] - touched)
    block = first[:, None] + torch.arange(touched, device=x.device)                            # [n, touched]
    pos = block[..., None] * BLOCK + torch.arange(BLOCK, device=x.device)                      # [n, touched, BLOCK]
    src = pos - lens[:, None, None]
    fresh = (src >= 0) & (src < counts[:, None, None])
    seq = torch.arange(n, device=x.device)[:, None]
    values = x.float()[seq[..., None], src.clamp(0, new - 1)]                                  # [n, touched, BLOCK, Hkv, d]
    values = values.masked_fill(~fresh[..., None, None], 0.0).permute(0, 1, 3, 2, 4)           # [n, touched, Hkv, BLOCK, d]
    was_code, was = code[seq, :, block], scale[seq, :, block]                                  # [n, touched, Hkv, ...]
    held = (lens[:, None] > block * BLOCK)[..., None]                                          # blocks with tokens of earlier calls
    now = _scale_of(values.abs().amax((-1, -2)))
    now = torch.where(held, torch.maximum(was, now), now)
    put = (values / now[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    kept = (was_code.view(torch.float8_e4m3fn).float() * (was / now)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    kept = torch.where((src < 0)[:, :, None, :, None], kept, was_code)
    change = fresh.any(-1)[..., None]                                                          # blocks that get a token
    put = torch.where(fresh[:, :, None, :, None], put, kept)
    code[seq, :, block] = torch.where(change[..., None, None], put, was_code)
    scale[seq, :, block] = torch.where(change, now, was)


def run(s):
    if own:
        from asr_amd import ops
        if s['op'] == 'logprobs':
            return ops.token_logprobs(s['logits'], s['tokens'], top=s['top'])
        if s['op'] == 'cross':
            return ops.cross_attention(s['q'], s['k'], s['v'], lens=s['lens'], pad=s['pad_flags'])
        if s['op'] == 'append':
            ops.kv8_append(s['k'], s['v'], s['k_cache'], s['v_cache'], s['k_scale'], s['v_scale'], s['lens'], counts=s['counts'])
            return s['k_cache'], s['v_cache'], s['k_scale'], s['v_scale']
        return ops.kv8_attention(s['q'], s['k_cache'], s['v_cache'], s['k_scale'], s['v_scale'], s['lens'], causal=s['causal'])
    if s['op'] == 'logprobs':
        return _plain_logprobs(s['logits'], s['tokens'], s['top'])
    if s['op'] == 'cross':
        return _plain_cross(s['q'], s['k'], s['v'], s['lens'], s['pad_flags'])
    if s['op'] == 'append':
        _plain_append(s['k'], s['k_cache'], s['k_scale'], s['lens'], s['counts'])
        _plain_append(s['v'], s['v_cache'], s['v_scale'], s['lens'], s['counts'])
        return s['k_cache'], s['v_cache'], s['k_scale'], s['v_scale']
    return _plain_attend(s['q'], s['k_cache'], s['v_cache'], s['k_scale'], s['v_scale'], s['lens'], s['causal'])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    """Bytes that have to move and operations that have to be done; ragged lengths count with their mean (three quarters
    of the longest), a causal chunk's newest tokens with half."""
    size = SIZE[case['dtype']]
    if case['op'] == 'logprobs':
        r, v = case['rows'], case['vocab']
        return {'bytes': r * v * size + r * (12 + 8 * case['top']), 'flops': 4.0 * r * v}
    d, hkv, n = case['d'], case['kv_heads'], case['n']
    if case['op'] == 'append':
        new = 0.75 * case['new'] if case['new'] > 1 else 1
        return {'bytes': n * hkv * 2 * (new * d * (size + 1) + 4 * max(1.0, new / BLOCK)), 'flops': n * hkv * 4.0 * new * d}
    tq, heads = case['tq'], case['heads']
    qo = 2 * n * tq * heads * d * size
    if case['op'] == 'cross':
        keys = 0.75 * case['tk'] if case['tk'] > 1 else 1
        return {'bytes': qo + n * hkv * keys * 2 * d * size, 'flops': 4.0 * n * heads * tq * keys * d}
    keys = (max(tq, case['capacity'] // 2) + case['capacity']) / 2
    seen = keys - (tq - 1) / 2 if case['causal'] else keys
    return {'bytes': qo + n * hkv * keys * 2 * (d + 4 / BLOCK), 'flops': 4.0 * n * heads * tq * seen * d}


# ---- the operators in 64 bits, from their definitions ------------------------------------------------------------------
def _exact_logprobs(s):
    lp, h, tops = [], [], []
    for x, token in zip(s['logits'].split(256), s['tokens'].long().split(256)):
        y = torch.log_softmax(x.double(), -1)
        lp.append(y.gather(-1, token[:, None])[:, 0])
        h.append(torch.special.entr(y.exp()).sum(-1))
        tops.append(y.sort(-1, descending=True).values[:, :s['top']])
    return torch.cat(lp), torch.cat(h), torch.cat(tops), None


def _exact_sequence(q, k, v, valid):
    """One sequence: q [tq, H, d], k, v [Hkv, tk, d], valid [tq, tk]."""
    out = torch.zeros_like(q, dtype=torch.float64)
    share = q.shape[1] // k.shape[0]
    for h in range(q.shape[1]):
        a = (q[:, h].double() @ k[h // share].double().t()) / q.shape[-1] ** 0.5
        p = torch.softmax(a.masked_fill(~valid, float('-inf')), -1)
        out[:, h] = torch.nan_to_num(p, nan=0.0) @ v[h // share].double()
    return out


def _exact_codes(x, cache, scale, lens, counts):
    """e4m3 by its definition: 3 bits behind the leading one, spacing 2^-9 at the least, halves to even."""
    def rounded(y):
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
        return (torch.round(y / step) * step).clamp(-448, 448)
    code, scale = cache.double(), scale.double().clone()
    x = x.double()
    for b in range(x.shape[0]):
        a, c = int(lens[b]), int(counts[b])
        for j in range(a // BLOCK, (a + c + BLOCK - 1) // BLOCK):
            lo, hi = max(a, j * BLOCK), min(a + c, (j + 1) * BLOCK)
            y = x[b, lo - a:hi - a].transpose(0, 1)                                            # [Hkv, tokens, d]
            need = torch.exp2(torch.ceil(torch.log2((y.abs().amax((1, 2)) / 448).clamp(min=2.0 ** MIN_EXP)) - 1e-13))
            if lo > j * BLOCK:
                need = torch.maximum(need, scale[b, :, j])
                code[b, :, j * BLOCK:lo] = rounded(code[b, :, j * BLOCK:lo] * (scale[b, :, j] / need)[:, None, None])
            code[b, :, lo:hi] = rounded(y / need[:, None, None])
            scale[b, :, j] = need
    return code, scale


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'logprobs':
        return _exact_logprobs(s)
    if case['op'] == 'append':
        k, ks = _exact_codes(s['k'], s['k_cache'], s['k_scale'], s['lens'], s['counts'])
        v, vs = _exact_codes(s['v'], s['v_cache'], s['v_scale'], s['lens'], s['counts'])
        return k, v, ks, vs
    tq, got = case['tq'], []
    for b in range(case['n']):
        length = int(s['lens'][b])
        if case['op'] == 'cross':
            k, v = s['k'][b].transpose(0, 1), s['v'][b].transpose(0, 1)
            valid = torch.arange(case['tk'], device='cuda') < length
            if case['pad']:
                valid = valid & ~s['pad_flags'][b]
            valid = valid.expand(tq, -1)
        else:
            k = s['k_cache'][b].double() * s['k_scale'][b].double().repeat_interleave(BLOCK, -1)[..., None]
            v = s['v_cache'][b].double() * s['v_scale'][b].double().repeat_interleave(BLOCK, -1)[..., None]
            at, i = torch.arange(case['capacity'], device='cuda'), torch.arange(tq, device='cuda')[:, None]
            valid = at <= length - tq + i if case['causal'] else (at < length).expand(tq, -1)
        got.append(_exact_sequence(s['q'][b], k, v, valid))
    return torch.stack(got)
