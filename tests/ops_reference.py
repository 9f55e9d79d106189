"""The operators of asr_amd.ops in 64 bits on the CPU, straight from their definitions, and the error bounds the tests hold the kernels to."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # torch.finfo(t).eps / 2
U = 2.0 ** -24


# ---- token_logprobs ----------------------------------------------------------------------------------------------------
def token_logprobs(logits, tokens, top):
    """[rows, vocab], [rows] -> log p, entropy, the alternatives' log p, their tokens (float64, int64)."""
    x = logits.detach().cpu().double()
    rows, vocab = x.shape
    m = x.max(-1, keepdim=True).values
    none = torch.isneginf(m)
    m = torch.where(none, torch.zeros_like(m), m)
    e = torch.exp(x - m)
    s = e.sum(-1, keepdim=True)
    y = x - m - torch.log(s)
    p = e / s
    h = -torch.where(p > 0, p * y, torch.zeros_like(p)).sum(-1)
    h = torch.where(torch.isnan(s[:, 0]), s[:, 0], h)
    y = torch.where(none & (s == 0), torch.full_like(y, -math.inf), y)
    h = torch.where(none[:, 0] & (s[:, 0] == 0), torch.zeros_like(h), h)
    lp = torch.empty(rows, dtype=torch.float64)
    for r, t in enumerate(tokens.tolist()):
        lp[r] = 0.0 if t < 0 else math.nan if t >= vocab else y[r, t]
    order = x.sort(dim=-1, descending=True, stable=True).indices[:, :top]            # stable: ties to the lower token
    return lp, h, y.gather(-1, order), order


def logprob_bound(logits):
    """Absolute error of log p and (times 1 + H) of the entropy, per row, in units that follow the float32 arithmetic: every e^(x-m) is off by at
    most (3 |x - m| + 4) u of itself (the difference, the factor log2 e, the product, exp2), which weighted by p is at most (3 (ln V + 1) + 4) u; a
    sum of V terms in strips of at least 256 threads adds (V / 256 + 32) u (a strip, its rescalings, 6 + 4 joins); x - m and the
    subtraction of ln S are rounded once each."""
    x = logits.detach().cpu().double()
    vocab = x.shape[-1]
    finite = torch.where(torch.isfinite(x) & (x > -1e30), x, torch.full_like(x, math.nan))
    span = (torch.nan_to_num(finite, nan=-math.inf).max(-1).values - torch.nan_to_num(finite, nan=math.inf).min(-1).values).clamp(min=0)
    span = torch.where(torch.isfinite(span), span, torch.zeros_like(span))
    return U * (3 * (math.log(vocab) + 1) + 4 + vocab / 256 + 32 + 3 * span + 2 * math.log(vocab))


# ---- attention ---------------------------------------------------------------------------------------------------------
def attention(q, k, v, admitted, scale):
    """q [n, tq, H, d]; k, v [n, Hkv, tk, d] in float64; admitted [n, tq, tk] -> out and what the error bound needs, in float64."""
    q = q.detach().cpu().double()
    n, tq, heads, d = q.shape
    out = torch.zeros(n, tq, heads, d, dtype=torch.float64)
    weight = torch.zeros_like(out)                            # sum p |v|
    size = torch.zeros(n, tq, heads, 1, dtype=torch.float64)  # largest sum |q| |k| times scale
    group = heads // k.shape[1]
    for b in range(n):
        for h in range(heads):
            kk = torch.nan_to_num(k[b, h // group], nan=0.0, posinf=0.0, neginf=0.0) if k.shape[2] else k[b, h // group]
            vv = torch.nan_to_num(v[b, h // group], nan=0.0, posinf=0.0, neginf=0.0) if k.shape[2] else v[b, h // group]
            if not k.shape[2]:
                continue
            s = (q[b, :, h] @ kk.T) * scale
            a = admitted[b]
            p = torch.softmax(s.masked_fill(~a, -math.inf), -1)
            p = torch.where(a, torch.nan_to_num(p, nan=0.0), torch.zeros_like(p))
            out[b, :, h] = p @ vv
            weight[b, :, h] = p @ vv.abs()
            size[b, :, h, 0] = ((q[b, :, h].abs() @ kk.abs().T) * abs(scale)).masked_fill(~a, 0).max(-1).values
    return out, weight, size


def attention_bound(out, weight, size, d, tk, dtype, vmax):
    """A score is off by at most (d + 8) u sum|q||k| scale (products exact or rounded once, d additions, the factor), so a probability by twice
    that plus 2^-22 (exp2) of itself, and half a step of its own type where it is rounded to 16 bits before it meets V (float16: 2^-25 at the
    least); the sums over tk keys add (tk / 8 + 64) u.  Numerator and denominator both carry it: twice.  The result is rounded once."""
    p = 2 * (d + 8) * U * size + 2.0 ** -22 + (tk / 8 + 64) * U
    if dtype != torch.float32:
        p = p + HALF_STEP[dtype]
    least = tk * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0
    return 2 * p * weight + least + HALF_STEP[dtype] * out.abs() + 1e-30


# ---- the 8-bit cache ---------------------------------------------------------------------------------------------------
BLOCK = 64
CODES = torch.tensor([(-1.0) ** (c >> 7) * (math.nan if c & 127 == 127 else (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10) if c >> 3 & 15 else
                                             (c & 7) * 2.0 ** -9) for c in range(256)], dtype=torch.float64)
_POSITIVE = CODES[:127]                                       # 0 .. 448 ascending


def to_code(x):
    """Nearest e4m3 value (not code number) of float64 x: halves to the even code, infinities to +-448, NaN stays."""
    a = x.abs().clamp(max=448.0)
    up = torch.searchsorted(_POSITIVE, a.contiguous()).clamp(max=126)
    lo = (up - 1).clamp(min=0)
    dl, du = a - _POSITIVE[lo], _POSITIVE[up] - a
    pick = torch.where(dl < du, lo, torch.where(du < dl, up, torch.where(lo % 2 == 0, lo, up)))
    y = _POSITIVE[pick] * torch.where(x < 0, -1.0, 1.0)
    return torch.where(torch.isnan(x), x, y)


def exponent(values):
    """Smallest e >= -100 with every finite |value| <= 448 * 2^e."""
    a = values.abs()
    a = a[torch.isfinite(a)]
    top = float(a.max()) if a.numel() else 0.0
    e = -100
    if top > 0:
        e = max(-100, math.frexp(top)[1] - 12)
        while top > 448.0 * 2.0 ** e:
            e += 1
    return e


def append(x, codes, scales, lens, counts):
    """One of K and V: x [n, new, Hkv, d]; codes (values of e4m3) [n, Hkv, capacity, d], scales, in float64 -> the new ones."""
    x = x.detach().cpu().double()
    codes, scales = codes.clone(), scales.clone()
    n, new, heads, _ = x.shape
    capacity = codes.shape[2]
    for b in range(n):
        a, c = int(lens[b]), min(new if counts is None else int(counts[b]), new)
        if a < 0:
            continue
        end = min(capacity, a + max(c, 0))
        for h in range(heads):
            for j in range(a // BLOCK, (end + BLOCK - 1) // BLOCK):
                lo, hi = max(a, j * BLOCK), min(end, (j + 1) * BLOCK)
                if lo >= hi:
                    continue
                e = exponent(x[b, lo - a:hi - a, h])
                if a > j * BLOCK:
                    was = round(math.log2(float(scales[b, h, j])))
                    if e > was:
                        codes[b, h, j * BLOCK:a] = to_code(codes[b, h, j * BLOCK:a] * 2.0 ** (was - e))
                    e = max(e, was)
                codes[b, h, lo:hi] = to_code(x[b, lo - a:hi - a, h] * 2.0 ** -e)
                scales[b, h, j] = 2.0 ** e
    return codes, scales


def values_of(cache):
    """e4m3 codes of a float8 tensor as float64 on the CPU."""
    return CODES[cache.detach().view(torch.uint8).cpu().long()]
