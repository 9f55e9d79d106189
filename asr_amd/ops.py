"""Operators on torch tensors in GPU memory (`include/asr_amd.h`, "operators on device memory").

    token_logprobs   log p(token), entropy and the most likely alternatives of rows of logits
    cross_attention  attention over the states of another sequence, e.g. an encoder's
    kv8_cache        an empty K/V cache held in 8 bits
    kv8_append       new keys and values behind what such a cache holds
    kv8_attention    attention over such a cache

The work is queued on the current stream of the tensors' device, like torch's own operators: nothing here waits for the GPU, results are
torch tensors of the caller's allocator, and a call can be captured into a graph.  Tensors that were made on another stream
need that stream waited for first (and `record_stream`), as with every torch operator.  There is no backward pass: tensors that
require gradients are refused while gradients are recorded.

Wrong types, shapes or devices raise ValueError; what the library itself refuses raises `AsrError`.
"""
from __future__ import annotations

import functools
import struct

import torch

from ._lib import AsrError, lib

KV8_BLOCK = 64                                # tokens of a head that share one scale (ASR_KV8_BLOCK)

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}             # enum asr_dtype
# the argument structs of include/asr_amd.h, packed as C lays them out
_LOGPROBS = struct.Struct('@6P2q4i')
_CROSS = struct.Struct('@7P14q7if')
_APPEND = struct.Struct('@8P8q6i')
_ATTEND = struct.Struct('@8P9q8if4x')


def _call(fn, packed, device):
    """fn(packed arguments) on `device`'s current stream."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(packed, torch.cuda.current_stream(index).cuda_stream)
    else:
        with torch.cuda.device(index):
            rc = fn(packed, torch.cuda.current_stream(index).cuda_stream)
    if rc:
        raise AsrError(rc, lib.asr_ops_last_error().decode('utf-8', 'replace'))


def _require(ok, what):
    if not ok:
        raise ValueError(what)


def _inputs(name, device, *tensors):
    _require(device.type == 'cuda', '%s: tensors must be in GPU memory' % name)
    grads = torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        _require(t.device == device, '%s: all tensors must be on one device' % name)
        _require(not (grads and t.requires_grad), '%s has no backward pass: detach its inputs or call it under torch.no_grad()' % name)


def _counts(name, what, t, n):
    _require(t.dtype == torch.int32 and t.shape == (n,) and t.is_contiguous(), '%s: %s must be int32 [%d]' % (name, what, n))


def token_logprobs(logits, tokens, top=0):
    """logits [..., vocab] (float32, bfloat16 or float16; vocabulary contiguous), tokens [...] (int32 or int64) ->
    (logprob [...], entropy [...], top_logprobs [..., top], top_tokens [..., top]) in float32 and int32.

    log p(token) and the entropy of softmax(logits) per row in float32, and the `top` (at most 32) most likely tokens with their log
    probabilities, the most likely first, ties to the lower token.  A negative token is "no token": its log probability is 0;
    one beyond the vocabulary gives NaN.  -infinity masks a token out; a row with nothing else has log p = -infinity, entropy 0."""
    _inputs('token_logprobs', logits.device, logits, tokens)
    dtype = _DTYPES.get(logits.dtype)
    _require(dtype is not None, 'token_logprobs: logits must be float32, bfloat16 or float16')
    _require(logits.dim() >= 1 and logits.shape[-1] >= 1, 'token_logprobs: logits must be [..., vocab] with a vocabulary')
    vocab, lead = logits.shape[-1], logits.shape[:-1]
    _require(tokens.shape == lead, 'token_logprobs: tokens must have the shape of logits without its last dimension')
    _require(tokens.dtype in (torch.int32, torch.int64), 'token_logprobs: tokens must be int32 or int64')
    _require(0 <= top <= min(32, vocab), 'token_logprobs: top must be in 0..min(32, vocab)')
    _require(vocab == 1 or logits.stride(-1) == 1, 'token_logprobs: the vocabulary must be contiguous')
    if logits.dim() != 2:
        logits = logits.reshape(-1, vocab) if logits.numel() else logits.new_empty((tokens.numel(), vocab))
    tokens = tokens.contiguous()
    rows, device = tokens.numel(), logits.device
    both = torch.empty((2,) + tuple(lead), dtype=torch.float32, device=device)
    logprob, entropy = both.unbind(0)
    top_logprobs = torch.empty(tuple(lead) + (top,), dtype=torch.float32, device=device)
    top_tokens = torch.empty(tuple(lead) + (top,), dtype=torch.int32, device=device)
    if rows:
        _call(lib.asr_token_logprobs,
              _LOGPROBS.pack(logits.data_ptr(), tokens.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), top_logprobs.data_ptr(),
                             top_tokens.data_ptr(), rows, logits.stride(0) if rows > 1 else 0, vocab, top, dtype, tokens.element_size()), device)
    return logprob, entropy, top_logprobs, top_tokens


@functools.lru_cache(maxsize=4096)
def _cross_workspace(n, tq, tk, heads, kv_heads, d, dtype):
    return lib.asr_cross_attention_workspace(n, tq, tk, heads, kv_heads, d, dtype)


@functools.lru_cache(maxsize=4096)
def _kv8_workspace(n, tq, capacity, heads, kv_heads, d, dtype):
    return lib.asr_kv8_attention_workspace(n, tq, capacity, heads, kv_heads, d, dtype)


def _rows(name, what, t, dims):
    """Strides of a [n, t, heads, d] tensor whose rows are contiguous."""
    _require(t.dim() == 4 and t.shape == dims, '%s: %s must be %s' % (name, what, list(dims)))
    s = t.stride()
    _require(s[3] == 1 or dims[3] == 1, '%s: the last dimension of %s must be contiguous' % (name, what))
    return s


def _output(name, q, out):
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _require(out.dtype == q.dtype and out.shape == q.shape, '%s: out must have the shape and type of q' % name)
    _require(all(s > 0 or n <= 1 for s, n in zip(out.stride(), out.shape)), '%s: out must not be expanded' % name)
    return out


def cross_attention(q, k, v, lens=None, pad=None, scale=None, out=None):
    """q [n, tq, heads, d], k and v [n, tk, kv_heads, d] (float32, bfloat16 or float16) -> [n, tq, heads, d] of q's type.

    softmax(scale q k^T) v per sequence and head, query head h reading key head h // (heads // kv_heads); scale defaults to
    1 / sqrt(d).  Admitted are the first lens[b] (int32 [n]; None: all) states of which pad[b] (bool or uint8 [n, tk]; None: none) is zero; whatever
    stands in the others does not matter, and a sequence without any gives zeros.  Beams of an utterance are its query rows.
    d is a multiple of 8 up to 128; rows start on 16 bytes; other strides are free (k and v may be the halves of one projection)."""
    name = 'cross_attention'
    _inputs(name, q.device, q, k, v, lens, pad, out)
    dtype = _DTYPES.get(q.dtype)
    _require(dtype is not None and k.dtype == q.dtype and v.dtype == q.dtype, '%s: q, k and v must be float32, bfloat16 or float16, all the same' % name)
    _require(q.dim() == 4 and k.dim() == 4, '%s: q must be [n, tq, heads, d] and k [n, tk, kv_heads, d]' % name)
    n, tq, heads, d = q.shape
    tk, kv_heads = k.shape[1], k.shape[2]
    qs = _rows(name, 'q', q, (n, tq, heads, d))
    ks = _rows(name, 'k', k, (n, tk, kv_heads, d))
    vs = _rows(name, 'v', v, (n, tk, kv_heads, d))
    if lens is not None:
        _counts(name, 'lens', lens, n)
    pad_stride = 0
    if pad is not None:
        _require(pad.dtype in (torch.bool, torch.uint8) and pad.shape == (n, tk) and (tk <= 1 or pad.stride(1) == 1),
                 '%s: pad must be bool or uint8 [n, tk], contiguous in tk' % name)
        pad_stride = pad.stride(0)
    out = _output(name, q, out)
    os = _rows(name, 'out', out, (n, tq, heads, d))
    size = _cross_workspace(n, tq, tk, heads, kv_heads, d, dtype)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _call(lib.asr_cross_attention,
          _CROSS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lens is None else lens.data_ptr(),
                      0 if pad is None else pad.data_ptr(), 0 if ws is None else ws.data_ptr(), *qs[:3], *ks[:3], *vs[:3], *os[:3],
                      pad_stride, size, n, tq, tk, heads, kv_heads, d, dtype, d ** -0.5 if scale is None else scale), q.device)
    return out


def kv8_cache(n, kv_heads, capacity, d, device='cuda'):
    """An empty cache for n sequences of up to `capacity` tokens (a multiple of KV8_BLOCK): (k_cache, v_cache, k_scale, v_scale), the
    codes as float8_e4m3fn [n, kv_heads, capacity, d] and their scales as float32 [n, kv_heads, capacity // KV8_BLOCK].  A value is
    code * scale; how many tokens a sequence holds is the caller's to keep."""
    _require(capacity % KV8_BLOCK == 0, 'kv8_cache: the capacity must be a multiple of %d tokens' % KV8_BLOCK)
    codes = [torch.zeros((n, kv_heads, capacity, d), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones((n, kv_heads, capacity // KV8_BLOCK), dtype=torch.float32, device=device) for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def _cache(name, k_cache, v_cache, k_scale, v_scale):
    _require(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.dtype == torch.float8_e4m3fn and v_cache.dtype == torch.float8_e4m3fn,
             '%s: k_cache and v_cache must be float8_e4m3fn [n, kv_heads, capacity, d]' % name)
    n, kv_heads, capacity, d = k_cache.shape
    s = k_cache.stride()
    _require(s == v_cache.stride() and s[3] == 1 and (s[2] == d or capacity <= 1), '%s: the caches must have equal strides and contiguous tokens' % name)
    for scale in (k_scale, v_scale):
        _require(scale.dtype == torch.float32 and scale.shape == (n, kv_heads, capacity // KV8_BLOCK) and scale.is_contiguous(),
                 '%s: scales must be float32 [n, kv_heads, capacity / %d], contiguous' % (name, KV8_BLOCK))
    return n, kv_heads, capacity, d, s


def kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, lens, counts=None):
    """Writes the new tokens k, v [n, new, kv_heads, d] (float32, bfloat16 or float16) into the caches, sequence b's first
    counts[b] (int32 [n]; None: all) of them at positions lens[b], lens[b] + 1, ...  The caller's lens stay as they are.

    A block of KV8_BLOCK tokens has one scale: the smallest power of two that keeps its magnitudes within 448.  A block that already
    held tokens keeps its scale or takes the larger one the new tokens need, and its older tokens are coded again under it.  Tokens past the
    capacity are dropped; a sequence with a negative length or no new token is left alone; no other position changes."""
    name = 'kv8_append'
    _inputs(name, k.device, k, v, k_cache, v_cache, k_scale, v_scale, lens, counts)
    n, kv_heads, capacity, d, cs = _cache(name, k_cache, v_cache, k_scale, v_scale)
    dtype = _DTYPES.get(k.dtype)
    _require(dtype is not None and v.dtype == k.dtype, '%s: k and v must be float32, bfloat16 or float16, both the same' % name)
    _require(k.dim() == 4, '%s: k must be [n, new, kv_heads, d]' % name)
    new = k.shape[1]
    ks = _rows(name, 'k', k, (n, new, kv_heads, d))
    vs = _rows(name, 'v', v, (n, new, kv_heads, d))
    _require(all(cs[i] > 0 or k_cache.shape[i] <= 1 for i in (0, 1)), '%s: the caches must not be expanded' % name)
    _counts(name, 'lens', lens, n)
    if counts is not None:
        _counts(name, 'counts', counts, n)
    _call(lib.asr_kv8_append,
          _APPEND.pack(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                       lens.data_ptr(), 0 if counts is None else counts.data_ptr(), *ks[:3], *vs[:3], cs[0], cs[1], n, new, kv_heads, d,
                       capacity, dtype), k.device)


def kv8_attention(q, k_cache, v_cache, k_scale, v_scale, lens, causal=False, scale=None, out=None):
    """q [n, tq, heads, d] (float32, bfloat16 or float16) over the first lens[b] (int32 [n]) tokens of each sequence's cache ->
    [n, tq, heads, d] of q's type.  causal: query i is the sequence's token lens[b] - tq + i, which the cache already holds, and sees nothing behind
    itself.  A query with nothing to see gives zeros; what stands behind lens[b] does not matter.  Query head h reads key head
    h // (heads // kv_heads); scale defaults to 1 / sqrt(d); d is a multiple of 16 up to 128."""
    name = 'kv8_attention'
    _inputs(name, q.device, q, k_cache, v_cache, k_scale, v_scale, lens, out)
    n, kv_heads, capacity, d, cs = _cache(name, k_cache, v_cache, k_scale, v_scale)
    dtype = _DTYPES.get(q.dtype)
    _require(dtype is not None, '%s: q must be float32, bfloat16 or float16' % name)
    _require(q.dim() == 4 and q.shape[0] == n and q.shape[3] == d, '%s: q must be [%d, tq, heads, %d]' % (name, n, d))
    _, tq, heads, _ = q.shape
    qs = _rows(name, 'q', q, (n, tq, heads, d))
    _counts(name, 'lens', lens, n)
    out = _output(name, q, out)
    os = _rows(name, 'out', out, (n, tq, heads, d))
    size = _kv8_workspace(n, tq, capacity, heads, kv_heads, d, dtype)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _call(lib.asr_kv8_attention,
          _ATTEND.pack(q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                       lens.data_ptr(), 0 if ws is None else ws.data_ptr(), *qs[:3], *os[:3], cs[0], cs[1], size, n, tq, heads, kv_heads,
                       d, capacity, dtype, 1 if causal else 0, d ** -0.5 if scale is None else scale), q.device)
    return out
