"""Operators on torch tensors in GPU memory (`include/asr_amd.h`, "operators on device memory").

    token_logprobs   log p(token), entropy and the most likely alternatives of rows of logits
    cross_attention  attention over the states of another sequence, e.g. an encoder's
    kv8_cache        an empty K/V cache held in 8 bits
    kv8_append       new keys and values behind what such a cache holds
    kv8_attention    attention over such a cache

The work is queued on the current stream of the tensors' device, like torch's own operators: nothing here waits for the GPU, results are
torch tensors of the caller's allocator, and a call can be captured into a graph.  Tensors that were made on another stream
need that stream waited for first (and `record_stream`), as with every torch operator.  There is no backward pass and no
forward-mode derivative: tensors that require gradients while these are recorded, and tensors with a tangent, are refused.  So are
tensors without memory of their own (fake ones, wrappers).

Wrong types, shapes or devices raise ValueError; what the library itself refuses raises `AsrError`.
"""
from __future__ import annotations

import functools
import struct

import torch
from torch.autograd import forward_ad

from ._lib import AsrError, lib

KV8_BLOCK = 64                                # tokens of a head that share one scale (ASR_KV8_BLOCK)

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}             # enum asr_dtype
# the argument structs of include/asr_amd.h, packed as C lays them out
_LOGPROBS = struct.Struct('@6P2q4i')
_CROSS = struct.Struct('@7P14q7if')
_APPEND = struct.Struct('@8P8q6i')
_ATTEND = struct.Struct('@8P9q8if4x')


_Tensor = torch.Tensor
_plain = torch._C._disabled_torch_dispatch_impl       # what tensors have for __torch_dispatch__ that are no wrappers
_changed = torch._C._increment_version                 # tensors that were written in place: autograd is told, as torch's own operators do
_raw_stream = torch._C._cuda_getCurrentRawStream      # the current stream's handle without the Stream object around it (1 us a call)


def _call(fn, packed, device, *more):
    """fn(packed arguments, more) on the current stream of the device with this number."""
    if device == torch.cuda.current_device():
        rc = fn(packed, *more, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(packed, *more, _raw_stream(device))
    if rc:
        raise AsrError(rc, lib.asr_ops_last_error().decode('utf-8', 'replace'))


# The checks below run before every call: a message is only put together when it is needed.
def _refused(name, *tensors):
    """Why these tensors cannot be used together - they have no memory, are not all on one GPU, want derivatives - or None."""
    device = tensors[0].get_device()
    if any(type(t).__torch_dispatch__ is not _plain for t in tensors):
        return ValueError('%s: tensors must have memory of their own (no fake tensors, no wrappers)' % name)
    if device < 0:
        return ValueError('%s: tensors must be in GPU memory' % name)
    if any(t.get_device() != device for t in tensors):
        return ValueError('%s: all tensors must be on one device' % name)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return ValueError('%s has no backward pass: detach its inputs or call it under torch.no_grad()' % name)
    if torch._C._is_fwd_grad_enabled() and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        return ValueError('%s has no forward-mode derivative: call it on the primals (torch.autograd.forward_ad.unpack_dual)' % name)
    return None


def _device(name, *tensors):
    """The number of the one device that holds all tensors (None entries are skipped)."""
    device = tensors[0].get_device()
    grads = torch.is_grad_enabled()
    odd = device < 0 or forward_ad._current_level >= 0                  # (tensors have tangents inside a dual level alone)
    for t in tensors:
        if t is not None and (t.get_device() != device or (grads and t.requires_grad) or type(t) is not _Tensor):
            odd = True
    if odd:
        error = _refused(name, *[t for t in tensors if t is not None])
        if error is not None:
            raise error
    return device


def _counts(name, what, t, n):
    if t.dtype is not torch.int32 or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError('%s: %s must be int32 [%d], contiguous' % (name, what, n))


def _rows(name, what, t, dims):
    """Strides of a tensor of these dimensions [n, rows, heads, d] whose last one is contiguous."""
    if t.shape != dims:
        raise ValueError('%s: %s must be %s, not %s' % (name, what, list(dims), list(t.shape)))
    a, b, c, one = t.stride()
    if one != 1 and dims[3] != 1:
        raise ValueError('%s: the last dimension of %s must be contiguous' % (name, what))
    return a, b, c


def _output(name, q, out, k=None, v=None):
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if k is not None and out.numel() and out.data_ptr() in (k.data_ptr(), v.data_ptr()):
        raise ValueError('%s: out must not overlap k or v' % name)
    if out.dtype != q.dtype or out.shape != q.shape:
        raise ValueError('%s: out must have the shape and type of q' % name)
    if not all(s > 0 or n <= 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError('%s: out must not be expanded' % name)
    return out


def token_logprobs(logits, tokens, top=0):
    """logits [..., vocab] (float32, bfloat16 or float16; vocabulary contiguous), tokens [...] (int32 or int64) ->
    (logprob [...], entropy [...], top_logprobs [..., top], top_tokens [..., top]) in float32 and int32.

    log p(token) and the entropy of softmax(logits) per row in float32, and the `top` (at most 32) most likely tokens with their log
    probabilities, the most likely first, ties to the lower token.  A negative token is "no token": its log probability is 0;
    one beyond the vocabulary gives NaN.  -infinity masks a token out; a row with nothing else has log p = -infinity, entropy 0."""
    device = _device('token_logprobs', logits, tokens)
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None:
        raise ValueError('token_logprobs: logits must be float32, bfloat16 or float16')
    shape = logits.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError('token_logprobs: logits must be [..., vocab] with a vocabulary')
    vocab, lead = shape[-1], tuple(shape[:-1])
    if tokens.shape != lead:
        raise ValueError('token_logprobs: tokens must have the shape of logits without its last dimension')
    if tokens.dtype is not torch.int32 and tokens.dtype is not torch.int64:
        raise ValueError('token_logprobs: tokens must be int32 or int64')
    if vocab > 1 << 30:
        raise ValueError('token_logprobs: a vocabulary of at most 2^30 tokens')
    if not 0 <= top <= min(32, vocab):
        raise ValueError('token_logprobs: top must be in 0..min(32, vocab)')
    if vocab > 1 and logits.stride(-1) != 1:
        raise ValueError('token_logprobs: the vocabulary must be contiguous')
    logprob = logits.new_empty(lead, dtype=torch.float32)
    entropy = logits.new_empty(lead, dtype=torch.float32)
    top_logprobs = logits.new_empty(lead + (top,), dtype=torch.float32)
    top_tokens = logits.new_empty(lead + (top,), dtype=torch.int32)
    rows = tokens.numel()
    if rows:
        if len(shape) != 2:
            logits = logits.reshape(rows, vocab)
        if not tokens.is_contiguous():
            tokens = tokens.contiguous()
        _call(lib.asr_token_logprobs,
              _LOGPROBS.pack(logits.data_ptr(), tokens.data_ptr(), logprob.data_ptr(), entropy.data_ptr(), top_logprobs.data_ptr(),
                             top_tokens.data_ptr(), rows, logits.stride(0) if rows > 1 else 0, vocab, top, dtype, tokens.element_size()), device)
    return logprob, entropy, top_logprobs, top_tokens


def _sizes(name, *sizes):
    if max(sizes) >= 1 << 31:
        raise ValueError('%s: sizes must be below 2^31' % name)


@functools.lru_cache(maxsize=4096)
def _cross_workspace(n, tq, tk, heads, kv_heads, d, dtype):
    _sizes('cross_attention', n, tq, tk, heads)
    return lib.asr_cross_attention_workspace(n, tq, tk, heads, kv_heads, d, dtype)


@functools.lru_cache(maxsize=4096)
def _kv8_workspace(n, tq, capacity, heads, kv_heads, d, dtype):
    _sizes('kv8_attention', n, tq, capacity, heads)
    return lib.asr_kv8_attention_workspace(n, tq, capacity, heads, kv_heads, d, dtype)


def cross_attention(q, k, v, lens=None, pad=None, scale=None, out=None):
    """q [n, tq, heads, d], k and v [n, tk, kv_heads, d] (float32, bfloat16 or float16) -> [n, tq, heads, d] of q's type.

    softmax(scale q k^T) v per sequence and head, query head h reading key head h // (heads // kv_heads); scale defaults to
    1 / sqrt(d).  Admitted are the first lens[b] (int32 [n]; None: all) states of which pad[b] (bool or uint8 [n, tk]; None: none) is zero; whatever
    stands in the others does not matter, and a sequence without any gives zeros.  Beams of an utterance are its query rows.
    d is a multiple of 8 up to 128; rows start on 16 bytes; other strides are free (k and v may be the halves of one projection).  out must not overlap the
    inputs (the same memory as k or v is refused)."""
    name = 'cross_attention'
    device = _device(name, q, k, v, lens, pad, out)
    dtype = _DTYPES.get(q.dtype)
    if dtype is None or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError('%s: q, k and v must be float32, bfloat16 or float16, all the same' % name)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError('%s: q must be [n, tq, heads, d] and k [n, tk, kv_heads, d]' % name)
    n, tq, heads, d = dims = q.shape
    _, tk, kv_heads, _ = k.shape
    kv_dims = (n, tk, kv_heads, d)
    qs = _rows(name, 'q', q, dims)
    ks = _rows(name, 'k', k, kv_dims)
    vs = _rows(name, 'v', v, kv_dims)
    if lens is not None:
        _counts(name, 'lens', lens, n)
    pad_stride = 0
    if pad is not None:
        if (pad.dtype is not torch.bool and pad.dtype is not torch.uint8) or pad.shape != (n, tk) or (tk > 1 and pad.stride(1) != 1):
            raise ValueError('%s: pad must be bool or uint8 [n, tk], contiguous in tk' % name)
        pad_stride = pad.stride(0)
    given = out is not None
    out = _output(name, q, out, k, v)
    size = _cross_workspace(n, tq, tk, heads, kv_heads, d, dtype)
    ws = q.new_empty((size,), dtype=torch.uint8) if size else None
    _call(lib.asr_cross_attention,
          _CROSS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lens is None else lens.data_ptr(),
                      0 if pad is None else pad.data_ptr(), 0 if ws is None else ws.data_ptr(), *qs, *ks, *vs, *out.stride()[:3],
                      pad_stride, size, n, tq, tk, heads, kv_heads, d, dtype, (d or 1) ** -0.5 if scale is None else scale), device)
    if given:
        _changed((out,))
    return out


def kv8_cache(n, kv_heads, capacity, d, device='cuda'):
    """An empty cache for n sequences of up to `capacity` tokens (a multiple of KV8_BLOCK): (k_cache, v_cache, k_scale, v_scale), the
    codes as float8_e4m3fn [n, kv_heads, capacity, d] and their scales as float32 [n, kv_heads, capacity // KV8_BLOCK].  A value is
    code * scale; how many tokens a sequence holds is the caller's to keep."""
    if capacity % KV8_BLOCK:
        raise ValueError('kv8_cache: the capacity must be a multiple of %d tokens' % KV8_BLOCK)
    codes = [torch.zeros((n, kv_heads, capacity, d), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones((n, kv_heads, capacity // KV8_BLOCK), dtype=torch.float32, device=device) for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def _cache(name, k_cache, v_cache, k_scale, v_scale):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype is not torch.float8_e4m3fn or v_cache.dtype is not torch.float8_e4m3fn:
        raise ValueError('%s: k_cache and v_cache must be float8_e4m3fn [n, kv_heads, capacity, d]' % name)
    n, kv_heads, capacity, d = k_cache.shape
    s = k_cache.stride()
    if s != v_cache.stride() or s[3] != 1 or (s[2] != d and capacity > 1):
        raise ValueError('%s: the caches must have equal strides and contiguous tokens' % name)
    dims = (n, kv_heads, capacity // KV8_BLOCK)
    for scale in (k_scale, v_scale):
        if scale.dtype is not torch.float32 or scale.shape != dims or not scale.is_contiguous():
            raise ValueError('%s: scales must be float32 %s, contiguous' % (name, list(dims)))
    return n, kv_heads, capacity, d, s


def kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, lens, counts=None):
    """Writes the new tokens k, v [n, new, kv_heads, d] (float32, bfloat16 or float16) into the caches, sequence b's first
    counts[b] (int32 [n]; None: all) of them at positions lens[b], lens[b] + 1, ...  The caller's lens stay as they are.

    A block of KV8_BLOCK tokens has one scale: the smallest power of two that keeps its magnitudes within 448.  A block that already
    held tokens keeps its scale or takes the larger one the new tokens need, and its older tokens are coded again under it.  Tokens past the
    capacity are dropped; a sequence with a negative length or no new token is left alone; no other position changes."""
    name = 'kv8_append'
    device = _device(name, k, v, k_cache, v_cache, k_scale, v_scale, lens, counts)
    n, kv_heads, capacity, d, cs = _cache(name, k_cache, v_cache, k_scale, v_scale)
    dtype = _DTYPES.get(k.dtype)
    if dtype is None or v.dtype is not k.dtype:
        raise ValueError('%s: k and v must be float32, bfloat16 or float16, both the same' % name)
    if k.dim() != 4:
        raise ValueError('%s: k must be [n, new, kv_heads, d]' % name)
    new = k.shape[1]
    if new >= 1 << 31 or capacity >= 1 << 31:
        raise ValueError('%s: sizes must be below 2^31' % name)
    dims = (n, new, kv_heads, d)
    ks = _rows(name, 'k', k, dims)
    vs = _rows(name, 'v', v, dims)
    if (cs[0] <= 0 and n > 1) or (cs[1] <= 0 and kv_heads > 1):
        raise ValueError('%s: the caches must not be expanded' % name)
    _counts(name, 'lens', lens, n)
    if counts is not None:
        _counts(name, 'counts', counts, n)
    _call(lib.asr_kv8_append,
          _APPEND.pack(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                       lens.data_ptr(), 0 if counts is None else counts.data_ptr(), *ks, *vs, cs[0], cs[1], n, new, kv_heads, d,
                       capacity, dtype), device)
    _changed((k_cache, v_cache, k_scale, v_scale))


def kv8_attention(q, k_cache, v_cache, k_scale, v_scale, lens, causal=False, scale=None, out=None, counts=None):
    """q [n, tq, heads, d] (float32, bfloat16 or float16) over the first lens[b] (int32 [n]) tokens of each sequence's cache ->
    [n, tq, heads, d] of q's type.  causal: query i is the sequence's token lens[b] - tq + i, which the cache already holds, and sees nothing behind
    itself.  A query with nothing to see gives zeros; what it does not see does not matter, NaN included.  Query head h reads key head
    h // (heads // kv_heads); scale defaults to 1 / sqrt(d); d is a multiple of 16 up to 128.

    counts (int32 [n]; None: tq for all): sequence b's queries are its first counts[b], like the new tokens of kv8_append with the same counts, and query
    i of a causal call is its token lens[b] - counts[b] + i; the rows behind them give zeros.  Without it the queries of every sequence end with its newest token.  out must not overlap the inputs."""
    name = 'kv8_attention'
    device = _device(name, q, k_cache, v_cache, k_scale, v_scale, lens, out, counts)
    n, kv_heads, capacity, d, cs = _cache(name, k_cache, v_cache, k_scale, v_scale)
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise ValueError('%s: q must be float32, bfloat16 or float16' % name)
    if q.dim() != 4:
        raise ValueError('%s: q must be [n, tq, heads, d]' % name)
    _, tq, heads, _ = q.shape
    qs = _rows(name, 'q', q, (n, tq, heads, d))
    _counts(name, 'lens', lens, n)
    if counts is not None:
        _counts(name, 'counts', counts, n)
    given = out is not None
    out = _output(name, q, out)
    size = _kv8_workspace(n, tq, capacity, heads, kv_heads, d, dtype)
    ws = q.new_empty((size,), dtype=torch.uint8) if size else None
    _call(lib.asr_kv8_attention_counts,
          _ATTEND.pack(q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                       lens.data_ptr(), 0 if ws is None else ws.data_ptr(), *qs, *out.stride()[:3], cs[0], cs[1], size, n, tq, heads, kv_heads,
                       d, capacity, dtype, 1 if causal else 0, (d or 1) ** -0.5 if scale is None else scale), device, 0 if counts is None else counts.data_ptr())
    if given:
        _changed((out,))
    return out
