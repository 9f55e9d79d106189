"""asr_amd.ops without a GPU: what is refused before anything is queued, and the reference the GPU tests compare with."""
import math

import pytest
import torch

from tests import ops_reference as R


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


@pytest.fixture(scope='module')
def lib():
    from asr_amd import _lib
    return _lib.lib


def test_tensors_outside_gpu_memory_are_refused(ops):
    q = torch.zeros(1, 1, 2, 64)
    k8, v8, ks, vs = ops.kv8_cache(1, 2, 64, 64, device='cpu')
    lens = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32)), lambda: ops.cross_attention(q, q, q),
                 lambda: ops.kv8_append(q, q, k8, v8, ks, vs, lens), lambda: ops.kv8_attention(q, k8, v8, ks, vs, lens)):
        with pytest.raises(ValueError, match='GPU memory'):
            call()


def test_cache_shapes(ops):
    k8, v8, ks, vs = ops.kv8_cache(3, 2, 192, 80, device='cpu')
    assert k8.shape == v8.shape == (3, 2, 192, 80) and k8.dtype == torch.float8_e4m3fn and ks.shape == vs.shape == (3, 2, 3)
    assert ops.KV8_BLOCK == R.BLOCK == 64
    with pytest.raises(ValueError):
        ops.kv8_cache(1, 1, 65, 64, device='cpu')


# argument structs by field, as asr_amd/ops.py packs them; no pointer is ever followed by a refused call
def _logprobs(ops, **kw):
    a = dict(logits=256, tokens=256, logprob=256, entropy=256, tops=256, top_tokens=256, rows=2, row_stride=8, vocab=8, top=2, dtype=0, token_bytes=4)
    a.update(kw)
    return ops._LOGPROBS.pack(*a.values())


def _cross(ops, **kw):
    a = dict(q=256, k=256, v=256, out=256, lens=0, pad=0, ws=0, qs=(128, 128, 64), ks=(128, 128, 64), vs=(128, 128, 64), os=(128, 128, 64),
             pad_stride=0, ws_bytes=0, n=1, tq=1, tk=4, heads=2, kv_heads=2, d=64, dtype=1, scale=0.125)
    a.update(kw)
    flat = []
    for x in a.values():
        flat.extend(x if isinstance(x, tuple) else (x,))
    return ops._CROSS.pack(*flat)


def _append(ops, **kw):
    a = dict(k=256, v=256, k8=256, v8=256, ks=256, vs=256, lens=256, counts=0, kst=(64, 64, 64), vst=(64, 64, 64), cs=(4096, 4096), n=1, new=1,
             kv_heads=1, d=64, capacity=64, dtype=0)
    a.update(kw)
    flat = []
    for x in a.values():
        flat.extend(x if isinstance(x, tuple) else (x,))
    return ops._APPEND.pack(*flat)


def _attend(ops, **kw):
    a = dict(q=256, out=256, k8=256, v8=256, ks=256, vs=256, lens=256, ws=0, qs=(64, 64, 64), os=(64, 64, 64), cs=(4096, 4096), ws_bytes=0, n=1,
             tq=1, heads=1, kv_heads=1, d=64, capacity=64, dtype=0, causal=0, scale=0.125)
    a.update(kw)
    flat = []
    for x in a.values():
        flat.extend(x if isinstance(x, tuple) else (x,))
    return ops._ATTEND.pack(*flat)


REFUSED = [
    ('asr_token_logprobs', _logprobs, dict(rows=-1)), ('asr_token_logprobs', _logprobs, dict(vocab=0)),
    ('asr_token_logprobs', _logprobs, dict(vocab=(1 << 30) + 1)), ('asr_token_logprobs', _logprobs, dict(top=33, vocab=100)),
    ('asr_token_logprobs', _logprobs, dict(top=9)), ('asr_token_logprobs', _logprobs, dict(top=-1)),
    ('asr_token_logprobs', _logprobs, dict(dtype=3)), ('asr_token_logprobs', _logprobs, dict(token_bytes=2)),
    ('asr_token_logprobs', _logprobs, dict(logits=0)), ('asr_token_logprobs', _logprobs, dict(tops=0)),
    ('asr_token_logprobs', _logprobs, dict(logits=258)), ('asr_token_logprobs', _logprobs, dict(row_stride=-8)),
    ('asr_cross_attention', _cross, dict(n=-1)), ('asr_cross_attention', _cross, dict(tk=-1)), ('asr_cross_attention', _cross, dict(kv_heads=0)),
    ('asr_cross_attention', _cross, dict(heads=3)), ('asr_cross_attention', _cross, dict(d=136)), ('asr_cross_attention', _cross, dict(d=0)),
    ('asr_cross_attention', _cross, dict(d=60)), ('asr_cross_attention', _cross, dict(dtype=7)), ('asr_cross_attention', _cross, dict(scale=math.nan)),
    ('asr_cross_attention', _cross, dict(scale=math.inf)), ('asr_cross_attention', _cross, dict(q=0)), ('asr_cross_attention', _cross, dict(k=0)),
    ('asr_cross_attention', _cross, dict(q=264)), ('asr_cross_attention', _cross, dict(ks=(128, 124, 64))),
    ('asr_cross_attention', _cross, dict(vs=(128, -128, 64))), ('asr_cross_attention', _cross, dict(os=(128, 128, 60))),
    ('asr_cross_attention', _cross, dict(tq=1 << 30)), ('asr_cross_attention', _cross, dict(n=1 << 23)),
    ('asr_cross_attention', _cross, dict(tk=100000)),                                          # needs a workspace
    ('asr_kv8_append', _append, dict(n=-1)), ('asr_kv8_append', _append, dict(d=24)), ('asr_kv8_append', _append, dict(d=144)),
    ('asr_kv8_append', _append, dict(capacity=65)), ('asr_kv8_append', _append, dict(dtype=3)), ('asr_kv8_append', _append, dict(lens=0)),
    ('asr_kv8_append', _append, dict(k=260)), ('asr_kv8_append', _append, dict(new=2, kst=(64, 62, 64))), ('asr_kv8_append', _append, dict(k8=264)),
    ('asr_kv8_append', _append, dict(cs=(4100, 4096))), ('asr_kv8_append', _append, dict(n=70000, v8=1024, vs=512)),
    ('asr_kv8_append', _append, dict(vs=512)), ('asr_kv8_append', _append, dict(v8=1024)),          # K and V in the same memory
    ('asr_kv8_append', _append, dict(v8=1024, vs=512, capacity=1 << 23, new=1 << 23)),
    ('asr_kv8_attention', _attend, dict(capacity=65)), ('asr_kv8_attention', _attend, dict(heads=3, kv_heads=2)),
    ('asr_kv8_attention', _attend, dict(d=72)), ('asr_kv8_attention', _attend, dict(dtype=3)), ('asr_kv8_attention', _attend, dict(scale=math.inf)),
    ('asr_kv8_attention', _attend, dict(lens=0)), ('asr_kv8_attention', _attend, dict(v8=0)), ('asr_kv8_attention', _attend, dict(q=260)),
    ('asr_kv8_attention', _attend, dict(cs=(4096, 4104))), ('asr_kv8_attention', _attend, dict(capacity=64000)),
]


@pytest.mark.parametrize('entry,pack,change', REFUSED, ids=['%s-%s' % (e[4:], '-'.join('%s=%s' % kv for kv in c.items())) for e, _, c in REFUSED])
def test_the_library_refuses(ops, lib, entry, pack, change):
    """Bad sizes, types, strides, alignments and workspaces end in a status and a message, on the host, before anything is queued."""
    rc = getattr(lib, entry)(pack(ops, **change), None)
    assert rc in (1, 5)                                       # ASR_ERR_ARG, ASR_ERR_CAPACITY
    assert entry[4:] in lib.asr_ops_last_error().decode()


@pytest.mark.parametrize('entry', ['asr_token_logprobs', 'asr_cross_attention', 'asr_kv8_append', 'asr_kv8_attention'])
def test_null_arguments_are_refused(lib, entry):
    assert getattr(lib, entry)(None, None) == 1


def test_nothing_to_do_is_no_error(ops, lib):
    assert lib.asr_token_logprobs(_logprobs(ops, rows=0, logits=0), None) == 0
    assert lib.asr_cross_attention(_cross(ops, n=0, q=0), None) == 0
    assert lib.asr_cross_attention(_cross(ops, tq=0), None) == 0
    assert lib.asr_kv8_append(_append(ops, new=0, k=0), None) == 0
    assert lib.asr_kv8_attention(_attend(ops, tq=0), None) == 0


def test_workspace_sizes(lib):
    assert lib.asr_cross_attention_workspace(64, 10, 334, 16, 16, 64, 1) == 0
    assert lib.asr_cross_attention_workspace(1, 1, 100000, 1, 1, 64, 1) > 0
    assert lib.asr_cross_attention_workspace(1, 1, 100000, 3, 2, 64, 1) == 0                    # sizes that are refused anyway
    assert lib.asr_kv8_attention_workspace(1, 1, 65536, 8, 1, 128, 0) > 0


# ---- the reference itself ------------------------------------------------------------------------------------------------
def test_reference_codes_are_the_e4m3_ones():
    every = torch.arange(256, dtype=torch.uint8)
    assert torch.equal(torch.nan_to_num(R.CODES.float(), nan=-7.0), torch.nan_to_num(every.view(torch.float8_e4m3fn).float(), nan=-7.0))
    x = torch.randn(20000, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).float().double() * 100
    assert torch.equal(R.to_code(x.clamp(-448, 448)).float(), x.clamp(-448, 448).float().to(torch.float8_e4m3fn).float())
    halves = (R.CODES[:126] + R.CODES[1:127]) / 2
    assert torch.equal(R.to_code(halves).float(), halves.float().to(torch.float8_e4m3fn).float())


def test_reference_exponent():
    for top, e in ((448.0, 0), (449.0, 1), (224.0, -1), (1.75, -8), (1.7500001, -7), (0.0, -100), (2.0 ** -140, -100)):
        assert R.exponent(torch.tensor([top, -top / 3], dtype=torch.float64)) == e


def test_reference_attention_is_softmax():
    g = torch.Generator().manual_seed(2)
    q, k = torch.randn(2, 3, 4, 16, generator=g), torch.randn(2, 2, 9, 16, generator=g).double()
    v = torch.randn(2, 2, 9, 16, generator=g).double()
    out, _, _ = R.attention(q, k, v, torch.ones(2, 3, 9, dtype=torch.bool), 0.25)
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(1, 2), k.repeat_interleave(2, 1), v.repeat_interleave(2, 1), scale=0.25)
    assert torch.allclose(out, want.transpose(1, 2), atol=1e-12)
