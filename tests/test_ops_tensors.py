"""Tensors that asr_amd.ops cannot take although they say that they are on a GPU: refused, not computed as something else."""
import pytest
import torch
from torch._subclasses import FakeTensorMode
from torch.autograd import forward_ad


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


def _arguments(device):
    q, k = torch.ones(2, 3, 4, 64, device=device), torch.ones(2, 9, 4, 64, device=device)
    lens = torch.ones(2, dtype=torch.int32, device=device)
    code = torch.zeros(2, 4, 64, 64, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    scale = torch.ones(2, 4, 1, device=device)
    return q, k, lens, (code, code.clone(), scale, scale.clone())


def _calls(ops, q, k, lens, cache):
    return {'token_logprobs': lambda: ops.token_logprobs(q[0, 0], torch.arange(4, device=q.device), top=2),
            'cross_attention': lambda: ops.cross_attention(q, k, k, lens=lens), 'kv8_attention': lambda: ops.kv8_attention(q, *cache, lens),
            'kv8_append': lambda: ops.kv8_append(k, k, *cache, lens)}


OPERATORS = ['token_logprobs', 'cross_attention', 'kv8_attention', 'kv8_append']


@pytest.mark.parametrize('name', OPERATORS)
def test_fake_tensors_are_refused(ops, name):
    with FakeTensorMode():
        call = _calls(ops, *_arguments('cuda'))[name]
        with pytest.raises(ValueError, match='memory of their own'):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize('name', OPERATORS)
def test_tensors_with_a_tangent_are_refused(ops, name):
    q, k, lens, cache = _arguments('cuda')
    with forward_ad.dual_level():
        for a, b in ((forward_ad.make_dual(q, q.clone()), k), (q, forward_ad.make_dual(k, k.clone()))):
            call = _calls(ops, a, b, lens, cache)[name]
            if name == 'cross_attention' or (name == 'kv8_append') == (b is not k):
                with pytest.raises(ValueError, match='forward-mode'):
                    call()
                with torch.no_grad(), pytest.raises(ValueError, match='forward-mode'):
                    call()
                with torch.inference_mode():
                    call()                                       # (no derivatives are followed there)
            else:
                call()                                           # (the dual tensor is not one of its arguments)
        _calls(ops, q, k, lens, cache)[name]()
    _calls(ops, torch.nn.Parameter(q, requires_grad=False), k, lens, cache)[name]()
