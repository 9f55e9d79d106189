"""Outputs in the memory of keys, values or caches are refused; halves of one allocation that lie between each other are not the same memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


@pytest.mark.parametrize('tq', [9, 100])
def test_out_in_the_memory_of_keys_or_values_is_refused(ops, tq):
    q, k, v = (torch.randn(2, tq, 4, 64, device='cuda').bfloat16() for _ in range(3))
    kept = [x.clone() for x in (q, k, v)]
    for out in (k, v, k.view(2, tq, 4, 64)):
        with pytest.raises(ValueError, match='overlap'):
            ops.cross_attention(q, k, v, out=out)
    assert all(torch.equal(a, b) for a, b in zip((q, k, v), kept))
    want = ops.cross_attention(q, k, v)
    three = torch.stack([q, k, v], 2)                                # [n, tq, 3, heads, d]: q, k and v between each other
    wide = torch.cat([three, torch.zeros_like(three[:, :, :1])], 2)
    got = ops.cross_attention(wide[:, :, 0], wide[:, :, 1], wide[:, :, 2], out=wide[:, :, 3])
    assert torch.equal(got, want)
    for i in range(3):
        assert torch.equal(wide[:, :, i], three[:, :, i])
