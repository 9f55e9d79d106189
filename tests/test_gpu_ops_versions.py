"""What the operators write in place counts as changed for autograd, as with torch's own in-place operators."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from asr_amd import ops as module
    return module


def _cache(ops):
    lens = torch.tensor([1, 2], dtype=torch.int32, device='cuda')
    return ops.kv8_cache(2, 2, 64, 64), torch.ones(2, 1, 2, 64, device='cuda'), lens


def test_a_saved_output_buffer_that_is_written_again_is_noticed(ops):
    cache, k, lens = _cache(ops)
    q = torch.randn(2, 3, 2, 64, device='cuda')
    calls = (lambda out: ops.cross_attention(q, q, q, out=out), lambda out: ops.kv8_attention(q, *cache, lens, out=out))
    for call in calls:
        out = torch.zeros(2, 3, 2, 64, device='cuda')
        w = torch.ones_like(out, requires_grad=True)
        loss = (w * call(out)).sum()                             # (saves out for the gradient of w)
        call(out)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            loss.backward()
        fresh = call(None)
        assert fresh._version == 0


def test_a_saved_cache_that_grows_is_noticed(ops):
    cache, k, lens = _cache(ops)
    for i in (2, 3):
        w = torch.ones_like(cache[i], requires_grad=True)
        loss = (w * cache[i]).sum()
        ops.kv8_append(k, k, *cache, lens)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            loss.backward()
    before = [t._version for t in cache]
    ops.kv8_append(k, k, *cache, lens)
    assert all(t._version > v for t, v in zip(cache, before))
    with torch.inference_mode():
        mine = ops.kv8_cache(2, 2, 64, 64)
        ops.kv8_append(k, k, *mine, lens)                        # (inference tensors have no version)
        ops.cross_attention(k, k, k, out=torch.empty_like(k))
