"""Where the tensors of a step are made."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_cache_stays_on_the_device_that_it_was_made_on(zt):
    """The current device may be another one when a step is taken: its tensors go where the pages are."""
    from zentorch_b200.cache import PagedKVCache
    cache = PagedKVCache(1, 4, 16, 1, 64, device="cuda")
    assert cache.device == cache.keys(0).device and cache.device.index == torch.cuda.current_device()
    cache.add("a")
    step = cache.step([("a", 3)])
    for t in (step.positions, step.slots, step.cu_seqlens_q, step.seq_lens, step.block_table):
        assert t.device == cache.device
