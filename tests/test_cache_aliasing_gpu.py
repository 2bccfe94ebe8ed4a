"""Tensors that share memory with what a call writes."""
import pytest
import torch

from _cache_ref import make_batch
from test_rope_cache_gpu import BF16, E4M3, caches, freq, ops, qkv  # noqa: F401

pytestmark = pytest.mark.gpu


def test_caches_that_share_memory_are_refused(ops):  # noqa: F811
    q, k, v = qkv(3, 2, 1, 64, BF16)
    pos, f, slots = torch.arange(3).cuda(), freq(64), torch.arange(3).cuda()

    def refused(match, *args):
        with pytest.raises(RuntimeError, match=match):
            ops.zentorch_rope_cache(*args, slots)

    both = torch.zeros(8, 2, 4, 1, 64, dtype=BF16, device="cuda")           # keys and values of a page side by side
    plain = torch.zeros(8, 4, 1, 64, dtype=BF16, device="cuda")
    ops.zentorch_rope_cache(q, k, v, pos, f, both[:, 0], both[:, 1], slots)
    refused("share memory with value_cache", q, k, v, pos, f, plain[:6], plain[2:])
    refused("share memory with value_cache", q, k, v, pos, f, both[:6, 0], both[2:, 0])
    refused("share memory with value_cache", q, k, v, pos, f, both[:6, 1], both[2:, 1])
    flat = both.view(16, 4, 1, 64)                                          # pages 2i are keys, 2i + 1 values
    refused("share memory with value_cache", q, k, v, pos, f, flat[2:10:2], flat[:8:2])
    ops.zentorch_rope_cache(q, k, v, pos, f, flat[2:10:2], flat[1:9:2], slots)
    refused("share memory with query", plain.view(32, 1, 64)[:3], k, v, pos, f, plain, both[:, 1])
    refused("share memory with key", q, plain.view(32, 1, 64)[4:7], v, pos, f, plain, both[:, 1])
    refused("share memory with value", q, k, plain.view(32, 1, 64)[29:], pos, f, both[:, 0], plain)


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_one_tensor_as_both_caches_holds_the_values(ops, cache):  # noqa: F811
    """Keys and values of a token go to one row then: it is the values that remain, in every run."""
    q, k, v = qkv(2000, 2, 4, 64, BF16)
    pos, f, slots = torch.arange(2000).cuda() + 5, freq(64), torch.randperm(2000).cuda()
    scales = (torch.ones(4, device="cuda"),) * 2 if cache == E4M3 else (None, None)
    for layout in ("plain", "joined"):
        c, _ = caches(125, 16, 4, 64, cache, layout)
        ops.zentorch_rope_cache(q, k, v, pos, f, c, c, slots, *scales)
        assert torch.equal(c.float().reshape(2000, 4, 64)[slots], v.to(cache).float())


def test_outputs_that_share_memory_are_refused(ops):  # noqa: F811
    c = make_batch([(5, 30)], 4, 2, 64, 16, BF16, seed=48)
    wide = torch.zeros(5, 6 * 64, dtype=BF16, device="cuda")                # rows of a fused projection
    q, tail = wide[:, :4 * 64].view(5, 4, 64), wide[:, 4 * 64:].view(5, 2, 64)
    into, args = ops.zentorch_paged_attention.out, (c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"])
    for other in (wide[:, :4 * 64].view(5, 4, 64), wide[:, 2 * 64:].view(5, 4, 64)):
        with pytest.raises(RuntimeError, match="share memory with query"):
            into(other, q, *args)
    into(tail, wide[:, :2 * 64].view(5, 2, 64), *args)                      # beside each other: fine
