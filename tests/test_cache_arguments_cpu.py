"""Arguments of the paged cache and its operators that are refused before anything changes: no GPU needed."""
import ctypes as C

import pytest
import torch

from _cache_ref import plain_copy_pages


def make_cache(**kw):
    from zentorch_b200.cache import PagedKVCache
    return PagedKVCache(**{**dict(layers=1, pages=6, page_size=4, kv_heads=1, head_dim=8, device="cpu", copy_pages=plain_copy_pages,
                                  dtype=torch.float32), **kw})


@pytest.mark.parametrize("count", [1.5, "1", None])
def test_a_step_takes_whole_numbers_of_tokens(zt, count):
    """... and a batch with another one leaves every sequence as it was."""
    cache = make_cache()
    cache.add("a")
    cache.add("b")
    cache.step([("a", 3)])
    with pytest.raises(TypeError):
        cache.step([("a", 2), ("b", count)])
    with pytest.raises(TypeError):
        cache.truncate("a", 1.5)
    assert cache.length("a") == 3 and cache.pages("a") == (0,) and cache.length("b") == 0 and cache.free_pages == 5
    assert cache.step([("a", torch.tensor(2).item()), ("b", torch.tensor(1))]).cu_seqlens_q.tolist() == [0, 2, 3]


def test_a_copy_that_fails_leaves_the_cache_as_it_was(zt):
    def fails(caches, src, dst):
        raise RuntimeError("no copy")
    cache = make_cache(copy_pages=fails)
    cache.add("a")
    cache.step([("a", 6)])
    cache.fork("a", "b")
    with pytest.raises(RuntimeError, match="no copy"):
        cache.step([("a", 4), ("b", 1)])
    assert cache.pages("a") == cache.pages("b") == (0, 1) and cache.length("a") == cache.length("b") == 6 and cache.free_pages == 4
    cache.free("b")
    assert cache.free_pages == 4
    cache.free("a")
    assert cache.free_pages == 6
    for name in "abc":
        cache.add(name)
        cache.step([(name, 4)])
    cache.free("a")
    with pytest.raises(RuntimeError, match="no copy"):
        cache.compact()
    assert cache.pages("b") == (1,) and cache.pages("c") == (2,) and cache.free_pages == 4


@pytest.mark.parametrize("head_dim", [4, 68, 136, 256])
def test_a_decoder_layer_takes_heads_that_its_attention_reads(zt, head_dim):
    """The cache would be filled before the attention refused it."""
    from zentorch_b200 import tp

    class Lin:
        world = 1
    with pytest.raises(ValueError, match="multiple of 8 elements up to 128"):
        tp.DecoderLayer(Lin(), 8, 2, head_dim, torch.ones(2))
    assert tp.DecoderLayer(Lin(), 8, 2, head_dim, torch.ones(2), ops=object()).head_dim == head_dim      # another attention
    assert tp.DecoderLayer(Lin(), 8, 2, 80, torch.ones(2)).head_dim == 80


def test_a_softmax_scale_whose_base_two_form_is_infinite(zt):
    from zentorch_b200 import _capi
    lib, p = _capi.lib(), _capi.PagedAttentionArgs()
    p.tokens, p.batch, p.q_heads, p.kv_heads, p.head_dim, p.dtype, p.cache_dtype = 4, 2, 8, 4, 64, _capi.ZT_BF16, _capi.ZT_BF16
    p.page_size, p.max_blocks, p.num_pages = 16, 4, 8
    for scale, text in ((3e38, b"positive and finite"), (2e38, b"null tensor pointer")):
        p.scale = scale
        assert lib.zt_paged_attention(C.byref(p), None) == 1 and text in lib.zt_last_error()
