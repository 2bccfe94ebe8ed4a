"""Caches whose byte and element offsets do not fit 32 bits: the far pages hold what the near ones do not."""
import pytest
import torch

from _cache_ref import assert_attention, attention_ref, make_batch
from test_paged_attention_gpu import BF16, E4M3, capi, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [64, 63])                # whole boxes of a page; pages that are copied row by row
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_attention_over_far_pages(capi, cache, page):  # noqa: F811
    hkv, d = 8, 64
    pages = 2 ** 32 // (page * hkv * d) + 4000            # 2^32 elements and more
    c = make_batch([(1, 300), (40, 200)], 16, hkv, d, page, BF16, cache, seed=49)
    far = {}
    for name in ("k_cache", "v_cache"):
        near, raw = c[name].view(torch.uint8) if cache == E4M3 else c[name], torch.uint8 if cache == E4M3 else BF16
        far[name] = torch.zeros(pages, page, hkv, d, dtype=raw, device="cuda")
        far[name][pages - near.shape[0]:] = near
        far[name] = far[name].view(cache)
    moved = dict(c, **far, table=torch.where(c["table"] < 2 ** 20, c["table"] + pages - c["k_cache"].shape[0], c["table"]))
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], k_scale=c["k_scale"],
                               v_scale=c["v_scale"])
    for algo in ("dealt", "rows8", "rows16", "slices1", "slices8", "tcgen05"):
        got = run(capi, moved, algo)
        assert_attention(got, ref, bound, algo)
        assert torch.equal(got, run(capi, c, algo)), algo
