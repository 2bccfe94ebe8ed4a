"""A key that outweighs thousands of others by far and has no value of its own (an attention sink): the output is what the
others add up to, so their small probabilities must survive products in fp16."""
import pytest
import torch

from _cache_ref import assert_attention, attention_ref, make_batch
from test_paged_attention_gpu import ALGOS, BF16, E4M3, F16, capi, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("gap", [14.0, 20.4, 22.7, 25.2])      # log2 of the sink's weight over that of another key
@pytest.mark.parametrize("at", [0, 4000])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (F16, E4M3), (BF16, E4M3)])
def test_a_sink_among_equal_keys(capi, algo, gap, at, dtype, cache):  # noqa: F811
    """Beside the bound of every test: a probability below fp16's normal numbers is off by half the spacing of its subnormals,
    2^-25; the products take probabilities times 2^7 relative to the row's largest, so that is 2^-32 of the output's sum per
    key and unit of its value."""
    kv = 8192
    c = make_batch([(1, kv), (3, kv - 90)], 4, 2, 64, 64, dtype, cache, seed=45)
    c["q"].zero_()
    c["q"][..., 0] = 1
    raw_k, raw_v = torch.zeros(c["k_cache"].shape), torch.ones(c["v_cache"].shape)
    raw_v += torch.randint(0, 2, raw_v.shape, generator=torch.Generator().manual_seed(1)) * 0.25
    for b in (0, 1):
        page = int(c["table"][b, at // 64])
        raw_k[page, at % 64, :, 0] = 16
        raw_v[page, at % 64] = 0
    c["k_cache"], c["v_cache"] = raw_k.to(cache).cuda(), raw_v.to(cache).cuda()
    if cache == E4M3:
        c["k_scale"].fill_(1.0), c["v_scale"].fill_(1.0)
    scale = gap * 0.6931471805599453 / 16
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], scale=scale, k_scale=c["k_scale"],
                               v_scale=c["v_scale"])
    got = run(capi, c, algo, scale=scale)
    assert_attention(got, ref, bound + kv * 1.25 * 2.0 ** -32, f"gap {gap}")


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scores_beyond_the_precision_of_their_reference(capi, algo, dtype):  # noqa: F811
    """Scores of up to 2^27.6, 16 apart in fp32: the exponent's reference is that far from a score at most, which must neither overflow
    a probability nor lose it.  Each row is the value of its largest key, ahead of every other by far more than that."""
    kv, n = 300, 40
    c = make_batch([(n, kv)], 4, 2, 64, 16, dtype, seed=46)
    c["q"].zero_()
    c["q"][..., 0] = 30000
    rank = torch.randperm(kv, generator=torch.Generator().manual_seed(2)).float()
    for page, ids in enumerate(rank.split(16)):
        c["k_cache"][c["table"][0, page].long(), :len(ids)] = 0
        c["k_cache"][c["table"][0, page].long(), :len(ids), :, 0] = ((ids + 1) * 128).to(dtype).cuda()[:, None]
    got = run(capi, c, algo, scale=0.125).float().cpu()
    k = ((rank + 1) * 128).to(dtype).float()
    pages = c["table"][0, :19].long()
    v = c["v_cache"][pages].flatten(0, 1)[:kv].float().cpu()
    for i in range(n):
        seen = k[:kv - n + i + 1]
        best = seen == seen.max()                        # (in bf16 some keys are equal)
        want = v[:kv - n + i + 1][best].mean(0).repeat_interleave(2, 0)
        tol = 2.0 ** -8 if dtype == BF16 else 2.0 ** -11
        assert bool(((got[i] - want).abs() <= 3 * tol * v.abs().max()).all()), i
