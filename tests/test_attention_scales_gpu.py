"""Softmax and cache scales at their ends: NaN, zero, and far below one."""
import pytest
import torch

from _cache_ref import assert_attention, attention_ref, make_batch
from test_paged_attention_gpu import ALGOS, BF16, E4M3, F16, capi, check, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_a_scale_of_nan_stays_nan(capi, algo, which):  # noqa: F811
    c = make_batch([(40, 70), (1, 90), (3, 2), (2, 0)], 4, 2, 64, 16, BF16, E4M3, seed=42)      # rows 41, 44 and 45 see nothing
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], k_scale=c["k_scale"],
                               v_scale=c["v_scale"])
    c[which][1] = float("nan")
    got = run(capi, c, algo)
    none = torch.tensor([41, 44, 45])
    seen = torch.tensor([i for i in range(46) if i not in none.tolist()])
    assert got[seen, 2:].isnan().all() and (got[none] == 0).all()
    assert_attention(got[:, :2], ref[:, :2], bound[:, :2])


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_key_scale_of_zero_is_a_mean(capi, algo, dtype):  # noqa: F811
    c = make_batch([(40, 70), (1, 90), (3, 2)], 4, 2, 64, 16, dtype, E4M3, seed=43)
    c["k_scale"][0] = 0.0
    check(capi, c, algo, window=50)


@pytest.mark.parametrize("algo", ALGOS)
def test_a_small_softmax_scale_over_large_elements(capi, algo):  # noqa: F811
    """Scores of ordinary size from products of 2^110 or so: the scale counts as it is."""
    c = make_batch([(40, 70), (1, 90)], 4, 2, 64, 16, BF16, seed=44)
    c["q"].mul_(2.0 ** 55)
    c["k_cache"].mul_(2.0 ** 55)
    check(capi, c, algo, scale=2.0 ** -113, window=50)
