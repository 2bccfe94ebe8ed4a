"""Values that are not finite in the paged attention, one pair to a column: what a row gets follows from the values that it sees."""
import pytest
import torch

from _cache_ref import attention_ref, make_batch
from test_paged_attention_gpu import ALGOS, BF16, F16, capi, run  # noqa: F401  (capi is a fixture)

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def check_special(got, ref, bound):
    """Equal where the definition gives NaN or an infinity, within the bound elsewhere."""
    got, fine = got.double().cpu(), torch.isfinite(ref)
    assert torch.equal(got.isnan(), ref.isnan())
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf])
    assert bool(((got - ref).abs()[fine] <= bound[fine]).all())


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("early,late", [(INF, NAN), (-INF, NAN), (INF, -INF), (-INF, INF), (INF, INF), (NAN, INF)])
@pytest.mark.parametrize("n,kv,window", [(100, 300, 0), (100, 300, 60), (300, 300, 0)])
def test_two_values_in_one_column(capi, algo, dtype, early, late, n, kv, window):  # noqa: F811
    """Rows that see the first of two keys of a tile and not the second have the first one's value in that column, whatever the
    second one holds; nothing else in those rows is special."""
    c = make_batch([(n, kv), (1, 20)], 4, 2, 64, 16, dtype, seed=41)
    for key, value in ((kv - 60, early), (kv - 20, late)):
        c["v_cache"][c["table"][0, key // 16].long(), key % 16, 1, 17] = value
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], window=window)
    assert not torch.isfinite(ref).all()
    check_special(run(capi, c, algo, window=window), ref, bound)
