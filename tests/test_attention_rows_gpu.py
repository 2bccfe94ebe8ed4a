"""Rows of the output that belong to no sequence."""
import pytest
import torch

from _cache_ref import assert_attention, attention_ref, make_batch
from test_paged_attention_gpu import ALGOS, BF16, capi, run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("algo", ALGOS)
def test_rows_before_the_first_sequence(capi, algo):  # noqa: F811
    """Prefix sums that start above zero (a part of a larger batch's): zeros in a new output, left as they were in the caller's."""
    c = make_batch([(7, 7), (2, 30), (3, 50)], 4, 2, 64, 16, BF16, seed=47, tail=6)
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"])
    c.update(cu=c["cu"][1:].clone(), lens=c["lens"][1:].clone(), table=c["table"][1:].clone())
    held = [torch.full_like(c["q"], 7.0) for _ in range(4)]
    torch.cuda.synchronize()
    del held                                             # (memory that a new output of this size is made of)
    got = run(capi, c, algo)
    assert_attention(got[7:12], ref[7:12], bound[7:12])
    assert (got[:7] == 0).all() and (got[12:] == 0).all()
    mine = torch.full_like(got, 7.0)
    torch.ops.zentorch.zentorch_paged_attention.out(mine, c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], 3)
    assert_attention(mine[7:12], ref[7:12], bound[7:12])
    assert (mine[:7] == 7).all() and (mine[12:] == 7).all()
