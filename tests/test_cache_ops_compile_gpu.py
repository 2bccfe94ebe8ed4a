"""The operators between the linears under torch.compile and under torch's own checks of a custom operator."""
import pytest
import torch

from _cache_ref import make_batch
from test_rope_cache_gpu import BF16, E4M3, freq, ops, qkv  # noqa: F401

pytestmark = pytest.mark.gpu
CHECKS = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")


def pair(pages, page, hkv, d, dtype=BF16):
    both = torch.zeros(pages, 2, page, hkv, d, device="cuda").to(dtype)
    return both[:, 0], both[:, 1]


def test_torchs_own_checks(ops):  # noqa: F811
    q, k, v = qkv(5, 4, 2, 64, BF16)
    pos, f, slots = torch.arange(5).cuda(), freq(64), torch.arange(5).cuda()
    one = torch.ones(2, device="cuda")
    torch.library.opcheck(ops.zentorch_rope.default, (q, k, pos, f), dict(interleaved=True), test_utils=CHECKS)
    torch.library.opcheck(ops.zentorch_rope_cache.default, (q, k, v, pos, f, *pair(3, 4, 2, 64), slots), test_utils=CHECKS)
    torch.library.opcheck(ops.zentorch_rope_cache.default, (q, k, v, pos, f, *(torch.zeros(3, 4, 2, 64, device="cuda").to(E4M3) for _ in range(2)),
                                                            slots, one, one), test_utils=("test_faketensor",))
    caches = [torch.randn(4, 8, 16, device="cuda") for _ in range(3)]
    torch.library.opcheck(ops.zentorch_cache_copy_pages.default, (caches, slots[:2], slots[2:4]), test_utils=CHECKS)
    c = make_batch([(1, 30), (4, 40)], 4, 2, 64, 16, BF16, seed=50, table_fill=0)
    c["k_cache"], c["v_cache"] = c["k_cache"].nan_to_num(), c["v_cache"].nan_to_num()
    args = (c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], 4)
    torch.library.opcheck(ops.zentorch_paged_attention.default, args, dict(window=7), test_utils=CHECKS)
    torch.library.opcheck(ops.zentorch_paged_attention.out, (torch.zeros(5, 4, 64, dtype=BF16, device="cuda"), *args), test_utils=CHECKS)


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_a_compiled_step_writes_what_an_eager_one_does(ops, backend):  # noqa: F811
    """Rotary positions into the cache, a page copy, attention over both, compiled as one graph: the caches and the outputs of
    the eager calls, bit for bit, call after call."""
    f, pos = freq(64), torch.arange(6).cuda()
    src, dst = torch.tensor([0]).cuda(), torch.tensor([2]).cuda()
    cu, lens = torch.tensor([0, 6], dtype=torch.int32).cuda(), torch.tensor([6], dtype=torch.int32).cuda()
    table = torch.tensor([[2, 1]], dtype=torch.int32).cuda()

    def step(q, k, v, both, slots, out):
        kc, vc = both[:, 0], both[:, 1]
        q = ops.zentorch_rope_cache(q, k, v, pos, f, kc, vc, slots)
        ops.zentorch_cache_copy_pages([both], src, dst)
        y = ops.zentorch_paged_attention(q, kc, vc, cu, lens, table, 6)
        ops.zentorch_paged_attention.out(out, q, kc, vc, cu, lens, table, 6, window=3)
        a, b = ops.zentorch_rope(y, k, pos, f)
        return y * 2, a, b

    torch._dynamo.reset()
    compiled = torch.compile(step, backend=backend, fullgraph=True)
    state = [[torch.zeros(3, 2, 4, 2, 64, dtype=BF16, device="cuda"), torch.zeros(6, 4, 64, dtype=BF16, device="cuda")] for _ in range(2)]
    slots = torch.arange(6).cuda()
    for i in range(3):
        x = qkv(6, 4, 2, 64, BF16, seed=i)
        want, got = (fn(*x, s[0], slots, s[1]) for fn, s in ((step, state[0]), (compiled, state[1])))
        for a, b in zip([*want, *state[0]], [*got, *state[1]]):
            assert torch.equal(a, b)
