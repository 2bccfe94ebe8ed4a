"""zentorch_paged_attention against a 64-bit evaluation: every kernel, at the sizes, masks, layouts and types where it can go
wrong.  Bounds are derived in _cache_ref.attention_ref."""
import pytest
import torch

from _cache_ref import assert_attention, attention_ref, make_batch

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
ROWS = {"rows8": 8, "rows16": 16}                  # the streaming kernel for so many rows per kv head; "dealt": 32 in most tests
ALGOS = ["dealt", *ROWS, "slices1", "slices3", "slices8", "tcgen05"]


@pytest.fixture(scope="module")
def capi(zt):
    from zentorch_b200 import _capi
    assert torch.cuda.is_available() and _capi.lib().zt_device_supported() == 1
    return _capi


def run(capi, c, algo=None, **kw):
    scales = dict(k_scale=c["k_scale"], v_scale=c["v_scale"])
    if algo is None:
        return torch.ops.zentorch.zentorch_paged_attention(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"],
                                                           c["max_q"], **scales, **kw)
    if algo == "tcgen05":
        code = capi.ZT_ALGO_TCGEN05
    else:
        code = capi.ZT_ALGO_SKINNY | (1 if algo in ROWS or algo == "dealt" else 1 + int(algo[6:])) << 8
    max_q = c["max_q"]
    if algo in ROWS:      # (it need not be exact)
        max_q = max(1, ROWS[algo] * c["k_cache"].shape[2] // c["q"].shape[1])
    return capi.paged_attention(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], max_q, algo=code, **scales, **kw)


def check(capi, c, algo=None, what="", **kw):
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], k_scale=c["k_scale"],
                               v_scale=c["v_scale"], **kw)
    got = run(capi, c, algo, **kw)
    assert_attention(got, ref, bound, what)
    return got


RAGGED = [(1, 1), (1, 17), (5, 5), (3, 64), (0, 40), (1, 129), (33, 200), (2, 0), (7, 3), (64, 64)]


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_ragged_batch(capi, algo, cache, dtype):
    """Lengths from none to several tiles, sequences without new tokens, more new tokens than keys (rows that see nothing)."""
    c = make_batch(RAGGED, 8, 2, 64, 16, dtype, E4M3 if cache == "e4m3" else dtype, seed=1)
    check(capi, c, algo)


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("d", [16, 80, 96, 112, 128])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_head_sizes(capi, algo, d, cache):
    c = make_batch([(1, 70), (19, 150), (130, 130)], 4, 2, d, 16, BF16, E4M3 if cache == "e4m3" else BF16, seed=d)
    check(capi, c, algo)


@pytest.mark.parametrize("algo", ALGOS)
def test_head_size_of_eight(capi, algo):
    check(capi, make_batch([(1, 70), (19, 150)], 4, 2, 8, 16, BF16, seed=3), algo)
    check(capi, make_batch([(1, 70), (19, 150)], 4, 2, 72, 16, F16, seed=4), algo)


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (5, 1), (14, 2), (40, 8), (33, 1), (130, 1)])
def test_head_groups(capi, algo, hq, hkv):
    """Groups that divide no tile, groups wider than a tile."""
    c = make_batch([(1, 90), (4, 40), (9, 300)], hq, hkv, 64, 16, BF16, seed=hq)
    check(capi, c, algo)


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("page", [1, 3, 8, 24, 32, 128, 200, 512])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_page_sizes(capi, algo, page, cache):
    """Pages that end inside a tile, pages wider than one."""
    c = make_batch([(1, 333), (40, 257), (1, 1)], 4, 2, 128, page, F16, E4M3 if cache == "e4m3" else F16, seed=page)
    check(capi, c, algo)


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("layout", ["joined", "heads"])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_cache_layouts(capi, algo, layout, cache):
    c = make_batch([(1, 333), (40, 257)], 8, 2, 128, 16, BF16, E4M3 if cache == "e4m3" else BF16, seed=5, layout=layout)
    assert not c["k_cache"].is_contiguous()
    check(capi, c, algo)


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 7, 64, 100])
def test_masks(capi, algo, causal, window):
    c = make_batch([(1, 333), (150, 150), (70, 400), (9, 4)], 6, 2, 64, 16, BF16, seed=window)
    check(capi, c, algo, causal=causal, window=window)


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("causal", [True, False])
def test_the_largest_window_is_none(capi, algo, causal):
    """Also where a sequence has more new tokens than keys, whose positions begin below zero."""
    c = make_batch([(1, 333), (9, 4), (5, 0), (40, 40)], 6, 2, 64, 16, BF16, seed=31)
    assert torch.equal(run(capi, c, algo, causal=causal, window=2 ** 31 - 1), run(capi, c, algo, causal=causal))


@pytest.mark.parametrize("max_q", [None, 1, 10 ** 6])
def test_most_new_tokens_need_not_be_exact(capi, max_q):
    """max_query_len only chooses the kernel: one that is too small, too large or unknown gives every row all the same."""
    c = make_batch([(1, 333), (150, 300), (0, 9), (1, 1)], 8, 2, 64, 16, BF16, seed=32)
    check(capi, dict(c, max_q=max_q), None)


@pytest.mark.parametrize("algo", ALGOS)
def test_pages_behind_a_window_may_be_gone(capi, algo):
    """Pages that no new token sees any more are not read: their table entries may be anything."""
    c = make_batch([(3, 500)], 4, 2, 64, 16, BF16, seed=9)
    c["table"][0, :(497 - 100 + 1) // 16] = -7
    ref = dict(c, table=c["table"].clamp_min(0))
    out, bound = attention_ref(ref["q"], torch.nan_to_num(c["k_cache"]), torch.nan_to_num(c["v_cache"]), c["cu"], c["lens"],
                               ref["table"], window=100)
    assert_attention(run(capi, c, algo, window=100), out, bound)


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_long_contexts_are_cut_between_ctas(capi, algo, cache):
    c = make_batch([(1, 40000), (2, 9000)], 8, 2, 128, 64, BF16, E4M3 if cache == "e4m3" else BF16, seed=11)
    check(capi, c, algo)


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_sequences_that_see_nothing_between_others(capi, algo, cache):
    """Many items without any keys after one whose last tile is copied row by row: none may wait for another."""
    c = make_batch([(3, 50)] + [(2, 0)] * 2000 + [(40, 70)] + [(1, 0)] * 7, 4, 2, 64, 16, BF16, E4M3 if cache == "e4m3" else BF16, seed=25)
    check(capi, c, algo)


@pytest.mark.parametrize("algo", ALGOS)
def test_many_sequences(capi, algo):
    c = make_batch([(1, 1 + (37 * i) % 211) for i in range(300)], 4, 2, 64, 16, BF16, seed=12)
    check(capi, c, algo)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_prompts_and_chunks(capi, cache):
    """The dispatcher's own choice for whole prompts, chunks over a context and decode rows in one batch."""
    c = make_batch([(700, 700), (1, 1500), (256, 1800), (31, 31), (1, 64)], 8, 2, 128, 16, BF16,
                   E4M3 if cache == "e4m3" else BF16, seed=13)
    check(capi, c)
    check(capi, c, window=300)
    check(capi, c, causal=False)


@pytest.mark.parametrize("algo", ALGOS)
def test_sharp_and_growing_scores(capi, algo):
    """Maxima that grow by far more than the lazy rescaling allows, key after key; and one key that takes all."""
    c = make_batch([(40, 700)], 4, 2, 64, 16, BF16, seed=14)
    row = torch.arange(c["k_cache"].shape[0] * 16, device="cuda")
    order = torch.zeros_like(row)
    pages = c["table"][0, :44].long()
    order.view(-1, 16)[pages] = torch.arange(44 * 16, device="cuda").view(44, 16)
    c["k_cache"].mul_((order.float() * 0.02 + 0.1).to(BF16).view(-1, 16, 1, 1))
    check(capi, c, algo)
    check(capi, c, algo, scale=3.0)


@pytest.mark.parametrize("algo", ALGOS)
def test_tail_rows(capi, algo):
    """Rows behind the last sequence: zeros in a new output, left as they were in the caller's."""
    c = make_batch([(2, 30), (3, 50)], 4, 2, 64, 16, BF16, seed=15, tail=6)
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"])
    got = run(capi, c, algo)
    assert_attention(got, ref, bound)
    assert (got[5:] == 0).all()
    mine = torch.full((11, 3, 4, 64), 7.0, dtype=BF16, device="cuda")[:, 1]
    torch.ops.zentorch.zentorch_paged_attention.out(mine, c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], 3)
    assert_attention(mine[:5], ref[:5], bound[:5])
    assert (mine[5:] == 7).all()
    c = make_batch([(2, 30)], 5, 1, 72, 16, BF16, seed=15, tail=700)      # a tail wider than the grid, heads of 144 bytes
    got = run(capi, c, algo)
    assert (got[2:] == 0).all() and (got[:2] != 0).any()


def test_unaligned_query_and_output(capi):
    c = make_batch([(2, 30), (40, 50)], 4, 2, 64, 16, BF16, seed=16)
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"])
    wide = torch.full((42, 4 * 64 + 3), 5.0, dtype=BF16, device="cuda")
    wide[:, 3:] = c["q"].reshape(42, -1)
    out = torch.zeros(42, 4, 65, dtype=BF16, device="cuda")[..., 1:]
    torch.ops.zentorch.zentorch_paged_attention.out(out, wide[:, 3:].view(42, 4, 64), c["k_cache"], c["v_cache"], c["cu"], c["lens"],
                                                    c["table"])
    assert_attention(out, ref, bound)


@pytest.mark.parametrize("algo", ALGOS)
def test_results_repeat(capi, algo):
    c = make_batch([(1, 5000), (50, 3000), (1, 77)], 8, 2, 128, 16, BF16, seed=17)
    a, b = run(capi, c, algo), run(capi, c, algo)
    assert torch.equal(a, b)


@pytest.mark.parametrize("algo", ALGOS)
def test_nan_and_infinite_queries_stay_in_their_rows(capi, algo):
    c = make_batch([(5, 300), (1, 40)], 4, 2, 64, 16, BF16, seed=18)
    clean = run(capi, c, algo)
    c["q"][2, 1, 5], c["q"][3, 2, 0] = float("nan"), float("inf")
    got = run(capi, c, algo)
    assert got[2, 1].isnan().all() and got[3, 2].isnan().all()
    keep = torch.ones(6, 4, dtype=torch.bool, device="cuda")
    keep[2, 1] = keep[3, 2] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_a_key_of_nan_among_tiles_of_rows(capi, algo, cache):
    """Rows of several tiles, some of which see the key: NaN in all their columns, the bound of every other row."""
    n, kv, key = 200, 300, 180
    c = make_batch([(n, kv), (1, 20)], 4, 2, 64, 16, BF16, E4M3 if cache == "e4m3" else BF16, seed=33)
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], k_scale=c["k_scale"],
                               v_scale=c["v_scale"])
    raw = c["k_cache"].view(torch.uint8) if cache == "e4m3" else c["k_cache"]
    raw[c["table"][0, key // 16].long(), key % 16, 1, 9] = 0x7f if cache == "e4m3" else float("nan")
    got = run(capi, c, algo)
    hit = torch.zeros(n + 1, 4, dtype=torch.bool)
    hit[key - (kv - n):n, 2:] = True
    assert got.cpu()[hit].isnan().all()
    assert bool(((got.double().cpu() - ref).abs()[~hit] <= bound[~hit]).all())


@pytest.mark.parametrize("algo", ALGOS)
def test_nan_in_a_key_reaches_the_rows_that_see_it(capi, algo):
    c = make_batch([(4, 40)], 2, 1, 64, 16, BF16, seed=19)
    clean = run(capi, c, algo)
    c["k_cache"][c["table"][0, 2].long(), 38 - 32] = float("nan")      # key 38: new tokens 2 and 3 see it
    got = run(capi, c, algo)
    assert torch.equal(got[:2], clean[:2]) and got[2:].isnan().all()


@pytest.mark.parametrize("algo", ALGOS)
@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128)])
@pytest.mark.parametrize("n,kv,window", [(4, 40, 0), (30, 300, 100), (200, 400, 0), (300, 300, 7)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(capi, algo, cache, dtype, d, n, kv, window):
    """NaN and infinities in values of keys that some rows of a tile see and others do not: the latter keep their results, the former
    get them in their columns and nowhere else.  What is finite is held to the bound of every other test (rows that the tensor
    cores spoilt are summed again in another order, so bits may differ); the streaming kernel leaves even the bits."""
    c = make_batch([(1, 20), (n, kv), (3, 9)], 4, 2, d, 16, dtype, E4M3 if cache == "e4m3" else dtype, seed=26)
    clean = run(capi, c, algo, window=window)
    raw = c["v_cache"].view(torch.uint8) if cache == "e4m3" else c["v_cache"]
    special = [(kv - 2, 0, 3, float("nan")), (kv - n // 2, 1, 17, float("inf")), (kv - n // 2, 1, d - 1, float("-inf")),
               (max(kv - n - 1, 0), 0, 30, float("nan")), (kv - 1, 1, 8, float("inf")), (kv - 1, 1, 17, float("-inf"))]
    want = clean.double()
    pos = torch.arange(kv - n, kv, device="cuda")
    for key, h, col, value in special:
        if cache == "e4m3":
            value = float("nan")                                # the type has no infinities
        raw[c["table"][1, key // 16].long(), key % 16, h, col] = 0x7f if cache == "e4m3" else value
        sees = (pos >= key) & ((pos - window < key) if window else True)
        want[1:1 + n, 2 * h:2 * h + 2, col] += torch.where(sees, value, 0.0).unsqueeze(1)
    got = run(capi, c, algo, window=window)
    fine = torch.isfinite(want)
    assert not fine.all()
    if algo != "tcgen05":
        assert torch.equal(got[fine], clean[fine])
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], window=window, k_scale=c["k_scale"],
                               v_scale=c["v_scale"])
    keep = fine.cpu()
    assert torch.equal(torch.isfinite(ref), keep)
    assert bool(((got.double().cpu() - ref).abs()[keep] <= bound[keep]).all())
    assert torch.equal(got.double()[~fine].nan_to_num(5e4, 6e4, 7e4), want[~fine].nan_to_num(5e4, 6e4, 7e4))


def test_bad_pages_and_lengths_are_reported(capi):
    c = make_batch([(1, 60), (1, 100)], 4, 2, 64, 16, BF16, seed=20)
    good = run(capi, c)
    c["table"][0, 1] = c["k_cache"].shape[0]
    got = run(capi, c)
    assert capi.poll_device_status(reset=True) == 106
    assert torch.equal(got[1], good[1]) and torch.isfinite(got).all()
    c["table"][0, 1] = 0
    c["lens"][0] = 10 ** 9
    c["table"][0] = c["table"][1]
    run(capi, c)
    assert capi.poll_device_status(reset=True) == 106
    c["lens"][0], c["cu"][2] = 60, 50
    run(capi, c)
    assert capi.poll_device_status(reset=True) == 106


def test_captured_call_follows_the_lengths(capi):
    """A captured decode step replayed for growing lengths, on its own stream, twice in flight on two streams."""
    c = make_batch([(1, 600), (1, 90)], 8, 2, 128, 16, BF16, seed=21)
    d = make_batch([(1, 700), (1, 10)], 8, 2, 128, 16, BF16, seed=22)
    ops = torch.ops.zentorch
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x, s in ((c, streams[0]), (d, streams[1])):
        run(capi, x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(ops.zentorch_paged_attention(x["q"], x["k_cache"], x["v_cache"], x["cu"], x["lens"], x["table"], 1))
        graphs.append(graph)
    for lens in ([1, 1], [600, 90], [333, 64]):
        for x, g, s in ((c, graphs[0], streams[0]), (d, graphs[1], streams[1])):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                x["lens"].copy_(torch.minimum(torch.tensor(lens, dtype=torch.int32), torch.tensor([600, 10], dtype=torch.int32)), non_blocking=False)
                g.replay()
        torch.cuda.synchronize()
        for x, o in ((c, outs[0]), (d, outs[1])):
            ref, bound = attention_ref(x["q"], x["k_cache"], x["v_cache"], x["cu"], x["lens"], x["table"])
            assert_attention(o, ref, bound, str(lens))


def test_empty_calls(capi):
    c = make_batch([(1, 16)], 4, 2, 64, 16, BF16, seed=23)
    empty = c["q"][:0]
    cu = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert torch.ops.zentorch.zentorch_paged_attention(empty, c["k_cache"], c["v_cache"], cu, c["lens"], c["table"]).shape == (0, 4, 64)
    none = torch.ops.zentorch.zentorch_paged_attention(c["q"], c["k_cache"], c["v_cache"], cu[:1], c["lens"][:0], c["table"][:0])
    assert (none == 0).all()
    no_pages = torch.ops.zentorch.zentorch_paged_attention(c["q"], c["k_cache"][:0], c["v_cache"][:0], c["cu"],
                                                           torch.zeros_like(c["lens"]), c["table"][:, :0])
    assert (no_pages == 0).all()


def test_refusals(capi):
    c = make_batch([(1, 16)], 4, 2, 64, 16, BF16, seed=24)
    op = torch.ops.zentorch.zentorch_paged_attention
    args = [c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"]]

    def refused(match, at=None, value=None, **kw):
        a = list(args)
        if at is not None:
            a[at] = value
        with pytest.raises(RuntimeError, match=match):
            op(*a, **kw)

    refused("bfloat16 or float16", 0, c["q"].float())
    refused("heads of 64", 0, c["q"][..., :32])
    refused("multiple of the caches' heads", 0, c["q"][:, :3])
    refused("caches must be", 1, c["k_cache"].half())
    refused("shape of key_cache", 2, c["v_cache"][1:])
    refused("must be int32", 3, c["cu"].long())
    refused("one entry more", 3, c["cu"][:1])
    refused("row per sequence", 5, c["table"][:0])
    refused("input's device", 4, c["lens"].cpu())
    refused("window must not be negative", window=-1)
    refused("scale must be positive", scale=0.0)
    refused("belongs to a float8", k_scale=torch.ones(2, device="cuda"))
    into = torch.ops.zentorch.zentorch_paged_attention.out
    with pytest.raises(RuntimeError, match="share memory with query"):
        into(c["q"][:, :4], *args)
    with pytest.raises(RuntimeError, match="hold an element twice"):
        into(torch.zeros(1, 1, 64, dtype=BF16, device="cuda").expand(1, 4, 64), *args)
    refused("16-byte aligned", 1, torch.zeros(c["k_cache"].shape[0], 16, 2, 65, dtype=BF16, device="cuda")[..., 1:])
    e = c["k_cache"].nan_to_num().to(E4M3)
    with pytest.raises(RuntimeError, match="needs k_scale"):
        op(c["q"], e, e, c["cu"], c["lens"], c["table"])
    wide = torch.zeros(4, 16, 2, 136, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="head_dim must be a multiple"):
        op(torch.zeros(1, 4, 136, dtype=BF16, device="cuda"), wide, wide, c["cu"], c["lens"], c["table"])
