"""Values that are not finite in the paged attention, one pair to a column: what a row gets follows from the values that it sees."""
import pytest
import torch

from _cache_ref import attention_ref, make_batch
from test_paged_attention_gpu import ALGOS, BF16, E4M3, F16, capi, run  # noqa: F401  (capi is a fixture)

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


SHAPES = {"groups of 5, heads of 80, window": (10, 2, 80, 24, [(70, 300), (1, 90), (33, 20), (250, 250)], dict(window=64)),
          "one key head, wide group": (33, 1, 128, 16, [(40, 200), (9, 500)], {}),
          "not causal, window": (4, 4, 64, 7, [(150, 400), (5, 5)], dict(causal=False, window=30)),
          "heads of 16": (8, 2, 16, 32, [(300, 700), (64, 64)], {}),
          "cut between CTAs": (4, 2, 128, 16, [(200, 6000)], dict(window=5000))}


@pytest.mark.parametrize("algo", ["tcgen05", "dealt", "rows16", "slices3"])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("where", ["anywhere", "late"])
def test_scattered_values(capi, algo, cache, shape, where):  # noqa: F811
    """NaN and infinities in a handful of keys and values of every sequence and head (of an e4m3 cache, NaN among the values)."""
    hq, hkv, d, page, pairs, kw = SHAPES[shape]
    dtype = BF16 if where == "late" else F16
    c = make_batch(pairs, hq, hkv, d, page, dtype, E4M3 if cache == "e4m3" else dtype, seed=51)
    g, spoilt = torch.Generator().manual_seed(52), []
    for b, (n, kv) in enumerate(pairs):
        for h in range(hkv):
            for i in range(6):
                key = int(torch.randint(max(kv - n, 0) if where == "late" else 0, kv, (1,), generator=g))
                col, value = int(torch.randint(0, d, (1,), generator=g)), (NAN, INF, -INF)[i % 3]
                row = (c["table"][b, key // page].long(), key % page, h)
                if cache == "e4m3":
                    c["v_cache"].view(torch.uint8)[(*row, col)] = 0x7f if i % 2 else 0xff
                elif i == 5:
                    c["k_cache"][(*row, col)] = NAN
                    spoilt.append((b, h, key))
                elif i == 4:
                    c["v_cache"][row] = value
                else:
                    c["v_cache"][(*row, col if i else slice(0, 1))] = value
    ref, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"], k_scale=c["k_scale"],
                               v_scale=c["v_scale"], **kw)
    for b, h, key in spoilt:                             # (the reference takes scores of NaN for keys that are not seen)
        n, kv = pairs[b]
        pos, window = torch.arange(kv - n, kv), kw.get("window", 0)
        sees = ((pos >= key) | (not kw.get("causal", True))) & ((key > pos - window) | (not window))
        ref[int(c["cu"][b]):int(c["cu"][b + 1]), h * hq // hkv:(h + 1) * hq // hkv][sees] = NAN
    assert not torch.isfinite(ref).all()
    check_special(run(capi, c, algo, **kw), ref, bound)


@pytest.mark.parametrize("n,kv,key", [(512, 8000, 5), (512, 8000, 7999), (2048, 2048, 5), (2048, 2048, 1024)])
def test_one_spoilt_value_does_not_stall_the_batch(capi, n, kv, key):  # noqa: F811
    """Rows that are gone through again cost a bounded multiple of the call (8 - 110 here; one key after another in every row was
    600 and more)."""
    c = make_batch([(n, kv)], 32, 8, 128, 32, BF16, seed=53)

    def time():
        run(capi, c, "tcgen05")
        ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        ends[0].record()
        run(capi, c, "tcgen05")
        ends[1].record()
        torch.cuda.synchronize()
        return ends[0].elapsed_time(ends[1])
    clean = min(time() for _ in range(5))
    c["v_cache"][c["table"][0, key // 32].long(), key % 32, :, 3] = NAN
    assert min(time() for _ in range(2)) <= 200 * clean
