"""A decoder layer's steps as they are used: quantized projections, rotary positions, the paged cache and its attention, with
forks, cuts and compactions in between."""
import pytest
import torch

from _cache_ref import assert_attention, assert_rope, attention_ref, gather_rows, rope_ref
from _util import make_int8_case, make_woq_case

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D, INTER = 512, 8, 2, 64, 1024
SHAPES = {"q": (HIDDEN, HQ * D), "k": (HIDDEN, HKV * D), "v": (HIDDEN, HKV * D), "o": (HQ * D, HIDDEN),
          "gate": (HIDDEN, INTER), "up": (HIDDEN, INTER), "down": (INTER, HIDDEN)}


@pytest.fixture(scope="module")
def pkg(zt):
    from zentorch_b200 import _capi, cache, tp
    assert torch.cuda.is_available() and _capi.lib().zt_device_supported() == 1
    return _capi, cache, tp


def linears(pkg, kind):
    capi, _, tp = pkg
    full = {}
    for i, (name, (k, n)) in enumerate(SHAPES.items()):
        if kind == "woq":
            _, q, s, _, _ = make_woq_case(1, k, n, 128, seed=70 + i, bias=False)
            full[name] = (capi.woq_repack_weight(q.cuda()).t(), s.cuda(), None, None)
        else:
            _, w, ws, _ = make_int8_case(1, k, n, seed=70 + i)
            full[name] = (w.cuda(), ws.cuda(), None)
    return tp.DecoderLayerLinears(kind, full)


class Recorder:
    """torch.ops.zentorch, with the calls noted."""

    def __init__(self):
        self.rope, self.attention = None, None

    def zentorch_rope_cache(self, *args, **kw):
        out = torch.ops.zentorch.zentorch_rope_cache(*args, **kw)
        self.rope = (args, kw, out)
        return out

    def zentorch_paged_attention(self, *args, **kw):
        out = torch.ops.zentorch.zentorch_paged_attention(*args, **kw)
        self.attention = (args, kw, out)
        return out


@pytest.mark.parametrize("kind", ["woq", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_steps_with_forks_cuts_and_compactions(pkg, kind, dtype):
    capi, cache_mod, tp = pkg
    freq, factor = cache_mod.rope_frequencies(D, 500000.0, {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64},
                                              device="cuda")
    e4m3 = dtype == torch.float8_e4m3fn
    scales = dict(k_scale=torch.full((2, HKV), 0.02), v_scale=torch.full((2, HKV), 0.015)) if e4m3 else {}
    cache = cache_mod.PagedKVCache(2, 80, 16, HKV, D, dtype=dtype, **scales)
    for t in cache.layers:
        t.view(torch.uint8).fill_(0x7f)                     # NaN wherever nothing was stored
    rec = Recorder()
    layers = [tp.DecoderLayer(linears(pkg, kind), HQ, HKV, D, freq, factor, ops=rec) for _ in range(2)]
    history = {}                                            # sequence -> (k, v) rows per layer, in 64 bits
    g = torch.Generator(device="cuda").manual_seed(3)

    def run(new):
        step = cache.step(new)
        x = torch.randn(step.tokens, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
        starts = [0]
        for _, n in new:
            starts.append(starts[-1] + n)
        for i, layer in enumerate(layers):
            x = layer(x, cache, i, step)
            (q, k, v, pos, *_), kw, q_out = rec.rope
            assert_rope(q_out, q, pos, freq, factor, False)
            keys, arith = rope_ref(k, pos, freq, factor, False)
            for (name, n), at in zip(new, starts):
                rows = history.setdefault(name, [([], [], []), ([], [], [])])[i]
                rows[0].append(keys[at:at + n])
                rows[1].append(v[at:at + n].double().cpu())
                rows[2].append(arith[at:at + n])
            args, kw, out = rec.attention
            ref, bound = attention_ref(*args[:6], window=kw["window"], k_scale=kw["k_scale"], v_scale=kw["v_scale"])
            assert_attention(out, ref, bound, f"layer {i} of {new}")
        check_contents()
        return x

    def check_contents():
        for name, both in history.items():
            table = torch.tensor(cache.pages(name), dtype=torch.int32, device="cuda")
            for i, (ks, vs, arith) in enumerate(both):
                k, v, a = (torch.cat(t) if t else torch.zeros(0, HKV, D, dtype=torch.float64) for t in (ks, vs, arith))
                got_k, got_v = gather_rows(cache.keys(i), table, len(k)), gather_rows(cache.values(i), table, len(v))
                if e4m3:
                    k, a, v = k / 0.02, a / 0.02, v / 0.015
                    k, v = k.clamp(-448, 448), v.clamp(-448, 448)
                    # half a step: 2^-4 of the value, 2^-10 among the subnormals; the scale itself is an fp32 number
                    half = lambda x: (x.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) * (1 + 2.0 ** -20)   # noqa: E731
                    assert ((got_v - v).abs() <= half(v)).all()
                else:
                    half = lambda x: x.abs() * 2.0 ** -8                                                 # noqa: E731
                    assert torch.equal(got_v, v)
                assert ((got_k - k).abs() <= half(k) + 1.25 * a).all(), f"{name}, layer {i}"

    for name in ("a", "b"):
        cache.add(name)
    run([("a", 100), ("b", 7)])                             # two prompts
    run([("a", 1), ("b", 40)])                              # a decode row beside a chunk
    cache.fork("a", "c")
    history["c"] = [tuple([list(t) for t in rows]) for rows in history["a"]]
    run([("a", 1), ("b", 1), ("c", 3)])                     # the fork leaves the shared page
    cache.truncate("c", 90)
    for rows in history["c"]:
        for t in rows:
            whole = torch.cat(t)[:90]
            t.clear()
            t.append(whole)
    run([("c", 2), ("a", 1)])
    cache.free("b")
    del history["b"]
    assert cache.compact() > 0
    check_contents()
    run([("c", 1), ("a", 1)])
    assert cache.free_pages == 80 - len({p for n in history for p in cache.pages(n)})


def test_captured_decode_steps(pkg):
    """A layer's decode step captured once and replayed with the step's tensors refilled gives what it gives eagerly."""
    _, cache_mod, tp = pkg
    freq, factor = cache_mod.rope_frequencies(D, device="cuda")
    lin = linears(pkg, "woq")
    layer = tp.DecoderLayer(lin, HQ, HKV, D, freq, factor)
    caches = [cache_mod.PagedKVCache(1, 40, 16, HKV, D) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(4)
    prompt = torch.randn(50, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
    for c in caches:
        c.add("a"), c.add("b")
        layer(prompt, c, 0, c.step([("a", 20), ("b", 30)]))
    x = torch.zeros(2, HIDDEN, dtype=torch.bfloat16, device="cuda")
    held = None
    graph = torch.cuda.CUDAGraph()
    for i in range(20):
        new = torch.randn(2, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
        want = layer(new, caches[0], 0, caches[0].step([("a", 1), ("b", 1)]))
        step = caches[1].step([("a", 1), ("b", 1)])
        if held is None:
            held = step
            held.block_table = torch.nn.functional.pad(held.block_table, (0, 3))     # room for the pages to come
            x.copy_(new)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                layer(x, caches[1], 0, held)                                         # warm-up writes what the replay writes again
            torch.cuda.current_stream().wait_stream(side)
            with torch.cuda.graph(graph):
                out = layer(x, caches[1], 0, held)
        else:
            x.copy_(new)
            for name in ("positions", "slots", "cu_seqlens_q", "seq_lens"):
                getattr(held, name).copy_(getattr(step, name))
            held.block_table[:, :step.block_table.shape[1]].copy_(step.block_table)
        graph.replay()
        assert torch.equal(out, want), i
