"""The paged cache's bookkeeping, the rotary frequencies, and what the operators check before any device work: no GPU needed."""
import ctypes as C
import math
import os
import random
import sys
from pathlib import Path

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from _cache_ref import PlainOps, attention_ref, plain_copy_pages, rope_ref

ROOT = Path(__file__).resolve().parent.parent


def make_cache(pages=12, page=4, layers=2, **kw):
    from zentorch_b200.cache import PagedKVCache
    return PagedKVCache(layers, pages, page, 1, 8, device="cpu", copy_pages=plain_copy_pages, dtype=torch.float32, **kw)


def fill(cache, step, rng):
    """Writes a distinct number into every new slot of every layer and returns the numbers."""
    marks = [rng.random() for _ in range(step.tokens)]
    for layer in range(len(cache.layers)):
        for m, s in zip(marks, step.slots.tolist()):
            cache.keys(layer)[s // cache.page_size, s % cache.page_size] = m + layer
            cache.values(layer)[s // cache.page_size, s % cache.page_size] = -m - layer
    return marks


def read(cache, name, layer):
    pages = torch.tensor(cache.pages(name), dtype=torch.long)
    k = cache.keys(layer)[pages].flatten(0, 1)[:cache.length(name), 0, 0]
    v = cache.values(layer)[pages].flatten(0, 1)[:cache.length(name), 0, 0]
    assert torch.equal(k - layer, -(v + layer))
    return (k - layer).tolist()


def test_random_histories_keep_every_sequence(zt):
    """Random steps, forks, cuts, frees and compactions: each sequence reads back exactly what was written to it."""
    for seed in range(20):
        rng = random.Random(seed)
        cache = make_cache(pages=40, page=rng.choice([1, 3, 4, 16]))
        history, names = {}, iter(range(10 ** 6))
        for _ in range(60):
            move = rng.choice(["add", "step", "step", "step", "fork", "cut", "free", "compact"])
            if move == "add":
                n = next(names)
                cache.add(n)
                history[n] = []
            elif move == "fork" and history:
                a, n = rng.choice(list(history)), next(names)
                cache.fork(a, n)
                history[n] = list(history[a])
            elif move == "cut" and history:
                a = rng.choice(list(history))
                keep = rng.randint(0, len(history[a]))
                cache.truncate(a, keep)
                history[a] = history[a][:keep]
            elif move == "free" and history:
                a = rng.choice(list(history))
                cache.free(a)
                del history[a]
            elif move == "compact":
                cache.compact()
                used = {p for n in history for p in cache.pages(n)}
                assert used == set(range(len(used)))
            elif move == "step" and history:
                batch = [(a, rng.randint(0, 6)) for a in rng.sample(list(history), rng.randint(1, len(history)))]
                free, before = cache.free_pages, {a: (cache.pages(a), cache.length(a)) for a in history}
                try:
                    step = cache.step(batch)
                except MemoryError:
                    assert cache.free_pages == free and before == {a: (cache.pages(a), cache.length(a)) for a in history}
                    continue
                marks = fill(cache, step, rng)
                at = 0
                for i, (a, count) in enumerate(batch):
                    assert step.positions[at:at + count].tolist() == list(range(len(history[a]), len(history[a]) + count))
                    history[a] += [pytest.approx(m, abs=1e-6) for m in marks[at:at + count]]
                    at += count
                    assert step.cu_seqlens_q[i + 1] == at and step.seq_lens[i] == len(history[a])
                    pages = cache.pages(a)
                    assert step.block_table[i, :len(pages)].tolist() == list(pages)
                assert step.max_query_len == max(c for _, c in batch)
            for a in history:
                for layer in range(2):
                    assert read(cache, a, layer) == history[a]
            used = {p for n in history for p in cache.pages(n)}
            assert cache.free_pages == cache.num_pages - len(used)


def test_a_fork_copies_only_the_page_that_is_written(zt):
    copies = []

    def copy(caches, src, dst):
        copies.append((src.tolist(), dst.tolist()))
        plain_copy_pages(caches, src, dst)
    from zentorch_b200.cache import PagedKVCache
    cache = PagedKVCache(2, 12, 4, 1, 8, device="cpu", copy_pages=copy, dtype=torch.float32)
    cache.add("a")
    cache.step([("a", 6)])
    cache.fork("a", "b")
    cache.fork("a", "c")
    assert cache.pages("b") == cache.pages("a") == (0, 1) and cache.free_pages == 10
    cache.step([("a", 1), ("b", 1), ("c", 1)])                 # two of the three leave the shared page, the third keeps it
    assert copies == [([1, 1], [2, 3])]
    assert cache.pages("a") == (0, 2) and cache.pages("b") == (0, 3) and cache.pages("c") == (0, 1)
    cache.free("a")
    cache.free("c")
    assert cache.free_pages == 12 - 2
    cache.step([("b", 1)])
    assert len(copies) == 1
    assert cache.compact() == 1 and cache.pages("b") == (0, 1) and copies[-1] == ([3], [1])


def test_cache_refusals(zt):
    from zentorch_b200.cache import PagedKVCache
    cache = make_cache(pages=2)
    cache.add("a")
    with pytest.raises(ValueError, match="already"):
        cache.add("a")
    with pytest.raises(KeyError, match="no sequence"):
        cache.fork("b", "c")
    with pytest.raises(ValueError, match="once in a step"):
        cache.step([("a", 1), ("a", 1)])
    with pytest.raises(ValueError, match="negative"):
        cache.step([("a", -1)])
    with pytest.raises(MemoryError, match="needs 3 pages, 2 are free"):
        cache.step([("a", 9)])
    cache.step([("a", 8)])
    with pytest.raises(ValueError, match="cannot cut"):
        cache.truncate("a", 9)
    with pytest.raises(ValueError, match="positive"):
        PagedKVCache(1, 0, 4, 1, 8, device="cpu")
    with pytest.raises(ValueError, match="float8"):
        PagedKVCache(1, 1, 4, 1, 8, device="cpu", k_scale=torch.ones(1, 1))
    with pytest.raises(ValueError, match="k_scale must have shape"):
        PagedKVCache(1, 1, 4, 2, 8, device="cpu", dtype=torch.float8_e4m3fn, k_scale=torch.ones(1, 1))


def test_rope_frequencies(zt):
    from zentorch_b200.cache import rope_frequencies
    plain, one = rope_frequencies(128, 10000.0)
    want = [10000.0 ** (-2 * i / 128) for i in range(64)]
    assert one == 1.0 and torch.allclose(plain.double(), torch.tensor(want, dtype=torch.float64), rtol=2 ** -23)
    lin, _ = rope_frequencies(128, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.equal(lin, plain / 4)
    ntk, _ = rope_frequencies(128, 10000.0, {"type": "ntk", "factor": 4.0})
    assert ntk[0] == 1 and math.isclose(float(ntk[-1]), float(plain[-1]) / 4, rel_tol=1e-6)
    got, factor = rope_frequencies(128, 500000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                                   "high_freq_factor": 4.0, "original_max_position_embeddings": 8192})
    assert factor == 1.0
    for i in range(64):
        f = 500000.0 ** (-2 * i / 128)
        turns = 8192 * f / (2 * math.pi)
        keep = min(max((turns - 1) / 3, 0), 1)
        assert math.isclose(float(got[i]), f * keep + f / 8 * (1 - keep), rel_tol=1e-6)
    got, factor = rope_frequencies(64, 10000.0, {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096})
    assert math.isclose(factor, 0.1 * math.log(16) + 1)
    f = [10000.0 ** (-2 * i / 64) for i in range(32)]
    first = math.floor(32 * math.log(4096 / (32 * 2 * math.pi)) / math.log(10000))
    last = math.ceil(32 * math.log(4096 / (2 * math.pi)) / math.log(10000))
    for i in range(32):
        keep = 1 - min(max((i - first) / (last - first), 0), 1)
        assert math.isclose(float(got[i]), f[i] * keep + f[i] / 16 * (1 - keep), rel_tol=1e-6)
    assert rope_frequencies(0)[0].shape == (0,)
    for bad in ({"type": "other"}, {"type": "linear", "factor": 0.5}):
        with pytest.raises(ValueError):
            rope_frequencies(64, scaling=bad)
    with pytest.raises(ValueError, match="even"):
        rope_frequencies(7)


def test_reference_gradientless_sanity():
    """The 64-bit evaluation itself, against torch's own softmax attention and a rotation by hand."""
    from _cache_ref import make_batch
    c = make_batch([(3, 7)], 4, 2, 8, 4, torch.float16, device="cpu")
    out, bound = attention_ref(c["q"], c["k_cache"], c["v_cache"], c["cu"], c["lens"], c["table"])
    pages = c["table"][0, :2].long()
    k, v = (x[pages].flatten(0, 1)[:7].double().repeat_interleave(2, 1).transpose(0, 1) for x in (c["k_cache"], c["v_cache"]))
    mask = torch.arange(7)[None, :] <= torch.arange(4, 7)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(c["q"].double().transpose(0, 1), k, v, attn_mask=mask).transpose(0, 1)
    assert torch.allclose(out, want, atol=1e-12) and (bound > 0).all()
    x = torch.tensor([[[1.0, 0.0, 5.0]]])
    y, _ = rope_ref(x, torch.tensor([2]), torch.tensor([0.25]), 2.0, False)
    assert torch.allclose(y, torch.tensor([[[2 * math.cos(0.5), 2 * math.sin(0.5), 5.0]]], dtype=torch.float64))


def test_schemas_and_meta_kernels(zt):
    ops = torch.ops.zentorch
    q, k = torch.empty(5, 8, 64, dtype=torch.bfloat16, device="meta"), torch.empty(5, 2, 64, dtype=torch.bfloat16, device="meta")
    cache = torch.empty(9, 16, 2, 64, dtype=torch.bfloat16, device="meta")
    i = torch.empty(5, dtype=torch.int64, device="meta")
    n = torch.empty(3, dtype=torch.int32, device="meta")
    f = torch.empty(32, device="meta")
    qr, kr = ops.zentorch_rope(q, k, i, f)
    assert qr.shape == q.shape and kr.shape == k.shape and qr.dtype == torch.bfloat16
    assert ops.zentorch_rope_cache(q, k, k, i, f, cache, cache, i).shape == q.shape
    out = ops.zentorch_paged_attention(q, cache, cache, n, n[:2], torch.empty(2, 4, dtype=torch.int32, device="meta"))
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    assert ops.zentorch_cache_copy_pages([cache], i, i) is None
    assert "Tensor(a!) key_cache" in str(ops.zentorch_rope_cache.default._schema)
    assert "Tensor(a!)[] caches" in str(ops.zentorch_cache_copy_pages.default._schema)
    assert "Tensor(a!) out" in str(ops.zentorch_paged_attention.out._schema)
    with pytest.raises((RuntimeError, NotImplementedError)):          # no CPU kernels
        ops.zentorch_rope(torch.zeros(1, 1, 8), torch.zeros(1, 1, 8), torch.zeros(1, dtype=torch.int64), torch.zeros(4))


def test_c_entry_points_refuse_before_device_work(zt):
    from zentorch_b200 import _capi
    lib = _capi.lib()
    one = 4096  # never dereferenced: validation fails first

    def refused(rc, code, text):
        assert rc == code and text in lib.zt_last_error(), (rc, lib.zt_last_error())

    refused(lib.zt_rope(None, None), 1, b"null argument block")
    a = _capi.RopeArgs()
    a.tokens, a.q_heads, a.kv_heads, a.head_dim, a.rot_dim, a.dtype = 2, 4, 2, 64, 63, _capi.ZT_BF16
    refused(lib.zt_rope(C.byref(a), None), 1, b"must be even")
    a.rot_dim, a.dtype = 64, _capi.ZT_S8
    refused(lib.zt_rope(C.byref(a), None), 1, b"bfloat16, float16 or float32")
    a.dtype = _capi.ZT_BF16
    refused(lib.zt_rope(C.byref(a), None), 1, b"null tensor pointer")
    a.q = a.k = a.q_out = a.positions = a.inv_freq = one
    refused(lib.zt_rope(C.byref(a), None), 1, b"null pointer among")
    a.k_cache, a.cache_dtype = one, _capi.ZT_F32
    refused(lib.zt_rope(C.byref(a), None), 1, b"type of the key")
    a.cache_dtype = _capi.ZT_E4M3
    refused(lib.zt_rope(C.byref(a), None), 1, b"page size")
    a.page_size, a.v, a.v_cache, a.slots = 16, one, one, one
    refused(lib.zt_rope(C.byref(a), None), 1, b"needs k_scale")
    a.tokens = -1
    refused(lib.zt_rope(C.byref(a), None), 1, b"out of range")

    refused(lib.zt_cache_copy_pages(None, None), 1, b"null argument block")
    c = _capi.CacheCopyArgs()
    c.n_caches, c.n_pairs = 1, 1
    refused(lib.zt_cache_copy_pages(C.byref(c), None), 1, b"null pointer")
    c.n_pairs = -1
    refused(lib.zt_cache_copy_pages(C.byref(c), None), 1, b"negative size")
    c.n_pairs = 0
    assert lib.zt_cache_copy_pages(C.byref(c), None) == 0

    refused(lib.zt_paged_attention(None, None), 1, b"null argument block")
    p = _capi.PagedAttentionArgs()
    p.tokens, p.batch, p.q_heads, p.kv_heads, p.head_dim, p.dtype, p.cache_dtype = 4, 2, 6, 4, 64, _capi.ZT_BF16, _capi.ZT_BF16
    p.page_size, p.max_blocks, p.num_pages, p.scale = 16, 4, 8, 0.125
    refused(lib.zt_paged_attention(C.byref(p), None), 1, b"multiple of the key/value heads")
    p.q_heads = 8
    for field, bad, code, text in (("dtype", _capi.ZT_F32, 1, b"query must be"), ("cache_dtype", _capi.ZT_F16, 1, b"type of the query"),
                                   ("head_dim", 68, 2, b"multiple of 8"), ("head_dim", 136, 2, b"up to 128"), ("page_size", 0, 1, b"page size"),
                                   ("scale", float("nan"), 1, b"positive and finite"), ("window", -1, 1, b"window"),
                                   ("batch", 20000, 2, b"at most 16384"), ("max_blocks", 1 << 28, 2, b"2^30 keys"),
                                   ("tokens", 1 << 28, 2, b"query rows"), ("algo", 9, 1, b"unknown algo")):
        good = getattr(p, field)
        setattr(p, field, bad)
        refused(lib.zt_paged_attention(C.byref(p), None), code, text)
        setattr(p, field, good)
    refused(lib.zt_paged_attention(C.byref(p), None), 1, b"null tensor pointer")
    p.q = p.out = p.cu_seqlens_q = p.seq_lens = p.block_table = p.k_cache = p.v_cache = one
    p.q_stride[:], p.out_stride[:] = (8 * 64, 64), (8 * 64 + 1, 64)
    refused(lib.zt_paged_attention(C.byref(p), None), 1, b"query and output must be 16-byte aligned")
    p.out_stride[:] = (8 * 64, 64)
    p.k_cache_stride[:], p.v_cache_stride[:] = (16 * 4 * 64, 4 * 64, 64), (16 * 4 * 64, 4 * 64, 4)
    refused(lib.zt_paged_attention(C.byref(p), None), 1, b"caches must be 16-byte aligned")
    p.v_cache_stride[:] = (16 * 4 * 64, 4 * 64, 64)
    assert lib.zt_paged_attention_workspace_bytes(C.byref(p)) == 0            # short contexts: nothing is divided and joined
    blocks, p.max_blocks = p.max_blocks, 1024
    refused(lib.zt_paged_attention(C.byref(p), None), 4, b"workspace of 0 bytes")
    assert lib.zt_paged_attention_workspace_bytes(C.byref(p)) >= 2 * 3 * 148 * 8 * 64 * 4     # two cut items of 8 rows per CTA
    p.max_blocks = blocks
    p.tokens = 0
    assert lib.zt_paged_attention(C.byref(p), None) == 0


def _worker(rank, world, port, results):
    """DecoderLayer on two ranks against the same at one rank: a prompt, a chunk and a decode step, the oracle and plain
    evaluations standing in for the CUDA ops."""
    for p in (ROOT / "zendnn-pytorch-plugin_b200", ROOT / "oracle", ROOT / "tests"):
        sys.path.insert(0, str(p))
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import zentorch_oracle as O
        from _util import make_int8_case
        from zentorch_b200 import tp
        from zentorch_b200.cache import PagedKVCache, rope_frequencies
        hidden, hq, hkv, d, inter = 128, 4, 2, 32, 256
        shapes = {"q": (hidden, hq * d), "k": (hidden, hkv * d), "v": (hidden, hkv * d), "o": (hq * d, hidden),
                  "gate": (hidden, inter), "up": (hidden, inter), "down": (inter, hidden)}
        full = {n: make_int8_case(1, k, o, seed=60 + i, x_dtype=torch.float32)[1:] for i, (n, (k, o)) in enumerate(shapes.items())}
        freq, factor = rope_frequencies(d)

        def layer(r, w):
            lin = tp.DecoderLayerLinears("int8", full, r, w, linear_fn=lambda x, *p: O.dynamic_qlinear(x.float(), *p))
            return tp.DecoderLayer(lin, hq, hkv, d, freq, factor, ops=PlainOps), \
                PagedKVCache(1, 20, 4, hkv // w, d, dtype=torch.float32, device="cpu", copy_pages=plain_copy_pages)
        (one, cache1), (many, cache2) = layer(0, 1), layer(rank, world)
        from _cache_ref import U
        U.setdefault(torch.float32, 2.0 ** -24)
        g = torch.Generator().manual_seed(5)
        for name in ("a", "b"):
            cache1.add(name)
            cache2.add(name)
        for new in ([("a", 5), ("b", 1)], [("b", 7)], [("a", 1), ("b", 1)]):
            s1, s2 = cache1.step(new), cache2.step(new)
            x = torch.randn(s1.tokens, hidden, generator=g)
            y1, y2 = one(x, cache1, 0, s1), many(x, cache2, 0, s2)
            err = float((y1 - y2).abs().max() / y1.abs().max())
            assert err < 5e-2, f"sharded layer off by {err}"        # row-parallel int8 scales, as for the linears alone
        with_heads = cache1.keys(0)[:, :, rank * hkv // world:(rank + 1) * hkv // world]
        assert torch.allclose(with_heads, cache2.keys(0), atol=1e-5)      # column-parallel projections are exact
        results[rank] = "ok"
    except Exception as e:
        results[rank] = f"{type(e).__name__}: {e}"
    finally:
        dist.destroy_process_group()


def test_decoder_layer_with_attention_two_gloo_ranks(zt):
    port = 33500 + (os.getpid() % 2000)
    results = mp.Manager().dict()
    mp.spawn(_worker, args=(2, port, results), nprocs=2, join=True)
    assert dict(results) == {0: "ok", 1: "ok"}, dict(results)


def test_decoder_layer_refuses_heads_that_do_not_divide(zt):
    from zentorch_b200 import tp

    class Lin:
        world = 2
    with pytest.raises(ValueError, match="do not divide"):
        tp.DecoderLayer(Lin(), 8, 1, 64, torch.ones(32))
    with pytest.raises(ValueError, match="do not divide"):
        tp.DecoderLayer(Lin(), 6, 4, 64, torch.ones(32))
