"""zentorch_rope, zentorch_rope_cache and zentorch_cache_copy_pages against 64-bit evaluations; bounds in _cache_ref."""
import pytest
import torch

from _cache_ref import assert_rope, rope_ref

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(zt):
    assert torch.cuda.is_available() and zt.is_supported_device()
    return torch.ops.zentorch


def qkv(t, hq, hkv, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, (hq + 2 * hkv) * d, generator=g).to(dtype).cuda()
    q, k, v = x.split([hq * d, hkv * d, hkv * d], 1)
    return q.view(t, hq, d), k.view(t, hkv, d), v.view(t, hkv, d)


def freq(rot, theta=10000.0):
    return (theta ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / max(rot, 1))).float().cuda()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("t,hq,hkv,d,rot", [(1, 1, 1, 64, 64), (33, 8, 2, 128, 128), (5, 5, 1, 80, 32), (300, 3, 3, 96, 96), (7, 2, 1, 20, 6),
                                            (4, 4, 2, 256, 256), (3, 2, 2, 64, 0), (0, 4, 2, 64, 64), (9, 2, 1, 7, 2),
                                             (600, 128, 128, 128, 128), (40, 300, 200, 66, 64)])
def test_rope(ops, interleaved, dtype, t, hq, hkv, d, rot):
    q, k, _ = qkv(t, hq, hkv, d, dtype, seed=t)
    pos = torch.randint(0, 5000, (t,), generator=torch.Generator().manual_seed(1)).cuda()
    f = freq(rot)
    for p in (pos, pos.int()):
        qr, kr = ops.zentorch_rope(q, k, p, f, interleaved=interleaved, attention_factor=1.25)
        assert_rope(qr, q, pos, f, 1.25, interleaved, "query")
        assert_rope(kr, k, pos, f, 1.25, interleaved, "key")


def test_far_positions(ops):
    """Angles of positions up to the limit and below zero keep fp32 accuracy."""
    q, k, _ = qkv(6, 4, 2, 128, F32)
    pos = torch.tensor([0, 131071, 1000003, 2 ** 31 - 1, -5, -70001]).cuda()
    f = freq(128, 500000.0)
    qr, kr = ops.zentorch_rope(q, k, pos, f)
    assert_rope(qr, q, pos, f, 1.0, False)
    assert_rope(kr, k, pos, f, 1.0, False)


def test_unaligned_rows_and_head_major_inputs(ops):
    x = torch.randn(5, 3 * 64 + 1, device="cuda").to(BF16)[:, 1:].view(5, 3, 64)
    y = torch.randn(2, 5, 64, device="cuda").to(BF16).transpose(0, 1)
    pos, f = torch.arange(5, device="cuda") * 100, freq(64)
    qr, kr = ops.zentorch_rope(x, y, pos, f)
    assert_rope(qr, x, pos, f, 1.0, False)
    assert_rope(kr, y, pos, f, 1.0, False)
    z = torch.randn(64, 3, 5, device="cuda").to(BF16).permute(2, 1, 0)     # no unit stride along the head
    qr, _ = ops.zentorch_rope(z, y, pos, f, interleaved=True)
    assert_rope(qr, z, pos, f, 1.0, True)


def test_values_that_are_not_finite_stay_in_their_pairs(ops):
    q, k, _ = qkv(4, 2, 1, 64, BF16)
    pos, f = torch.arange(4).cuda() + 3, freq(64)
    clean, _ = ops.zentorch_rope(q, k, pos, f)
    q[1, 0, 5], q[2, 1, 40] = float("nan"), float("inf")
    got, _ = ops.zentorch_rope(q, k, pos, f)
    hit = torch.zeros(4, 2, 64, dtype=torch.bool, device="cuda")
    hit[1, 0, [5, 37]] = hit[2, 1, [8, 40]] = True
    assert not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], clean[~hit])


def caches(pages, page, hkv, d, cache, layout):
    def fill(*shape):
        return torch.full(shape, 3.0, device="cuda").to(cache)
    if layout == "joined":
        both = fill(pages, 2, page, hkv, d)
        return both[:, 0], both[:, 1]
    if layout == "heads":
        return fill(pages, hkv, page, d).transpose(1, 2), fill(pages, hkv, page, d).transpose(1, 2)
    return fill(pages, page, hkv, d), fill(pages, page, hkv, d)


@pytest.mark.parametrize("layout", ["plain", "joined", "heads"])
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, E4M3), (F16, E4M3), (F32, E4M3)])
@pytest.mark.parametrize("t,hq,hkv,d,rot,page,interleaved", [(1, 4, 2, 128, 128, 16, False), (50, 8, 2, 80, 40, 24, True),
                                                             (37, 3, 3, 64, 64, 1, False), (9, 2, 1, 20, 6, 8, True)])
def test_rope_cache(ops, layout, dtype, cache, t, hq, hkv, d, rot, page, interleaved):
    q, k, v = qkv(t, hq, hkv, d, dtype, seed=d)
    pages = -(-t // page) + 4
    kc, vc = caches(pages, page, hkv, d, cache, layout)
    g = torch.Generator().manual_seed(7)
    slots = torch.randperm(pages * page, generator=g)[:t]
    if t > 4:
        slots[3] = -1                                             # a padded token
    pos, f = torch.randint(0, 9000, (t,), generator=g).cuda(), freq(rot)
    ks = vs = None
    if cache == E4M3:
        ks, vs = torch.rand(hkv, generator=g).cuda() * 0.02 + 0.004, torch.rand(hkv, generator=g).cuda() * 0.02 + 0.004
    qr = ops.zentorch_rope_cache(q, k, v, pos, f, kc, vc, slots.cuda().int(), ks, vs, interleaved=interleaved)
    assert_rope(qr, q, pos, f, 1.0, interleaved)
    kr, arith = rope_ref(k, pos, f, 1.0, interleaved)
    rows_k, rows_v = (c.to(F32).cpu().double().reshape(pages * page, hkv, d) for c in (kc, vc))
    live = slots >= 0
    got_k, got_v = rows_k[slots[live]], rows_v[slots[live]]
    want_k, want_v, arith = kr[live], v.double().cpu()[live], arith[live]
    if cache == E4M3:
        want_k, want_v, arith = (x / s.double().cpu()[:, None] for x, s in ((want_k, ks), (want_v, vs), (arith, ks)))
        want_k, want_v = want_k.clamp(-448, 448), want_v.clamp(-448, 448)
        half = lambda x: (x.abs() * 2.0 ** -4).clamp_min(2.0 ** -10) * (1 + 2.0 ** -20)   # noqa: E731  subnormals 2^-9 apart
    else:
        u = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}[cache]
        half = lambda x: x.abs() * u + (2.0 ** -25 if cache == F16 else 0)                 # noqa: E731
    assert ((got_k - want_k).abs() <= half(want_k) + arith * 1.25).all()
    assert ((got_v - want_v).abs() <= (half(want_v) if cache == E4M3 else 0)).all()
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slots[live]] = False
    assert (rows_k[rest] == 3).all() and (rows_v[rest] == 3).all()


def test_e4m3_saturates_and_keeps_nan(ops):
    q, k, v = qkv(2, 1, 1, 64, BF16)
    v[0, 0, 0], v[0, 0, 1], v[1, 0, 0] = 1e6, -1e6, float("nan")
    kc, vc = caches(2, 4, 1, 64, E4M3, "plain")
    one = torch.ones(1, device="cuda")
    ops.zentorch_rope_cache(q, k, v, torch.arange(2).cuda(), freq(64), kc, vc, torch.tensor([1, 6]).cuda(), one, one)
    rows = vc.float().view(8, 64)
    assert rows[1, 0] == 448 and rows[1, 1] == -448 and rows[6, 0].isnan()


def test_cache_beyond_32_bits(ops):
    """Slots whose byte and element offsets do not fit 32 bits."""
    pages, page, hkv, d = 70000, 64, 8, 64                 # 2.3e9 elements each
    base = torch.empty(pages, page, hkv, d, dtype=E4M3, device="cuda")
    kc = vc = base
    q, k, v = qkv(3, 8, 8, 64, BF16)
    k = v
    one = torch.full((8,), 0.01, device="cuda")
    slots = torch.tensor([5, pages * page - 1, pages * page - 70], device="cuda")
    ops.zentorch_rope_cache(q, k, v, torch.zeros(3, dtype=torch.long, device="cuda"), freq(64), kc, vc, slots, one, one)
    want = (v.float() / 0.01).clamp(-448, 448).to(E4M3).float()
    assert torch.equal(base.view(torch.uint8).view(-1, 8, 64)[slots].view(E4M3).float(), want)
    out = ops.zentorch_paged_attention(v[1:2], base, base, torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                                       torch.tensor([1], dtype=torch.int32, device="cuda"),
                                       torch.tensor([[pages - 2]], dtype=torch.int32, device="cuda"), 1, k_scale=one, v_scale=one)
    first = base.view(torch.uint8)[pages - 2, 0].view(E4M3).float()
    if torch.isfinite(first).all():
        assert torch.allclose(out[0].float(), first * 0.01, rtol=2 ** -7, atol=1e-6)
    ops.zentorch_cache_copy_pages([base], torch.tensor([pages - 1], device="cuda"), torch.tensor([1], device="cuda"))
    assert torch.equal(base.view(torch.uint8)[1], base.view(torch.uint8)[pages - 1])


def test_slots_past_the_cache_are_reported(ops, zt):
    from zentorch_b200 import _capi
    q, k, v = qkv(3, 2, 1, 64, BF16)
    kc, vc = caches(2, 4, 1, 64, BF16, "plain")
    ops.zentorch_rope_cache(q, k, v, torch.arange(3).cuda(), freq(64), kc, vc, torch.tensor([0, 8, 2 ** 40]).cuda())
    assert _capi.poll_device_status(reset=True) == 106
    assert torch.equal(vc.view(8, 64)[0], v[0, 0]) and (vc.view(8, 64)[1:] == 3).all()


@pytest.mark.parametrize("dtype,shape", [(BF16, (9, 2, 16, 2, 64)), (E4M3, (9, 24, 3, 80)), (BF16, (9, 3, 1, 5)), (F32, (9, 33000))])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_copy_pages(ops, dtype, shape, index):
    g = torch.Generator().manual_seed(3)
    layers = [torch.randint(0, 100, shape, generator=g).to(dtype).cuda() for _ in range(70)]   # more than one launch holds
    before = [x.view(torch.uint8).clone() for x in layers]
    src, dst = torch.tensor([7, 0, -1, 7], dtype=index, device="cuda"), torch.tensor([1, 8, 3, 4], dtype=index, device="cuda")
    ops.zentorch_cache_copy_pages(layers, src, dst)
    for x, y in zip(layers, before):
        y[1], y[4], y[8] = y[7].clone(), y[7].clone(), y[0].clone()
        assert torch.equal(x.view(torch.uint8), y)


def test_copy_pages_of_views(ops):
    """One layer's pages within a buffer of all layers, and head-major pages."""
    both = torch.randn(6, 3, 8, 2, 64, device="cuda").to(BF16)
    want = both.clone()
    heads = torch.randn(6, 2, 8, 64, device="cuda").to(BF16)
    want_heads = heads.clone()
    i = torch.tensor([2, 3], device="cuda")
    ops.zentorch_cache_copy_pages([both[:, 1], heads.transpose(1, 2)], i, i - 2)
    want[:2, 1], want_heads[:2] = want[2:4, 1].clone(), want_heads[2:4].clone()
    assert torch.equal(both, want) and torch.equal(heads, want_heads)


def test_copy_pages_skips_caches_without_elements(ops):
    x = torch.arange(8 * 6, device="cuda").view(8, 6)
    y = x.clone()
    ops.zentorch_cache_copy_pages([x[:, :0], x], torch.tensor([5]).cuda(), torch.tensor([2]).cuda())
    y[2] = y[5]
    assert torch.equal(x, y)


def test_two_calls_at_once(ops):
    """Appends to different rows of one cache on two streams, while a third copies pages that neither touches."""
    kc, vc = caches(6, 4, 2, 64, BF16, "joined")
    f, pos = freq(64), torch.arange(4).cuda()
    src, dst = torch.tensor([4]).cuda(), torch.tensor([5]).cuda()
    batches = [qkv(4, 4, 2, 64, BF16, seed=s) for s in (1, 2)]
    slots = [torch.arange(4).cuda(), torch.arange(8, 12).cuda()]
    kc[4], vc[4] = 1.5, 2.5
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                outs[i] = ops.zentorch_rope_cache(*batches[i], pos, f, kc, vc, slots[i])
        with torch.cuda.stream(streams[2]):
            ops.zentorch_cache_copy_pages([kc, vc], src, dst)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert_rope(outs[i], batches[i][0], pos, f, 1.0, False)
        assert_rope(kc.reshape(24, 2, 64)[slots[i]], batches[i][1], pos, f, 1.0, False)
        assert torch.equal(vc.reshape(24, 2, 64)[slots[i]], batches[i][2])
    assert (kc[5] == 1.5).all() and (vc[5] == 2.5).all()


def test_copy_pages_past_the_cache_are_reported(ops, zt):
    from zentorch_b200 import _capi
    x = torch.randn(4, 64, device="cuda")
    y = x.clone()
    ops.zentorch_cache_copy_pages([x], torch.tensor([0, 4, 1]).cuda(), torch.tensor([7, 2, 3]).cuda())
    assert _capi.poll_device_status(reset=True) == 106
    y[3] = y[1]
    assert torch.equal(x, y)


def test_refusals(ops):
    q, k, v = qkv(3, 2, 1, 64, BF16)
    pos, f = torch.arange(3).cuda(), freq(64)
    kc, vc = caches(2, 4, 1, 64, BF16, "plain")

    def refused(match, call):
        with pytest.raises(RuntimeError, match=match):
            call()

    refused("dtype of the query", lambda: ops.zentorch_rope(q, k.float(), pos, f))
    refused("bfloat16, float16 or float32", lambda: ops.zentorch_rope(q.double(), k.double(), pos, f))
    refused("shape \\[3\\]", lambda: ops.zentorch_rope(q, k, pos[:2], f))
    refused("int32 or int64", lambda: ops.zentorch_rope(q, k, pos.float(), f))
    refused("rotates 128 elements", lambda: ops.zentorch_rope(q, k, pos, freq(128)))
    refused("1D float32", lambda: ops.zentorch_rope(q, k, pos, f.double()))
    refused("input's device", lambda: ops.zentorch_rope(q, k, pos.cpu(), f))
    many = torch.zeros(1, 2000, 67, dtype=BF16, device="cuda")
    refused("too many", lambda: ops.zentorch_rope(many, many, pos[:1], freq(64)))
    refused("shape and dtype of the key", lambda: ops.zentorch_rope_cache(q, k, v[:2], pos, f, kc, vc, pos))
    refused("caches must be", lambda: ops.zentorch_rope_cache(q, k, v, pos, f, kc.half(), vc.half(), pos))
    refused("needs k_scale", lambda: ops.zentorch_rope_cache(q, k, v, pos, f, kc.to(E4M3), vc.to(E4M3), pos))
    refused("hold an element twice", lambda: ops.zentorch_rope_cache(q, k, v, pos, f, kc[:1].expand_as(kc), vc, pos))
    refused("heads, the key", lambda: ops.zentorch_rope_cache(q, q, q, pos, f, kc, vc, pos))
    refused("one block of memory", lambda: ops.zentorch_cache_copy_pages([kc[..., :32]], pos[:1], pos[1:2]))
    refused("one number of pages", lambda: ops.zentorch_cache_copy_pages([kc, vc[:1]], pos[:1], pos[1:2]))
    refused("shape \\[1\\]", lambda: ops.zentorch_cache_copy_pages([kc], pos[:1], pos))


def test_other_stream_and_capture(ops):
    """The three run on the current stream and can be captured; a replay sees new inputs."""
    q, k, v = qkv(8, 4, 2, 64, BF16)
    kc, vc = caches(4, 4, 2, 64, BF16, "plain")
    pos, f, slots = torch.arange(8).cuda(), freq(64), torch.arange(8).cuda()
    src, dst = torch.tensor([0, 1]).cuda(), torch.tensor([2, 3]).cuda()
    s = torch.cuda.Stream()

    def step():
        out = ops.zentorch_rope_cache(q, k, v, pos, f, kc, vc, slots)
        ops.zentorch_cache_copy_pages([kc, vc], src, dst)
        return out
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    pos.add_(1000)
    v.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert_rope(out, q, pos, f, 1.0, False)
    assert torch.equal(vc.view(-1, 2, 64)[8:], v)
