"""Plain 64-bit evaluations of the rotary positions and the paged attention, with the bounds their kernels are held to."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative


def rope_ref(x, positions, inv_freq, factor, interleaved):
    """(result, bound on the fp32 arithmetic) of x [tokens, heads, d], both fp64 on the CPU."""
    x, rot = x.double().cpu(), 2 * inv_freq.numel()
    angle = positions.double().cpu()[:, None, None] * inv_freq.double().cpu()
    c, s = angle.cos() * factor, angle.sin() * factor
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    lo, hi, size = a * c - b * s, b * c + a * s, (a.abs() + b.abs()) * abs(factor)
    y, bound = x.clone(), torch.zeros_like(x)
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = lo, hi
        bound[..., 0:rot:2], bound[..., 1:rot:2] = size, size
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = lo, hi
        bound[..., :rot // 2], bound[..., rot // 2:rot] = size, size
    # angle: half a step of a remainder below half a turn, 2 pi 2^-26, and the sine's own error of about 2^-24; products and sum
    # three roundings of 2^-24: below 2^-21 together
    return y, bound * 2.0 ** -21


def assert_rope(got, x, positions, inv_freq, factor, interleaved, what=""):
    y, arith = rope_ref(x, positions, inv_freq, factor, interleaved)
    bound = y.abs() * U[got.dtype] + arith * (1 + U[got.dtype])
    if got.dtype == torch.float16:
        bound += 2.0 ** -25                       # half the spacing of its subnormals
    err = (got.double().cpu() - y).abs()
    assert bool((err <= bound).all()), f"{what}: off by up to {float((err / bound.clamp_min(1e-30)).max()):.2f} bounds"


def gather_rows(cache, table_row, length):
    """[length, heads, d] of one sequence, fp64 on the CPU."""
    page = cache.shape[1]
    n = -(-length // page) if length else 0
    raw = cache.view(torch.uint8) if cache.element_size() == 1 else cache
    rows = raw[table_row[:n].long()].flatten(0, 1)[:length] if n else raw[:0].flatten(0, 1)
    return (rows.view(cache.dtype) if cache.element_size() == 1 else rows).double().cpu()


def attention_ref(q, k_cache, v_cache, cu, lens, table, scale=None, causal=True, window=0, k_scale=None, v_scale=None):
    """(out, bound) of the whole batch.  The bound counts: the output's rounding (half a step of its type); the rounding of every
    probability to the type of the product (fp16 for an 8-bit cache); scores that are off by d, which moves probabilities and
    their sum by d each -- sums of up to 128 products in at most 8 accumulations of the tensor core that truncate (2^-23 each),
    and for an 8-bit cache query elements below 2^-25 of their row's largest -- ; the accumulation of the outputs over keys / 16
    steps, the additions of pieces and the exponential (64 steps of 2^-23)."""
    t, hq, d = q.shape
    hkv = k_cache.shape[2]
    g, scale = hq // hkv, d ** -0.5 if scale is None else scale
    u_out, u_p = U[q.dtype], 2.0 ** -11 if k_cache.element_size() == 1 else U[q.dtype]
    out, bound = torch.zeros(t, hq, d, dtype=torch.float64), torch.zeros(t, hq, d, dtype=torch.float64)
    cu, lens, table = cu.cpu().tolist(), lens.cpu().tolist(), table.to(k_cache.device)
    qd = q.double().cpu()
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        k, v = gather_rows(k_cache, table[b], length), gather_rows(v_cache, table[b], length)
        if k_scale is not None:
            k, v = k * k_scale.double().cpu()[:, None], v * v_scale.double().cpu()[:, None]
        pos, key = torch.arange(length - n, length)[:, None], torch.arange(length)[None, :]
        seen = torch.ones(n, length, dtype=torch.bool)
        if causal:
            seen &= key <= pos
        if window:
            seen &= key > pos - window
        for h in range(hq):
            qh, kh, vh = qd[cu[b]:cu[b + 1], h], k[:, h // g], v[:, h // g]
            s = (qh @ kh.t() * scale).masked_fill(~seen, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if length else s
            vis = torch.where(seen[..., None], vh[None], 0.0) if not torch.isfinite(vh).all() else None
            o = p @ vh if vis is None else torch.einsum("qk,qkd->qd", p, vis)
            a = p @ vh.abs().nan_to_num(0, 0, 0)
            size = (qh.abs() @ kh.abs().t() * scale).masked_fill(~seen, 0)
            off = size.amax(-1, keepdim=True) * 2.0 ** -20 if length else torch.zeros(n, 1)
            if k_cache.element_size() == 1 and length:
                off = off + qh.abs().amax(-1, keepdim=True) * kh.abs().sum(-1).amax() * scale * 2.0 ** -24
            out[cu[b]:cu[b + 1], h] = o
            bound[cu[b]:cu[b + 1], h] = u_out * o.abs() + a * (1 + u_out) * (u_p + 2 * off + (length / 16 + 64) * 2.0 ** -23)
    if q.dtype == torch.float16:
        bound += 2.0 ** -25
    return out, bound


def assert_attention(got, ref, bound, what=""):
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got.double().cpu() - ref).abs()
    worst = float((err / bound.clamp_min(1e-30)).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: off by {worst:.2f} bounds"


def make_batch(pairs, hq, hkv, d, page, dtype=torch.bfloat16, cache=None, seed=0, layout="plain", extra_pages=3, table_fill=None,
               tail=0, device="cuda"):
    """A ragged batch: `pairs` of (new tokens, keys).  Slots that belong to no key, and pages that belong to no sequence, hold NaN;
    table entries past a sequence's pages hold `table_fill` (default: ids far outside the cache)."""
    g = torch.Generator().manual_seed(seed)
    cache = cache or dtype
    per = [-(-kv // page) for _, kv in pairs]
    pages = sum(per) + extra_pages
    order = torch.randperm(pages, generator=g)
    nan = float("nan")
    e4m3 = cache == torch.float8_e4m3fn
    ks = vs = None
    full = torch.full((2, pages, page, hkv, d), nan)
    width = max(per, default=0) + 2
    table, at = torch.full((len(pairs), width), 2 ** 30 if table_fill is None else table_fill, dtype=torch.int32), 0
    for b, (_, kv) in enumerate(pairs):
        ids = order[at:at + per[b]]
        table[b, :per[b]] = ids.to(torch.int32)
        at += per[b]
        rows = torch.full((2, per[b] * page, hkv, d), nan)
        rows[:, :kv] = torch.randn(2, kv, hkv, d, generator=g)
        full[:, ids] = rows.view(2, per[b], page, hkv, d)
    if e4m3:
        ks, vs = (torch.rand(hkv, generator=g) * 0.02 + 0.01 for _ in range(2))
        full = torch.stack([(x / s[:, None]).clamp(-448, 448) for x, s in zip(full, (ks, vs))])
    full = full.to(cache)
    if layout == "joined":          # [pages, 2, page, heads, d]
        raw = full.view(torch.uint8) if e4m3 else full
        both = raw.transpose(0, 1).contiguous().to(device)
        kc, vc = (both[:, i].view(cache) if e4m3 else both[:, i] for i in (0, 1))
    elif layout == "heads":         # [pages, heads, page, d] in memory
        kc, vc = (x.transpose(1, 2).contiguous().to(device).transpose(1, 2) for x in (full.view(torch.uint8) if e4m3 else full))
        kc, vc = (x.view(cache) if e4m3 else x for x in (kc, vc))
    else:
        kc, vc = full[0].to(device), full[1].to(device)
    t = sum(n for n, _ in pairs) + tail
    qkv = (torch.randn(t, (hq + 2 * hkv) * d, generator=g) * 2).to(dtype).to(device)
    q = qkv[:, :hq * d].view(t, hq, d)                       # a view with the projection's row stride
    starts = [0]
    for n, _ in pairs:
        starts.append(starts[-1] + n)
    return dict(q=q, k_cache=kc, v_cache=vc, cu=torch.tensor(starts, dtype=torch.int32, device=device),
                lens=torch.tensor([kv for _, kv in pairs], dtype=torch.int32, device=device), table=table.to(device),
                k_scale=None if ks is None else ks.to(device), v_scale=None if vs is None else vs.to(device),
                max_q=max((n for n, _ in pairs), default=0))


class PlainOps:
    """The operators a decoder layer calls, evaluated plainly on the CPU (torch.ops.zentorch's names and arguments)."""

    @staticmethod
    def zentorch_rope_cache(query, key, value, positions, inv_freq, key_cache, value_cache, slot_mapping, k_scale=None, v_scale=None,
                            interleaved=False, attention_factor=1.0):
        q, k = (rope_ref(t, positions, inv_freq, attention_factor, interleaved)[0] for t in (query, key))
        page = key_cache.shape[1]
        live = slot_mapping >= 0
        at = slot_mapping[live]
        key_cache[at // page, at % page] = k[live].to(key_cache.dtype)
        value_cache[at // page, at % page] = value[live].to(value_cache.dtype)
        return q.to(query.dtype)

    @staticmethod
    def zentorch_paged_attention(query, key_cache, value_cache, cu_seqlens_q, seq_lens, block_table, max_query_len=None, scale=None,
                                 causal=True, window=0, k_scale=None, v_scale=None):
        return attention_ref(query, key_cache, value_cache, cu_seqlens_q, seq_lens, block_table, scale, causal, window)[0].to(query.dtype)


def plain_copy_pages(caches, src, dst):
    for c in caches:
        c[dst.long()] = c[src.long()]
