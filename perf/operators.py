"""Performance cases of the operators between a decoder layer's linears: rotary positions, the paged key/value cache
and the attention that reads it.

A case names its operator -- ``rope`` (rotary positions of queries and keys), ``append`` (rotary positions, with the new keys
and values written to their slots of the cache), ``copy`` (pages of a cache copied for a fork or a compaction) or ``attn``
(attention of the new tokens of a batch over the paged cache) -- and its sizes and options.  ``own = True`` makes the calls of
``torch.ops.zentorch``; otherwise the same operators are computed with elementary torch operations in 32 bits.

The inputs are synthetic: queries N(0, 2), keys and values N(0, 1), cache pages handed out in random order, lengths drawn from
the case's ranges.  Queries, keys and values are views of a fused projection's output, as the layer has them.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}
_E4M3_MAX = 448.0


def _rope(name, tokens, hq, hkv, d, rot, dtype="bf16", interleaved=False, scaling="none", far=8192):
    return dict(name=name, op="rope", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, dtype=dtype, interleaved=interleaved,
                scaling=scaling, far=far)


def _append(name, tokens, hq, hkv, d, rot, page, dtype="bf16", cache="bf16", interleaved=False, scaling="none", far=8192):
    return dict(name=name, op="append", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, page=page, dtype=dtype, cache=cache,
                interleaved=interleaved, scaling=scaling, far=far)


def _copy(name, layers, pages, pairs, page, hkv, d, cache="bf16"):
    return dict(name=name, op="copy", layers=layers, pages=pages, pairs=pairs, page=page, hkv=hkv, d=d, cache=cache)


def _attn(name, batch, q, kv, hq, hkv, d, page, dtype="bf16", cache="bf16", causal=True, window=0, lens=1):
    return dict(name=name, op="attn", batch=batch, q_lo=q[0], q_hi=q[1], kv_lo=kv[0], kv_hi=kv[1], hq=hq, hkv=hkv, d=d,
                page=page, dtype=dtype, cache=cache, causal=causal, window=window, lens=lens)


def listed():
    return [
        # a decode step of 32 requests at far positions, frequencies stretched band by band: latency counts
        _rope("rope_decode", 32, 32, 8, 128, 128, scaling="llama3", far=131072),
        # prompt processing, half of the head rotated in interleaved pairs, keys of every head
        _rope("rope_prompt", 8192, 32, 32, 128, 64, interleaved=True, scaling="yarn", far=32768),
        # a decode step: the new tokens of 64 requests go to their slots
        _append("append_decode", 64, 32, 8, 128, 128, 16, scaling="llama3", far=131072),
        # a prompt of a large model goes to an 8-bit cache
        _append("append_prompt_e4m3", 8192, 64, 8, 128, 128, 64, cache="e4m3", scaling="linear", far=16384),
        # forked requests: the eight pages that are written next are copied in all layers
        _copy("copy_fork", 32, 256, 8, 16, 8, 128),
        # compaction of a cache: 512 pages move to the front in all layers
        _copy("copy_compact", 32, 1400, 512, 16, 8, 128),
        # one request, one token, a short context: the smallest call
        _attn("attn_decode_one", 1, (1, 1), (700, 700), 32, 8, 128, 16),
        # a decode batch with ragged contexts
        _attn("attn_decode_batch", 64, (1, 1), (500, 8000), 32, 8, 128, 16),
        # long documents in an 8-bit cache, one token each
        _attn("attn_decode_long", 4, (1, 1), (90000, 131072), 64, 8, 128, 64, cache="e4m3"),
        # chunked prompt processing: 512 tokens over a context of tens of thousands
        _attn("attn_chunk", 2, (512, 512), (16000, 32000), 32, 8, 128, 32),
        # a whole prompt: the largest call
        _attn("attn_prompt", 1, (8192, 8192), (8192, 8192), 32, 8, 128, 128),
        # a mixed batch whose sizes fit no tile: five heads to a key head, heads of 80, pages of 24 slots, a sliding window
        _attn("attn_mixed", 12, (1, 300), (40, 5000), 10, 2, 80, 24, dtype="f16", cache="f16", window=1000),
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], uniform over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi, max(lo, int(round(v / step)) * step))


def _heads(rng):
    hkv = rng.choice([1, 2, 4, 8, 8, 8])
    return hkv * rng.choice([1, 2, 4, 4, 5, 7, 8]), hkv


def draw(rng):
    op = rng.choice(["rope", "append", "copy", "attn", "attn", "attn", "attn"])
    hq, hkv = _heads(rng)
    d = rng.choice([64, 80, 96, 128, 128, 128])
    if op == "rope":
        c = _rope("", _log_int(rng, 1, 8192), hq, hkv, d, rng.choice([d, d, d // 2]), rng.choice(["bf16", "bf16", "f16", "f32"]),
                  rng.random() < 0.5, rng.choice(["none", "linear", "llama3", "yarn"]), _log_int(rng, 1000, 1000000))
    elif op == "append":
        dtype = rng.choice(["bf16", "bf16", "f16"])
        c = _append("", _log_int(rng, 1, 8192), hq, hkv, d, rng.choice([d, d, d // 2]), rng.choice([8, 16, 16, 24, 32, 64, 128]),
                    dtype, rng.choice([dtype, "e4m3"]), rng.random() < 0.5, rng.choice(["none", "linear", "llama3", "yarn"]),
                    _log_int(rng, 1000, 1000000))
    elif op == "copy":
        page, cache, layers = rng.choice([8, 16, 24, 32, 64]), rng.choice(["bf16", "f16", "e4m3"]), rng.choice([1, 2, 8, 28, 32])
        most = 512 * 32 * 16 * 8 * 128 * 2 // (layers * page * hkv * d * _BYTES[cache])
        pairs = _log_int(rng, 1, max(1, min(2000, most)))
        c = _copy("", layers, 2 * pairs + rng.randint(1, 100), pairs, page, hkv, d, cache)
    else:
        dtype = rng.choice(["bf16", "bf16", "f16"])
        cache = rng.choice([dtype, dtype, "e4m3"])
        page = rng.choice([8, 16, 16, 24, 32, 64, 128])
        window = rng.choice([0, 0, 0, _log_int(rng, 64, 4096)])
        kind = rng.choice(["decode", "decode", "chunk", "prompt", "mixed"])
        while True:
            kv_hi = _log_int(rng, 16, 131072 if kind == "decode" else 32768)
            kv_lo = rng.randint(max(1, kv_hi // 10), kv_hi)
            if kind == "decode":
                q = (1, rng.choice([1, 1, 1, 4]))
                batch = _log_int(rng, 1, 256)
            elif kind == "chunk":
                n = _log_int(rng, 16, 2048)
                q, batch = (n, n), _log_int(rng, 1, 8)
            elif kind == "prompt":
                q, batch = (kv_hi, kv_hi), _log_int(rng, 1, 8)
            else:
                q, batch = (1, _log_int(rng, 16, 1024)), _log_int(rng, 2, 64)
            c = _attn("", batch, q, (kv_lo, kv_hi), hq, hkv, d, page, dtype, cache, rng.random() < 0.9, window, rng.randrange(1 << 20))
            padded = batch * max(x for x, _ in _lengths(c))                 # the plain form pads queries and contexts
            contexts = batch * max(x for _, x in _lengths(c))
            w, top = work(c), work(_attn("", 1, (8192, 8192), (8192, 8192), 32, 8, 128, 128))
            if (w["flops"] <= top["flops"] and w["bytes"] <= 1.2e9 and contexts * hkv * d <= 1 << 30
                    and padded * hq * max(x for _, x in _lengths(c)) <= 1 << 31):
                break
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------------------------
def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _lengths(c):
    """(new tokens, tokens in the cache with them) of each sequence; of the case alone."""
    r = random.Random(c["lens"])
    got = []
    for _ in range(c["batch"]):
        kv = r.randint(c["kv_lo"], c["kv_hi"])
        got.append((min(kv, r.randint(c["q_lo"], c["q_hi"])), kv))
    return got


def _frequencies(c):
    """Angles per position of the rotated pairs, and the factor of the cosines and sines: theta^(-2i/rot), for long contexts
    divided by the stretch everywhere (linear) or in the slow bands alone (llama3, yarn)."""
    half, theta, stretch, before = c["rot"] // 2, 500000.0, 8.0, 8192.0
    f = theta ** (-torch.arange(half, dtype=torch.float64) / half)
    turns = before * f / (2 * math.pi)          # turns within the original context
    factor = 1.0
    if c["scaling"] == "linear":
        f = f / stretch
    elif c["scaling"] == "llama3":
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / stretch
    elif c["scaling"] == "yarn":
        keep = ((turns.log() - math.log(1.0)) / (math.log(32.0) - math.log(1.0))).clamp(0, 1)
        f = keep * f + (1 - keep) * f / stretch
        factor = 0.1 * math.log(stretch) + 1.0
    return f.float().cuda(), factor


def _qkv(g, c, tokens):
    """Views of a fused projection's output, [tokens, heads, d] each."""
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    x = _randn(g, tokens, (hq + 2 * hkv) * d).to(_DTYPES[c["dtype"]])
    q, k, v = x.split([hq * d, hkv * d, hkv * d], dim=1)
    return q.view(tokens, hq, d), k.view(tokens, hkv, d), v.view(tokens, hkv, d)


def _cache(g, c, pages):
    """Keys and values as pages of slots; an 8-bit cache holds them divided by a scale per head."""
    shape = (pages, c["page"], c["hkv"], c["d"])
    k, v = _randn(g, *shape), _randn(g, *shape)
    if c["cache"] != "e4m3":
        return k.to(_DTYPES[c["cache"]]), v.to(_DTYPES[c["cache"]]), None, None
    ks = torch.rand(c["hkv"], generator=g, device="cuda") * 0.01 + 0.01
    vs = torch.rand(c["hkv"], generator=g, device="cuda") * 0.01 + 0.01
    return _to_e4m3(k, ks), _to_e4m3(v, vs), ks, vs


def _to_e4m3(x, scale):
    """x [..., heads, d] over its scale per head, saturating."""
    return (x / scale.unsqueeze(1)).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)


def prepare(case, seed):
    c, g = case, _rng(seed)
    s = {"case": c}
    if c["op"] in ("rope", "append"):
        s["q"], s["k"], s["v"] = _qkv(g, c, c["tokens"])
        s["positions"] = torch.randint(0, c["far"], (c["tokens"],), generator=g, device="cuda")
        s["inv_freq"], s["factor"] = _frequencies(c)
        if c["op"] == "append":
            pages = -(-c["tokens"] // c["page"]) + 8
            s["kc"], s["vc"], s["ks"], s["vs"] = _cache(g, c, pages)
            s["slots"] = torch.randperm(pages * c["page"], generator=g, device="cuda")[:c["tokens"]].contiguous()
    elif c["op"] == "copy":
        shape = (c["layers"], c["pages"], 2, c["page"], c["hkv"], c["d"])
        s["caches"] = torch.empty(shape, dtype=_DTYPES[c["cache"]], device="cuda")
        for layer in s["caches"]:
            layer.copy_(_randn(g, *shape[1:]).clamp(-_E4M3_MAX, _E4M3_MAX))
        s["layers"] = list(s["caches"].unbind(0))     # a model keeps one cache per layer
        order = torch.randperm(c["pages"], generator=g, device="cuda").to(torch.int32)
        s["src"], s["dst"] = order[:c["pairs"]].contiguous(), order[c["pairs"]:2 * c["pairs"]].contiguous()
    else:
        lengths = _lengths(c)
        tokens = sum(n for n, _ in lengths)
        s["q"] = (_qkv(g, c, tokens)[0] * 2).contiguous()
        per = [-(-kv // c["page"]) for _, kv in lengths]
        pages, widest = sum(per) + 8, max(per)
        s["kc"], s["vc"], s["ks"], s["vs"] = _cache(g, c, pages)
        order, table, at = torch.randperm(pages, generator=g, device="cuda").to(torch.int32), [], 0
        for n in per:
            table.append(torch.nn.functional.pad(order[at:at + n], (0, widest - n)))
            at += n
        s["table"] = torch.stack(table)
        starts = [0]
        for n, _ in lengths:
            starts.append(starts[-1] + n)
        s["cu"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["lens"] = torch.tensor([kv for _, kv in lengths], dtype=torch.int32, device="cuda")
        s["max_q"], s["max_kv"] = max(n for n, _ in lengths), max(kv for _, kv in lengths)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------
def _cos_sin(s, dtype):
    angle = s["positions"].double().unsqueeze(1) * s["inv_freq"].double()
    return (angle.cos() * s["factor"]).to(dtype).unsqueeze(1), (angle.sin() * s["factor"]).to(dtype).unsqueeze(1)


def _rotate(x, cos, sin, rot, interleaved):
    """x [tokens, heads, d] in the type of cos and sin; the first `rot` of each head rotated."""
    x = x.to(cos.dtype)
    head, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = head.chunk(2, dim=-1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_rope(s):
    c = s["case"]
    cos, sin = _cos_sin(s, torch.float32)
    return [_rotate(s[n], cos, sin, c["rot"], c["interleaved"]).to(_DTYPES[c["dtype"]]) for n in ("q", "k")]


def _plain_append(s):
    c = s["case"]
    cos, sin = _cos_sin(s, torch.float32)
    q, k = (_rotate(s[n], cos, sin, c["rot"], c["interleaved"]) for n in ("q", "k"))
    v = s["v"].float()
    kc, vc = s["kc"].view(-1, c["hkv"], c["d"]), s["vc"].view(-1, c["hkv"], c["d"])
    if c["cache"] == "e4m3":
        k, v = _to_e4m3(k, s["ks"]), _to_e4m3(v, s["vs"])
        kc, vc = kc.view(torch.uint8), vc.view(torch.uint8)
        k, v = k.view(torch.uint8), v.view(torch.uint8)
    kc[s["slots"]] = k.to(kc.dtype)
    vc[s["slots"]] = v.to(vc.dtype)
    return [q.to(_DTYPES[c["dtype"]]), s["kc"], s["vc"]]


def _plain_copy(s):
    raw = s["caches"].view(torch.uint8)
    raw[:, s["dst"]] = raw[:, s["src"]]
    return [s["caches"]]


def _gather(cache, table, scale, max_kv, dtype):
    """[batch, max_kv, heads, d] of a paged cache."""
    raw = cache.view(torch.uint8) if cache.element_size() == 1 else cache
    x = raw[table.long()].flatten(1, 2)[:, :max_kv]
    x = (x.view(cache.dtype) if cache.element_size() == 1 else x).to(dtype)
    return x if scale is None else x * scale.to(dtype).unsqueeze(1)


def _plain_attn(s):
    c = s["case"]
    tokens, hkv, group, d = s["q"].shape[0], c["hkv"], c["hq"] // c["hkv"], c["d"]
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(c["batch"], device="cuda"), new, output_size=tokens)
    row = torch.arange(tokens, device="cuda") - s["cu"].long()[seq]
    q = torch.zeros(c["batch"], s["max_q"], hkv, group, d, device="cuda")
    q[seq, row] = s["q"].float().view(tokens, hkv, group, d)
    k = _gather(s["kc"], s["table"], s["ks"], s["max_kv"], torch.float32)
    v = _gather(s["vc"], s["table"], s["vs"], s["max_kv"], torch.float32)
    scores = torch.einsum("bqhgd,bkhd->bhgqk", q, k) * d ** -0.5
    at = torch.arange(s["max_kv"], device="cuda")
    where = (s["lens"].long() - new).unsqueeze(1) + torch.arange(s["max_q"], device="cuda")     # positions of the queries
    seen = (at < s["lens"].unsqueeze(1)).unsqueeze(1).expand(-1, s["max_q"], -1)
    if c["causal"]:
        seen = seen & (at <= where.unsqueeze(2))
    if c["window"] > 0:
        seen = seen & (at > where.unsqueeze(2) - c["window"])
    seen = seen.unsqueeze(1).unsqueeze(1)
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp_(scores.sub_(torch.where(top.isinf(), 0.0, top)))
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgqk,bkhd->bqhgd", p.div_(torch.where(total == 0, 1.0, total)), v)
    return o[seq, row].reshape(tokens, c["hq"], d).to(_DTYPES[c["dtype"]])


# ---- one pass --------------------------------------------------------------------------------------------
def _ops():
    where = str(Path.cwd() / "zendnn-pytorch-plugin_b200")   # the working folder is the repository's root
    if where not in sys.path:
        sys.path.insert(0, where)
    import zentorch_b200  # noqa: F401  (registers torch.ops.zentorch)
    return torch.ops.zentorch


def _own(s):
    c, ops = s["case"], _ops()
    if c["op"] == "rope":
        return list(ops.zentorch_rope(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=c["interleaved"],
                                      attention_factor=s["factor"]))
    if c["op"] == "append":
        q = ops.zentorch_rope_cache(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["kc"], s["vc"], s["slots"],
                                    s["ks"], s["vs"], interleaved=c["interleaved"], attention_factor=s["factor"])
        return [q, s["kc"], s["vc"]]
    if c["op"] == "copy":
        ops.zentorch_cache_copy_pages(s["layers"], s["src"], s["dst"])
        return [s["caches"]]
    return ops.zentorch_paged_attention(s["q"], s["kc"], s["vc"], s["cu"], s["lens"], s["table"], s["max_q"],
                                        causal=c["causal"], window=c["window"], k_scale=s["ks"], v_scale=s["vs"])


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "append": _plain_append, "copy": _plain_copy, "attn": _plain_attn}[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------
def _visible(c, n, kv):
    """(pairs of a new token and a key that it sees, keys that some new token sees) of one sequence."""
    pairs, first, last = 0, kv, 0
    for i in range(n):
        pos = kv - n + i
        hi = pos + 1 if c["causal"] else kv
        lo = max(0, pos - c["window"] + 1) if c["window"] > 0 else 0
        if hi > lo:
            pairs, first, last = pairs + hi - lo, min(first, lo), max(last, hi)
    return pairs, max(0, last - first)


def work(case):
    c = case
    if c["op"] == "copy":
        return {"bytes": 2 * c["layers"] * c["pairs"] * 2 * c["page"] * c["hkv"] * c["d"] * _BYTES[c["cache"]] + 8 * c["pairs"], "flops": 0}
    e = _BYTES[c["dtype"]]
    if c["op"] == "attn":
        pairs = keys = tokens = 0
        for n, kv in _lengths(c):
            p, seen = _visible(c, n, kv)
            pairs, keys, tokens = pairs + p, keys + seen, tokens + n
        return {"bytes": 2 * tokens * c["hq"] * c["d"] * e + 2 * keys * c["hkv"] * c["d"] * _BYTES[c["cache"]] + 4 * (keys // c["page"]),
                "flops": 4 * pairs * c["hq"] * c["d"]}
    t, row = c["tokens"], c["d"]
    rotated = t * (c["hq"] + c["hkv"]) * c["rot"] // 2
    if c["op"] == "rope":
        return {"bytes": 2 * t * (c["hq"] + c["hkv"]) * row * e + 8 * t, "flops": 6 * rotated}
    return {"bytes": t * row * (2 * c["hq"] * e + 2 * c["hkv"] * (e + _BYTES[c["cache"]])) + 16 * t, "flops": 6 * rotated}


# ---- the definition in 64 bits ------------------------------------------------------------------------------
def _exact_turn(x, positions, inv_freq, factor, rot, interleaved):
    """Pair (a, b) of each head times the rotation by positions * inv_freq, as a complex product."""
    angle = positions.double()[:, None, None] * inv_freq.double()
    turn = torch.polar(torch.full_like(angle, factor), angle)
    x = x.double()
    head = x[..., :rot]
    pairs = head.unflatten(-1, (-1, 2)) if interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat((z, x[..., rot:]), dim=-1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] in ("rope", "append"):
        q, k = (_exact_turn(s[n], s["positions"], s["inv_freq"], s["factor"], c["rot"], c["interleaved"]) for n in ("q", "k"))
        if c["op"] == "rope":
            return [q, k]
        v, kc, vc = s["v"].double(), s["kc"].double(), s["vc"].double()
        if c["cache"] == "e4m3":
            k = (k / s["ks"].double()[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
            v = (v / s["vs"].double()[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
        kc.view(-1, c["hkv"], c["d"])[s["slots"]] = k
        vc.view(-1, c["hkv"], c["d"])[s["slots"]] = v
        return [q, kc, vc]
    if c["op"] == "copy":
        raw = s["caches"].view(torch.uint8)
        for layer in raw:
            layer[s["dst"].long()] = layer[s["src"].long()].clone()
        return [s["caches"]]
    out, group = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), c["hq"] // c["hkv"]
    at = 0
    for b, (n, kv) in enumerate(_lengths(c)):
        pages = s["table"][b, :-(-kv // c["page"])].long()
        pos = torch.arange(kv - n, kv, device="cuda")[:, None]
        key = torch.arange(kv, device="cuda")[None, :]
        seen = torch.ones(n, kv, dtype=torch.bool, device="cuda")
        if c["causal"]:
            seen &= key <= pos
        if c["window"] > 0:
            seen &= key > pos - c["window"]
        for h in range(c["hkv"]):
            k, v = (t.select(2, h)[pages].flatten(0, 1)[:kv].double() if t.element_size() > 1 else
                    t.view(torch.uint8).select(2, h)[pages].flatten(0, 1)[:kv].view(t.dtype).double() for t in (s["kc"], s["vc"]))
            if s["ks"] is not None:
                k, v = k * s["ks"][h].double(), v * s["vs"][h].double()
            for j in range(h * group, (h + 1) * group):
                score = s["q"][at:at + n, j].double() @ k.t() / math.sqrt(c["d"])
                p = torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1)
                out[at:at + n, j] = torch.nan_to_num(p, nan=0.0) @ v
        at += n
    return out
