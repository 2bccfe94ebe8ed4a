"""A paged key/value cache for the layers of a decoder, and what its operators need to know about a step.

The cache of a layer is a pair of tensors [pages, page_size, kv_heads, head_dim]; a sequence owns a list of pages, which it may
share with the sequences it was forked from or into.  The bookkeeping is host code without any device synchronisation; pages are
copied by ``torch.ops.zentorch.zentorch_cache_copy_pages`` on the current stream, in all layers by one launch::

    cache = PagedKVCache(layers=32, pages=4096, page_size=16, kv_heads=8, head_dim=128, device="cuda")
    cache.add("a")
    step = cache.step([("a", 700)])            # a prompt of 700 tokens: allocates its pages
    ...                                        # every layer: zentorch_rope_cache, zentorch_paged_attention (tp.DecoderLayer)
    cache.fork("a", "b")                       # shares the pages; the last one is copied when either writes to it
    step = cache.step([("a", 1), ("b", 1)])    # a decode step of both

``rope_frequencies`` gives the angles per position that ``zentorch_rope`` and ``zentorch_rope_cache`` take.
"""
from __future__ import annotations

import math
import operator
from dataclasses import dataclass
from typing import Callable, Dict, Hashable, List, Optional, Sequence, Tuple

import torch


# ---- rotary frequencies -------------------------------------------------------------------------------
def rope_frequencies(rot_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None, device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq [rot_dim / 2] fp32, attention_factor) of rotary positions over ``rot_dim`` elements of a head.

    ``scaling`` stretches them for contexts longer than those of training, by its ``type`` (or ``rope_type``), as checkpoint
    configurations name them:

    * ``linear``: every angle divided by ``factor``;
    * ``ntk``: theta raised so that the slowest pair is divided by ``factor`` and the fastest is left;
    * ``llama3``: pairs with more than ``high_freq_factor`` turns in ``original_max_position_embeddings`` are left, those with
      fewer than ``low_freq_factor`` divided by ``factor``, those between blended linearly in their turns;
    * ``yarn``: the same blend, linear in the pair's number between those with ``beta_fast`` (32) and ``beta_slow`` (1) turns, and
      cosines and sines times ``attention_factor`` (0.1 ln factor + 1).
    """
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError(f"the rotated part of a head must be even, got {rot_dim}")
    half = rot_dim // 2
    number = torch.arange(half, dtype=torch.float64)
    scaling = dict(scaling or {})
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    known = ("default", "linear", "ntk", "llama3", "yarn")
    if kind not in known:
        raise ValueError(f"unknown rotary scaling {kind!r}, one of {known}")
    factor = float(scaling.get("factor", 1.0))
    if not factor >= 1.0:
        raise ValueError(f"the stretch factor must be at least 1, got {factor}")
    if kind == "ntk" and rot_dim > 2:
        theta = theta * factor ** (rot_dim / (rot_dim - 2))
    freq = theta ** (-number / max(half, 1))
    attention_factor = 1.0
    if kind == "linear":
        freq = freq / factor
    elif kind in ("llama3", "yarn"):
        context = float(scaling["original_max_position_embeddings"])
        if kind == "llama3":
            low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
            if not high > low:
                raise ValueError(f"high_freq_factor ({high}) must exceed low_freq_factor ({low})")
            keep = ((context * freq / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        else:
            fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

            def pair_with(turns):      # the (fractional) pair that makes so many turns in the context
                return half * math.log(context / (turns * 2 * math.pi)) / math.log(theta)

            first, last = max(math.floor(pair_with(fast)), 0), min(math.ceil(pair_with(slow)), rot_dim - 1)
            keep = 1 - ((number - first) / max(last - first, 1e-3)).clamp(0, 1)
            attention_factor = float(scaling.get("attention_factor") or 0.1 * math.log(factor) + 1.0)
        freq = keep * freq + (1 - keep) * freq / factor
    return freq.to(torch.float32).to(device if device is not None else "cpu"), attention_factor


# ---- the cache ----------------------------------------------------------------------------------------
@dataclass
class CacheStep:
    """One step of a batch, as the operators take it.  Tokens are the new tokens of the sequences, one sequence after another."""
    positions: torch.Tensor      # [tokens] int64
    slots: torch.Tensor          # [tokens] int64: page * page_size + offset of each new token
    cu_seqlens_q: torch.Tensor   # [sequences + 1] int32
    seq_lens: torch.Tensor       # [sequences] int32, with the new tokens
    block_table: torch.Tensor    # [sequences, pages of the longest] int32
    max_query_len: int

    @property
    def tokens(self) -> int:
        return self.positions.shape[0]


class _Sequence:
    __slots__ = ("pages", "length")

    def __init__(self, pages, length):
        self.pages, self.length = pages, length


class PagedKVCache:
    """Pages of keys and values for ``layers`` layers.

    ``dtype`` is that of the activations, or ``torch.float8_e4m3fn`` with ``k_scale`` / ``v_scale`` [layers, kv_heads] fp32 (ones
    if not given): stored values are divided by them.  ``zentorch_paged_attention`` reads bfloat16, float16 and float8_e4m3fn with
    heads of a multiple of 8 elements (16 in 8 bits) up to 128; other caches (float32, wider heads) can be filled and copied, for
    an attention of the caller's.  ``copy_pages(caches, src, dst)`` replaces the operator, for checks on a
    machine without a GPU.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16, device="cuda",
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                 copy_pages: Optional[Callable] = None):
        if min(layers, pages, page_size, kv_heads, head_dim) < 1:
            raise ValueError("layers, pages, page_size, kv_heads and head_dim must be positive")
        self.page_size, self.num_pages = int(page_size), int(pages)
        # keys and values of a page next to each other: a page is one block to copy
        self.layers = [torch.zeros((pages, 2, page_size, kv_heads, head_dim), dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype,
                                   device=device) for _ in range(layers)]
        self.device = self.layers[0].device      # with its index: the current device may change
        if dtype == torch.float8_e4m3fn:
            self.layers = [t.view(dtype) for t in self.layers]
            ones = torch.ones(layers, kv_heads, dtype=torch.float32, device=self.device)
            self.k_scale = ones if k_scale is None else k_scale.to(device=self.device, dtype=torch.float32).contiguous()
            self.v_scale = ones if v_scale is None else v_scale.to(device=self.device, dtype=torch.float32).contiguous()
            for name, t in (("k_scale", self.k_scale), ("v_scale", self.v_scale)):
                if t.shape != (layers, kv_heads):
                    raise ValueError(f"{name} must have shape {(layers, kv_heads)}, got {tuple(t.shape)}")
        else:
            if k_scale is not None or v_scale is not None:
                raise ValueError("scales belong to a float8_e4m3fn cache")
            self.k_scale = self.v_scale = None
        self._copy = copy_pages
        self._free: List[int] = list(range(pages - 1, -1, -1))      # a stack: the lowest ids go out first
        self._owners = [0] * pages
        self._sequences: Dict[Hashable, _Sequence] = {}

    # -- sequences
    def __contains__(self, name) -> bool:
        return name in self._sequences

    def length(self, name) -> int:
        return self._get(name).length

    def pages(self, name) -> Tuple[int, ...]:
        return tuple(self._get(name).pages)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _get(self, name) -> _Sequence:
        try:
            return self._sequences[name]
        except KeyError:
            raise KeyError(f"no sequence {name!r} in the cache") from None

    def _new_name(self, name):
        if name in self._sequences:
            raise ValueError(f"sequence {name!r} is in the cache already")

    def add(self, name) -> None:
        """An empty sequence."""
        self._new_name(name)
        self._sequences[name] = _Sequence([], 0)

    def fork(self, parent, child) -> None:
        """A sequence that starts as ``parent`` is now, sharing its pages."""
        self._new_name(child)
        s = self._get(parent)
        for page in s.pages:
            self._owners[page] += 1
        self._sequences[child] = _Sequence(list(s.pages), s.length)

    def free(self, name) -> None:
        """Drops a sequence; pages that no other one shares become free."""
        s = self._get(name)
        del self._sequences[name]
        self._release(s.pages)

    def truncate(self, name, length: int) -> None:
        """Takes back the tokens from ``length`` on (rejected drafts, an edited prompt)."""
        s, length = self._get(name), operator.index(length)
        if not 0 <= length <= s.length:
            raise ValueError(f"cannot cut a sequence of {s.length} tokens to {length}")
        keep = -(-length // self.page_size)
        self._release(s.pages[keep:])
        s.pages, s.length = s.pages[:keep], length

    def _release(self, pages: Sequence[int]) -> None:
        for page in reversed(pages):
            self._owners[page] -= 1
            if self._owners[page] == 0:
                self._free.append(page)

    # -- steps
    def step(self, new: Sequence[Tuple[Hashable, int]]) -> CacheStep:
        """Room for ``new`` tokens [(sequence, count), ...] and the tensors of the step.  A last page that others share is copied
        first (on the current stream).  Raises MemoryError, with nothing changed, when the free pages do not suffice."""
        new = [(name, operator.index(count)) for name, count in new]
        names = [n for n, _ in new]
        if len(set(names)) != len(names):
            raise ValueError("a sequence may appear once in a step")
        plan, need = [], 0
        shared = {}                                    # page -> sequences of this step that leave it
        for name, count in new:
            s = self._get(name)
            if count < 0:
                raise ValueError(f"negative number of new tokens for {name!r}")
            split = False
            if count > 0 and s.length % self.page_size:       # tokens go into the last page, which must be this sequence's own
                last = s.pages[-1]
                split = self._owners[last] - shared.get(last, 0) > 1
                if split:
                    shared[last] = shared.get(last, 0) + 1
            fresh = -(-(s.length + count) // self.page_size) - len(s.pages)
            need += fresh + split
            plan.append((s, count, fresh, split))
        if need > len(self._free):
            raise MemoryError(f"the step needs {need} pages, {len(self._free)} are free")
        src, dst, taken = [], [], 0
        for s, _, fresh, split in plan:
            if split:
                src.append(s.pages[-1])
                dst.append(self._free[-1 - taken])
            taken += split + fresh
        self._copy_pages(src, dst)                     # (where it raises, nothing has changed)
        positions, slots, starts, lens = [], [], [0], []
        for s, count, fresh, split in plan:
            if split:
                self._owners[s.pages[-1]] -= 1
                s.pages[-1] = self._take()
            s.pages.extend(self._take() for _ in range(fresh))
            t, end = s.length, s.length + count
            positions.extend(range(t, end))
            while t < end:                                    # page by page
                first = s.pages[t // self.page_size] * self.page_size + t % self.page_size
                here = min(end - t, self.page_size - t % self.page_size)
                slots.extend(range(first, first + here))
                t += here
            s.length = end
            starts.append(starts[-1] + count)
            lens.append(s.length)
        width = max((len(s.pages) for s, *_ in plan), default=0)
        table = [s.pages + [0] * (width - len(s.pages)) for s, *_ in plan]
        return CacheStep(self._tensor(positions, torch.int64), self._tensor(slots, torch.int64), self._tensor(starts, torch.int32),
                         self._tensor(lens, torch.int32), self._tensor(table, torch.int32).view(len(plan), width),
                         max((count for _, count, *_ in plan), default=0))

    def _take(self) -> int:
        page = self._free.pop()
        self._owners[page] = 1
        return page

    def _tensor(self, values, dtype) -> torch.Tensor:
        t = torch.tensor(values, dtype=dtype)
        return t if self.device.type == "cpu" else t.pin_memory().to(self.device, non_blocking=True)

    def compact(self) -> int:
        """Moves pages to the front of the cache, in all layers by one launch, and returns how many moved.  Afterwards the pages in
        use are 0 .. n - 1; tensors of earlier steps are out of date."""
        used = self.num_pages - len(self._free)
        holes = sorted(p for p in self._free if p < used)
        high = [p for p in range(used, self.num_pages) if self._owners[p]]
        moved = dict(zip(high, holes))
        self._copy_pages(list(moved), list(moved.values()))
        for old, page in moved.items():
            self._owners[page], self._owners[old] = self._owners[old], 0
        for s in self._sequences.values():
            s.pages = [moved.get(p, p) for p in s.pages]
        self._free = list(range(self.num_pages - 1, used - 1, -1))
        return len(moved)

    def _copy_pages(self, src: List[int], dst: List[int]) -> None:
        if not src:
            return
        fn = self._copy or torch.ops.zentorch.zentorch_cache_copy_pages
        fn(self.layers, self._tensor(src, torch.int32), self._tensor(dst, torch.int32))

    # -- layers
    def keys(self, layer: int) -> torch.Tensor:
        return self.layers[layer][:, 0]

    def values(self, layer: int) -> torch.Tensor:
        return self.layers[layer][:, 1]

    def scales(self, layer: int):
        """(k_scale, v_scale) of a layer, None where the cache is not 8-bit."""
        return (None, None) if self.k_scale is None else (self.k_scale[layer], self.v_scale[layer])
