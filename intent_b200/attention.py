"""The attention half of a transformer layer for serving, on a paged cache.

``PagedKVCache`` keeps the keys and values of many sequences in pages, of 16-bit elements or in 4 bits, and makes, for every step
of new tokens, the tensors that the attention programs take.  ``W4A16Attention`` chains the int4 projection to queries, keys
and values, the norms and the rotation with the append (``paged_kv_append``), the attention over the pages
(``paged_decode_attention`` where every sequence has one new token, ``paged_attention`` otherwise) and the int4 output
projection; with ``cache_bits=4`` the programs for a cache in 4 bits take their places.  Everything runs on the current
stream; no step reads a device value back to the host.

    cache = PagedKVCache(layers=2, pages=1024, kv_heads=8, head_dim=128)
    layer = W4A16Attention(hidden=4096, heads=32, kv_heads=8, head_dim=128)
    rotary = rotary_table(32768, 128, device="cuda")
    step = cache.step({"a": 700, "b": 45})                  # two prompts: their tokens' rows in this order
    y = layer.forward(x, weights, rotary, *cache.layer(0), step)
    step = cache.step({"a": 1, "b": 1})                     # a token each
    ...
    cache.release("a")

    cache = PagedKVCache(layers=2, pages=4096, kv_heads=8, head_dim=128, bits=4, group_size=64)     # the same calls
    layer = W4A16Attention(hidden=4096, heads=32, kv_heads=8, head_dim=128, cache_bits=4, cache_group=64)
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, NamedTuple

from . import dtypes, programs
from .compiler import compile as _compile
from .targets import B200Target


def rotary_table(positions: int, rotary_dim: int, *, base: float = 10000.0, device=None):
    """[positions, rotary_dim] f32: row p holds cos and then sin of p * base^(-2 i / rotary_dim), worked out in 64 bits
    (on the CPU where no device is given)."""
    import torch

    if positions <= 0 or rotary_dim <= 0 or rotary_dim % 16:
        raise ValueError("positions must be positive and rotary_dim a positive multiple of 16")
    place = torch.arange(positions, dtype=torch.float64, device=device)[:, None]
    angle = place * base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


@dataclass(frozen=True)
class AttentionStep:
    """What the attention programs need to know about a step of new tokens: the same for all layers."""

    positions: Any        # [T] i32, of every new token in its sequence
    slots: Any            # [T] i64, its place in the cache
    page_table: Any       # [B, W] i32
    query_offsets: Any    # [B + 1] i32, the sequences' rows
    kv_lengths: Any       # [B] i32, the new tokens among them
    single: bool          # every sequence has one new token
    longest: int = 0      # positions end here: tokens of the longest sequence that has new ones


class QuantisedPages(NamedTuple):
    """Keys or values of one layer in 4 bits."""

    codes: Any            # [pages, kv_heads, page_size, head_dim / 2] u8
    scales: Any           # [pages, kv_heads, page_size, 2 * head_dim / group_size]: scale and minimum of every group


class PagedKVCache:
    """Keys and values of all layers in pages of ``page_size`` tokens, and which pages a sequence has.  A sequence is a
    name of the caller's; it begins with its first step and ends with :meth:`release`.

    ``bits=4``: groups of ``group_size`` elements of a head are held as codes of 4 bits with a scale and a minimum (4.5 bits an
    element with groups of 64); ``k`` and ``v`` hold the codes, ``k_scales`` and ``v_scales`` the rest."""

    def __init__(self, *, layers: int, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, act_dtype="bf16",
                 device=None, bits: int = 16, group_size: int = 64):
        import torch

        if min(layers, pages, kv_heads) <= 0:
            raise ValueError("layers, pages and kv_heads must be positive")
        if head_dim not in (64, 128):
            raise ValueError(f"heads must have 64 or 128 elements, got {head_dim}")
        if not 16 <= page_size <= 256 or page_size & (page_size - 1):
            raise ValueError(f"a page must hold a power of two from 16 to 256 tokens, got {page_size}")
        if bits not in (4, 16):
            raise ValueError(f"elements are held in 4 or 16 bits, not {bits}")
        if bits == 4 and (group_size not in (32, 64, 128) or group_size > head_dim):
            raise ValueError(f"groups must have 32, 64 or 128 elements, up to {head_dim}, got {group_size}")
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        shape = (layers, pages, kv_heads, page_size)
        dtype = dtypes.torch_dtype(dtypes.dtype(act_dtype))
        self.bits, self.group_size, self.act_dtype = bits, group_size if bits == 4 else None, act_dtype
        if bits == 4:
            self.k, self.v = (torch.empty((*shape, head_dim // 2), dtype=torch.uint8, device=device) for _ in range(2))
            self.k_scales, self.v_scales = (torch.empty((*shape, 2 * head_dim // group_size), dtype=dtype, device=device)
                                            for _ in range(2))
            self._reader = None
        else:
            self.k, self.v = (torch.empty((*shape, head_dim), dtype=dtype, device=device) for _ in range(2))
        self.page_size = page_size
        self._free = list(range(pages - 1, -1, -1))
        self._pages: dict = {}          # sequence -> its pages
        self._lengths: dict = {}        # sequence -> its tokens

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence) -> int:
        """Tokens of a sequence, 0 for one that has not begun."""
        return self._lengths.get(sequence, 0)

    def layer(self, index: int):
        """Keys and values of one layer: [pages, kv_heads, page_size, head_dim] each, or :class:`QuantisedPages`."""
        if self.bits == 4:
            return QuantisedPages(self.k[index], self.k_scales[index]), QuantisedPages(self.v[index], self.v_scales[index])
        return self.k[index], self.v[index]

    def read(self, index: int, sequence, start: int = 0, stop: int | None = None):
        """Keys and values of one layer of a sequence's tokens from ``start`` to ``stop`` (its end), [tokens, kv_heads, head_dim]
        each, in 16 bits."""
        import torch

        if sequence not in self._lengths:
            raise KeyError(sequence)
        length = self._lengths[sequence]
        stop = length if stop is None else stop
        if not 0 <= start <= stop <= length:
            raise ValueError(f"the sequence has {length} tokens, not those from {start} to {stop}")
        place, size = torch.arange(start, stop, device="cpu"), self.page_size
        slots = torch.tensor(self._pages[sequence], dtype=torch.int64, device="cpu")[place // size] * size + place % size
        device = self.k.device
        if device.type == "cuda":
            slots = slots.pin_memory().to(device, non_blocking=True)
        k, v = self.layer(index)
        if self.bits == 16:
            return tuple(cache[slots // size, :, slots % size] for cache in (k, v))
        if self._reader is None:
            self._reader = _compile(programs.paged_kv_read_int4, target=B200Target(device.index),
                                    constexprs={"ACT_DTYPE": self.act_dtype, "GROUP_SIZE": self.group_size})
        return self._reader.run(slots, *k, *v)

    def step(self, new_tokens: dict) -> AttentionStep:
        """Room for so many new tokens of each sequence, and where they go.  Where there are not enough pages left,
        MemoryError; a step that fails, in this way or another, changes nothing."""
        import numpy as np
        import torch

        names, counts = list(new_tokens), [int(n) for n in new_tokens.values()]
        if not names or min(counts) < 0:
            raise ValueError("a step needs sequences, and no fewer than 0 new tokens of each")
        size = self.page_size
        lengths = [self.length(name) + n for name, n in zip(names, counts)]
        missing = [-(-length // size) - len(self._pages.get(name, ())) for name, length in zip(names, lengths)]
        if sum(missing) > len(self._free):
            raise MemoryError(f"{sum(missing)} pages are needed and {len(self._free)} are free")
        pages, free = [], len(self._free)
        for name, more in zip(names, missing):
            pages.append(self._pages.get(name, []) + self._free[free - more:free][::-1])
            free -= more
        tokens, batch = sum(counts), len(names)
        width = max(1, max(-(-length // size) for length in lengths))
        words = np.zeros(tokens + batch * width + 2 * batch + 1, dtype=np.int32)
        positions, table, offsets, ends = np.split(words, np.cumsum([tokens, batch * width, batch + 1]))
        slots = np.empty(tokens, dtype=np.int64)
        table = table.reshape(batch, width)
        table[:] = -1
        at = 0
        for row, (count, length) in enumerate(zip(counts, lengths)):
            held = np.asarray(pages[row], dtype=np.int64)
            table[row, :len(held)] = held
            place = np.arange(length - count, length)
            positions[at:at + count] = place
            slots[at:at + count] = held[place // size] * size + place % size
            at += count
            offsets[row + 1] = at
            ends[row] = length
        device = self.k.device
        copies = [torch.from_numpy(words), torch.from_numpy(slots)]
        if device.type == "cuda":        # (the allocator of pinned memory waits for copies under way before it gives it again)
            copies = [c.pin_memory().to(device, non_blocking=True) for c in copies]
        parts = torch.split(copies[0], [tokens, batch * width, batch + 1, batch])
        step = AttentionStep(parts[0], copies[1], parts[1].view(batch, width), parts[2], parts[3], all(n == 1 for n in counts),
                             max((length for count, length in zip(counts, lengths) if count), default=0))
        del self._free[free:]
        self._pages.update(zip(names, pages))
        self._lengths.update(zip(names, lengths))
        return step

    def release(self, sequence) -> None:
        """Ends a sequence; its pages are free again (for steps that follow on the same stream)."""
        if sequence not in self._lengths:
            raise KeyError(sequence)
        self._free.extend(reversed(self._pages.pop(sequence)))
        del self._lengths[sequence]


@dataclass(frozen=True)
class AttentionWeights:
    """Static weights of one layer; packed and scales as ``weight_only_int4_matmul`` takes them."""

    qkv_packed: Any       # [hidden / 8, (heads + 2 kv_heads) * head_dim] i32: queries, keys, values
    qkv_scales: Any
    out_packed: Any       # [heads * head_dim / 8, hidden] i32
    out_scales: Any
    q_norm: Any = None    # [head_dim], with norm=True
    k_norm: Any = None


class W4A16Attention:
    """Attention of one layer with int4 group-quantised projections on one GPU."""

    def __init__(self, *, hidden: int, heads: int, kv_heads: int, head_dim: int, group_size: int = 128, zero_point=8,
                 act_dtype="bf16", norm: bool = True, eps: float = 1e-6, pairs: str = "halves", window: int = 0, scale=None,
                 target: B200Target | None = None, cache_bits: int = 16, cache_group: int = 64):
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
            raise ValueError(f"{heads} query heads do not share {kv_heads} key heads evenly")
        if cache_bits not in (4, 16):
            raise ValueError(f"a cache holds its elements in 4 or 16 bits, not {cache_bits}")
        self.hidden, self.heads, self.kv_heads, self.head_dim, self.norm = hidden, heads, kv_heads, head_dim, norm
        self.cache_bits = cache_bits

        def bind(definition, constexprs):
            return _compile(definition, target=target, constexprs={"ACT_DTYPE": act_dtype, **constexprs})

        self.project = bind(programs.weight_only_int4_matmul, {"GROUP_SIZE": group_size, "ZERO_POINT": zero_point})
        rotation, attention = {"NORM": norm, "EPS": eps, "PAIRS": pairs}, {"WINDOW": window, "SCALE": scale}
        if cache_bits == 4:
            group = {"GROUP_SIZE": cache_group}
            self.append = bind(programs.paged_kv_append_int4, {**rotation, **group})
            self.attend = bind(programs.paged_attention_int4, {**attention, **group})
            self.attend_single = bind(programs.paged_decode_attention_int4, {**attention, **group})
        else:
            self.append = bind(programs.paged_kv_append, rotation)
            self.attend = bind(programs.paged_attention, attention)
            self.attend_single = bind(programs.paged_decode_attention, attention)

    def forward(self, x, weights: AttentionWeights, rotary, k_cache, v_cache, step: AttentionStep):
        """x [T, hidden], the step's tokens in its order -> [T, hidden]; keys and values are stored in the caches, which are a
        layer of a :class:`PagedKVCache`."""
        tokens, heads = x.shape[0], self.heads + 2 * self.kv_heads
        if step.positions.shape[0] != tokens:
            raise ValueError(f"the step has {step.positions.shape[0]} tokens, x has {tokens}")
        if x.shape[1] != self.hidden:
            raise ValueError(f"x has {x.shape[1]} columns, not {self.hidden}")
        if weights.out_packed.shape[0] * 8 != self.heads * self.head_dim or weights.out_packed.shape[1] != self.hidden:
            raise ValueError(f"the output projection must be packed from [{self.heads * self.head_dim}, {self.hidden}]")
        if step.longest > rotary.shape[0]:      # (the keys of positions without an angle would be stored as NaN)
            raise ValueError(f"a sequence has {step.longest} tokens, the rotary table {rotary.shape[0]} positions")
        quantised = isinstance(k_cache, tuple)
        if quantised != (self.cache_bits == 4) or quantised != isinstance(v_cache, tuple):
            raise TypeError(f"the layer was made for a cache of {self.cache_bits} bits")
        caches = (*k_cache, *v_cache) if quantised else (k_cache, v_cache)
        qkv = self.project.run(x, weights.qkv_packed, weights.qkv_scales)
        if qkv.shape[1] != heads * self.head_dim:
            raise ValueError(f"the projection has {qkv.shape[1]} columns, not {heads * self.head_dim}")
        q, k, v = qkv.view(tokens, heads, self.head_dim).split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        norms = (weights.q_norm, weights.k_norm) if self.norm else ()
        q = self.append.run(q, k, v, step.positions, step.slots, rotary, *norms, *caches)
        if step.single:
            out = self.attend_single.run(q, *caches, step.page_table, step.kv_lengths)
        else:
            out = self.attend.run(q, *caches, step.page_table, step.query_offsets, step.kv_lengths)
        return self.project.run(out.view(tokens, self.heads * self.head_dim), weights.out_packed, weights.out_scales)

    def check(self) -> None:
        """Synchronise and raise if a bounded wait of a device kernel gave up in an earlier call."""
        for artifact in (self.project, self.append, self.attend, self.attend_single):
            artifact.check()
