"""Performance cases of the cache held in 4 bits: the append that quantises keys and values, reading them back, and attention
over the pages for chunks of new tokens and for single tokens.

``listed()`` holds the fixed cases, ``draw`` gives further ones of the same ranges, ``prepare`` makes what a serving program has
in hand before the call (projection outputs, caches, page tables, the step's positions and slots), ``run`` is one pass: with
``own`` through the public programs, without it in elementary operations in 32 bits (64 for what is rounded to a code).
``exact`` is the definition in 64 bits.

A group of ``group`` consecutive elements of a head is held as codes n from 0 to 15 and two numbers of the 16-bit type, a scale
s and a minimum m: the value is m + s n.  Two codes share a byte, the even element in its low half.
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
POSITIONS = 1 << 17          # rows of the rotation table: the longest sequence served


def listed():
    return [
        # The next token of one sequence, stored and looked at again: the smallest call.
        {"name": "append_token", "kind": "append", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "group": 64, "rotary": 128, "pairs": "halves", "norm": True, "packed": True, "page": 64},
        # A decode step of 48 sequences, small heads, half of each rotated, neighbouring pairs, no norm.
        {"name": "append_step_d64", "kind": "append", "tokens": 48, "heads": 32, "kv_heads": 8, "dim": 64, "dtype": "f16",
         "group": 32, "rotary": 32, "pairs": "neighbours", "norm": False, "packed": False, "page": 16},
        # A long prompt.
        {"name": "append_prompt", "kind": "append", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "group": 64, "rotary": 128, "pairs": "halves", "norm": True, "packed": True, "page": 64},
        # A prefix of an odd length is handed to something that takes 16 bits.
        {"name": "read_prefix", "kind": "read", "tokens": 6001, "kv_heads": 8, "dim": 64, "dtype": "f16", "group": 32,
         "page": 16},
        # Many sequences leave the cache at once.
        {"name": "read_many", "kind": "read", "tokens": 65536, "kv_heads": 8, "dim": 128, "dtype": "bf16", "group": 128,
         "page": 64},
        # One sequence's next token over a short history: latency.
        {"name": "decode_one", "kind": "decode", "batch": 1, "longest": 2000, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "group": 64, "page": 64, "window": 0},
        # A decode step of 64 sequences with histories of all lengths up to 8192.
        {"name": "decode_batch", "kind": "decode", "batch": 64, "longest": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "group": 64, "page": 64, "window": 0},
        # Many short histories, as many key heads as query heads, small pages, heads and groups.
        {"name": "decode_many_d64", "kind": "decode", "batch": 200, "longest": 2048, "heads": 16, "kv_heads": 16, "dim": 64,
         "dtype": "f16", "group": 32, "page": 16, "window": 0},
        # A few very long histories with few key heads: one sequence has to be shared by many multiprocessors.
        {"name": "decode_long", "kind": "decode", "batch": 4, "longest": 131072, "heads": 32, "kv_heads": 4, "dim": 128,
         "dtype": "bf16", "group": 128, "page": 128, "window": 0},
        # A short question at the end of a history: few rows, the cache counts.
        {"name": "chunk_short", "kind": "chunk", "batch": 1, "chunk": 33, "singles": 0, "longest": 8000, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "group": 64, "page": 64, "window": 0},
        # A chunk of a long prompt, the largest contraction.
        {"name": "chunk_prompt", "kind": "chunk", "batch": 1, "chunk": 4096, "singles": 0, "longest": 16384, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "group": 32, "page": 64, "window": 0},
        # A mixed step: chunks of prompts beside sequences that decode one token, with a sliding window, small heads.
        {"name": "chunk_mixed_d64", "kind": "chunk", "batch": 24, "chunk": 1000, "singles": 20, "longest": 6000, "heads": 32,
         "kv_heads": 4, "dim": 64, "dtype": "f16", "group": 64, "page": 32, "window": 2048},
    ]


def _size(rng, low, high):
    """A size between ``low`` and ``high``, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "decode", "decode", "chunk", "chunk"])
    heads, kv_heads = rng.choice([(32, 8), (32, 4), (16, 16), (28, 4), (8, 1), (40, 8), (64, 8)])
    dim = rng.choice([64, 128])
    case = {"kind": kind, "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(["f16", "bf16"]),
            "group": rng.choice([32, 64, dim]), "page": rng.choice([16, 32, 64, 128])}
    if kind == "read":
        return {**case, "tokens": _size(rng, 1, 65536 * 8 // max(kv_heads, 8))}
    case["heads"] = heads
    if kind == "append":
        return {**case, "tokens": _size(rng, 1, 8192 * 32 // max(heads, 32)), "rotary": rng.choice([32, 64, dim]),
                "pairs": rng.choice(["halves", "neighbours"]), "norm": rng.random() < 0.6, "packed": rng.random() < 0.7}
    case["window"] = rng.choice([0, 0, 0, _size(rng, 16, 4096)])
    if kind == "decode":
        batch = _size(rng, 1, 256)
        most = min(POSITIONS, (1 << 29) // (batch * kv_heads * dim))             # what the largest listed ones hold
        return {**case, "batch": batch, "longest": _size(rng, 16, most)}
    chunk = _size(rng, 1, 4096)
    batch = _size(rng, 1, 32)
    longest = _size(rng, max(chunk, 16), 16384)
    limit = 4096 * 16384 * 32                          # scores of the largest listed one
    batch = max(1, min(batch, limit // (chunk * longest * heads)))
    while chunk * longest * heads * batch > limit:     # one sequence of many heads
        chunk = max(1, chunk // 2)
    return {**case, "batch": batch, "chunk": chunk, "singles": rng.randint(0, batch - 1), "longest": longest}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Cache lengths (the new tokens among them) and numbers of new tokens, spread by the golden ratio: the sequence
    with the longest history first, every length between one page and it behind."""
    B, longest = case["batch"], case["longest"]
    chunk = case.get("chunk", 1)
    lengths, counts = [], []
    for b in range(B):
        part = (b * 0.6180339887498949) % 1.0
        n = 1 if b >= B - case.get("singles", 0) else max(1, round(chunk * (1 - 0.5 * part)))
        lengths.append(max(n, round(longest * (1 - 0.95 * part))))
        counts.append(n)
    return lengths, counts


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    device = _device()
    g = torch.Generator(device=device).manual_seed(seed)
    dtype, D, HK, page = DTYPES[case["dtype"]], case["dim"], case["kv_heads"], case["page"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device, dtype=torch.float32)

    def filled(pages, offset):
        """A cache of ``pages`` pages of normal numbers, around an ``offset`` of its own in every channel."""
        codes = torch.empty((pages, HK, page, D // 2), dtype=torch.uint8, device=device)
        scales = torch.empty((pages, HK, page, 2 * D // case["group"]), dtype=dtype, device=device)
        channels = offset * normal(HK, 1, D)
        some = max(1, (1 << 25) // (HK * page * D))
        for first in range(0, pages, some):
            n = min(some, pages - first)
            codes[first:first + n], scales[first:first + n] = _quantise(normal(n, HK, page, D) + channels, case["group"], dtype)
        return codes, scales

    state = {"case": case, "dtype": dtype}
    if case["kind"] in ("append", "read"):
        T = case["tokens"]
        pages = -(-2 * T // page) + 1        # twice the tokens: what is there already stays
        order = torch.randperm(pages, generator=g, device=device)[:-(-T // page)]
        at = torch.arange(T, device=device)
        state.update(slots=order[at // page] * page + at % page, k_cache=filled(pages, 0.5), v_cache=filled(pages, 0.0))
        if case["kind"] == "read":
            return state
        HQ, R = case["heads"], case["rotary"]
        if case["packed"]:                   # slices of the projection's output
            qkv = normal(T, HQ + 2 * HK, D).to(dtype)
            q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
        else:
            q, k, v = normal(T, HQ, D).to(dtype), normal(T, HK, D).to(dtype), normal(T, HK, D).to(dtype)
        angle = torch.arange(POSITIONS, device=device, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, R, 2, device=device, dtype=torch.float64) / R)
        start = torch.randint(0, POSITIONS - T + 1, (1,), generator=g, device=device)
        state.update(q=q, k=k, v=v, rotary=torch.cat([angle.cos(), angle.sin()], 1).float(),
                     positions=(start + torch.arange(T, device=device)).to(torch.int32),
                     weights=((1 + 0.1 * normal(2, D)).to(dtype).unbind(0) if case["norm"] else ()))
        return state

    lengths, counts = _lengths(case)
    width = -(-max(lengths) // page)
    used = [-(-n // page) for n in lengths]
    pages = sum(used)
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    held = torch.arange(width, device=device)[None] < torch.tensor(used, device=device)[:, None]
    table = torch.zeros((len(used), width), dtype=torch.int32, device=device)
    table[held] = order
    offsets = torch.tensor([0] + counts, device=device).cumsum(0).to(torch.int32)
    state.update(q=normal(sum(counts), case["heads"], D).to(dtype), k_cache=filled(pages, 0.5), v_cache=filled(pages, 0.0),
                 page_table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device=device), offsets=offsets,
                 most=max(counts), width=width)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------
@lru_cache(maxsize=None)
def _artifact(name, dtype, group, constants=()):
    import intent_b200 as ib

    return ib.compile(getattr(ib.programs, name), constexprs={"ACT_DTYPE": dtype, "GROUP_SIZE": group, **dict(constants)})


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        s, dtype, group = state, case["dtype"], case["group"]
        caches = (*s["k_cache"], *s["v_cache"])
        if kind in ("append", "read"):
            read = _artifact("paged_kv_read_int4", dtype, group)
            if kind == "read":
                return read.run(s["slots"], *caches)
            append = _artifact("paged_kv_append_int4", dtype, group,
                               (("NORM", case["norm"]), ("EPS", EPS), ("PAIRS", case["pairs"])))
            q = append.run(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rotary"], *s["weights"], *caches)
            return q, *read.run(s["slots"], *caches)
        if kind == "decode":
            attend = _artifact("paged_decode_attention_int4", dtype, group, (("WINDOW", case["window"]),))
            return attend.run(s["q"], *caches, s["page_table"], s["lengths"])
        attend = _artifact("paged_attention_int4", dtype, group, (("WINDOW", case["window"]),))
        return attend.run(s["q"], *caches, s["page_table"], s["offsets"], s["lengths"])
    if kind == "read":
        return _stored(state, "k_cache"), _stored(state, "v_cache")
    if kind == "append":
        weights = state["weights"] or (None, None)
        q = _rotate(state, state["q"].float(), weights[0]).to(state["dtype"])
        page, inside = state["slots"] // case["page"], state["slots"] % case["page"]
        for name, rows in (("k_cache", _rotate(state, state["k"].double(), weights[1])), ("v_cache", state["v"].double())):
            codes, scales = _quantise(rows, case["group"], state["dtype"])
            state[name][0][page, :, inside] = codes
            state[name][1][page, :, inside] = scales
        return q, _stored(state, "k_cache"), _stored(state, "v_cache")
    return _attend(state)


def _quantise(x, group, dtype):
    """Rows [..., D] -> codes [..., D / 2] and scales [..., 2 D / group]."""
    y = x.unflatten(-1, (-1, group))
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    scales = torch.cat([high / 15 - low / 15, low], -1).to(dtype)
    s, m = scales.to(x.dtype).split(1, -1)
    n = torch.where(s == 0, 0.0, (y - m) / torch.where(s == 0, 1.0, s)).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return n[..., 0::2] | (n[..., 1::2] << 4), scales.flatten(-2)


def _values(codes, scales, group):
    """Rows [..., D] in 32 bits."""
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, group))
    s, m = scales.float().unflatten(-1, (-1, 2)).split(1, -1)
    return (m + s * n).flatten(-2)


def _stored(state, name):
    page, inside = state["slots"] // state["case"]["page"], state["slots"] % state["case"]["page"]
    codes, scales = state[name]
    return _values(codes[page, :, inside], scales[page, :, inside], state["case"]["group"]).to(state["dtype"])


def _rotate(state, y, weight):
    case = state["case"]
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.to(y.dtype)
    R = case["rotary"]
    rows = state["rotary"][state["positions"].long()][:, None].to(y.dtype)
    cos, sin = rows[..., :R // 2], rows[..., R // 2:]
    turned = y[..., :R]
    if case["pairs"] == "halves":
        a, b = turned[..., :R // 2], turned[..., R // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., R:]], -1)


def _attend(state):
    """All sequences at once, padded to the longest: [batch, key heads, rows of the group, tokens]."""
    case, q = state["case"], state["q"]
    B, HQ, HK, D, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    n, length = state["most"], state["width"] * page
    lengths, offsets, table = state["lengths"].long(), state["offsets"].long(), state["page_table"].long()
    counts = offsets[1:] - offsets[:-1]
    at = torch.arange(n, device=q.device)
    real = at[None] < counts[:, None]                                   # [B, n]
    rows = torch.where(real, offsets[:-1, None] + at, 0)
    x = q[rows].float().view(B, n, HK, HQ // HK, D).permute(0, 2, 3, 1, 4).reshape(B, HK, -1, D)

    def gathered(cache):
        return _values(*(part[table].transpose(1, 2).reshape(B, HK, length, -1) for part in cache), case["group"])

    scores = torch.matmul(x, gathered(state["k_cache"]).transpose(2, 3)).view(B, HK, HQ // HK, n, length)
    scores *= D ** -0.5
    position = (lengths - counts)[:, None] + at                         # [B, n]
    token = torch.arange(length, device=q.device)
    hidden = token > position[:, :, None]
    if case["window"]:
        hidden |= token <= position[:, :, None] - case["window"]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(B, HK, -1, length), gathered(state["v_cache"])).view(B, HK, HQ // HK, n, D) / total
    return out.permute(0, 3, 1, 2, 4).reshape(B, n, HQ, D)[real].to(q.dtype)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def _meaning(cache, group):
    """What a cache's rows stand for."""
    codes, scales = cache
    parts = []
    for i in range(0, codes.shape[-1], group // 2):
        pair = scales[..., 4 * i // group:4 * i // group + 2].double()
        some = codes[..., i:i + group // 2].int()
        parts.append((torch.stack((some % 16, some // 16), -1).flatten(-2).double() * pair[..., :1]).add_(pair[..., 1:]))
    return torch.cat(parts, -1)


def _rounded(x, group, dtype):
    """What is left of the rows after they were held in 4 bits."""
    parts = []
    for i in range(0, x.shape[-1], group):
        some = x[..., i:i + group]
        least = some.min(-1, keepdim=True).values
        m = least.to(dtype).double()
        s = ((some.max(-1, keepdim=True).values - least) / 15).to(dtype).double()
        parts.append(m + s * torch.clamp(torch.round(torch.nan_to_num((some - m) / s, nan=0.0)), 0, 15))
    return torch.cat(parts, -1)


def exact(case, seed):
    state = prepare(case, seed)
    group, page = case["group"], case["page"]
    if case["kind"] == "read":
        return tuple(_meaning([part.transpose(1, 2).flatten(0, 1)[state["slots"]] for part in state[c]], group)
                     for c in ("k_cache", "v_cache"))
    if case["kind"] == "append":
        return (_exact_rotation(case, state, state["q"], 0),
                _rounded(_exact_rotation(case, state, state["k"], 1), group, state["dtype"]),
                _rounded(state["v"].double(), group, state["dtype"]))
    lengths, counts = _lengths(case)
    ratio = case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    first = 0
    for b, (length, n) in enumerate(zip(lengths, counts)):
        pages = state["page_table"][b, :-(-length // page)].long()
        for h in range(case["kv_heads"]):
            keys, values = (_meaning([part[pages, h] for part in state[c]], group).reshape(-1, case["dim"])[:length]
                            for c in ("k_cache", "v_cache"))
            for i in range(0, n, 1024):
                m = min(1024, n - i)
                position = torch.arange(length - n + i, length - n + i + m, device=keys.device)[:, None]
                token = torch.arange(length, device=keys.device)
                seen = (token <= position) & ((token > position - case["window"]) if case["window"] else True)
                x = state["q"][first + i:first + i + m, h * ratio:(h + 1) * ratio].double()
                logits = torch.einsum("mgd,ld->mgl", x, keys) / math.sqrt(case["dim"])
                logits = torch.where(seen[:, None], logits, -math.inf)
                weights = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
                out[first + i:first + i + m, h * ratio:(h + 1) * ratio] = torch.einsum("mgl,ld->mgd", weights, values)
        first += n
    return out


def _exact_rotation(case, state, x, which):
    y = x.double()
    if case["norm"]:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["dim"] + EPS) * state["weights"][which].double()
    R = case["rotary"]
    table = state["rotary"].double()[state["positions"].long()]
    turn = torch.complex(table[:, :R // 2], table[:, R // 2:])[:, None]
    first, second = ((slice(0, R // 2), slice(R // 2, R)) if case["pairs"] == "halves"
                     else (slice(0, R, 2), slice(1, R, 2)))
    z = torch.complex(y[..., first], y[..., second]) * turn
    out = y.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    D, HK = case["dim"], case["kv_heads"]
    row = D // 2 + 4 * D // case["group"]                 # a token's keys or values of a head, as they are held
    if case["kind"] == "read":
        return {"bytes": float(case["tokens"] * (2 * HK * (row + 2 * D) + 8)), "flops": float(4 * case["tokens"] * HK * D)}
    HQ = case["heads"]
    if case["kind"] == "append":
        T = case["tokens"]
        size = T * (2 * (HQ + 2 * HK) * D + case["rotary"] * 4 + 12       # rows in, angles, position and slot
                    + 2 * HQ * D + 2 * HK * row + 2 * HK * 2 * D)         # queries, what is held, what it stands for
        return {"bytes": float(size), "flops": float(T * ((HQ + HK) * (3 * case["rotary"] + (4 * D if case["norm"] else 0))
                                                          + 12 * HK * D))}
    lengths, counts = _lengths(case)
    window = case["window"]
    read = pairs = 0
    for length, n in zip(lengths, counts):
        first = length - n
        read += length - (max(0, first - window + 1) if window else 0)
        seen = n * first + n * (n + 1) // 2
        if window:
            over = max(0, length - window)                # the last query leaves that many tokens out
            kept = max(0, over - n)                       # those before it one fewer each
            seen -= (over * (over + 1) - kept * (kept + 1)) // 2
        pairs += seen
    rows = sum(counts)
    size = read * HK * 2 * row + rows * HQ * D * 4 + 4 * sum(-(-length // case["page"]) for length in lengths) + 8 * len(lengths)
    return {"bytes": float(size), "flops": float(4 * pairs * HQ * D)}
