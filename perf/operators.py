"""Performance cases of the attention programs: rotation and norms of queries and keys, the append to a paged cache,
and attention over the pages for chunks of new tokens and for single tokens.

``listed()`` holds the fixed cases, ``draw`` gives further ones of the same ranges, ``prepare`` makes what a serving
program has in hand before the call (projection outputs, caches, page tables, the step's positions and slots), ``run``
is one pass: with ``own`` through the public programs, without it in elementary operations in 32 bits.  ``exact`` is the
definition in 64 bits.
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
        # One token of one sequence through the norms and the rotation, without a cache: the smallest call.
        {"name": "rope_token", "kind": "rope", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "rotary": 128, "pairs": "halves", "norm": True, "packed": True},
        # A batch of prompts of an odd total length, small heads, half of each rotated, neighbouring pairs, no norm.
        {"name": "rope_prompt_d64", "kind": "rope", "tokens": 6001, "heads": 32, "kv_heads": 8, "dim": 64, "dtype": "f16",
         "rotary": 32, "pairs": "neighbours", "norm": False, "packed": False},
        # The append of a decode step of 64 sequences.
        {"name": "append_decode", "kind": "append", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "rotary": 128, "pairs": "halves", "norm": True, "packed": True, "page": 64},
        # The append of a long prompt.
        {"name": "append_prompt", "kind": "append", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "rotary": 128, "pairs": "halves", "norm": True, "packed": True, "page": 64},
        # One sequence's next token over a short history: latency.
        {"name": "decode_one", "kind": "decode", "batch": 1, "longest": 1000, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "page": 64, "window": 0},
        # A decode step of 64 sequences with histories of all lengths up to 8192.
        {"name": "decode_batch", "kind": "decode", "batch": 64, "longest": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "page": 64, "window": 0},
        # Many short histories, as many key heads as query heads, small pages and heads.
        {"name": "decode_many_d64", "kind": "decode", "batch": 200, "longest": 2048, "heads": 16, "kv_heads": 16, "dim": 64,
         "dtype": "f16", "page": 16, "window": 0},
        # A few very long histories with few key heads: one sequence has to be shared by many multiprocessors.
        {"name": "decode_long", "kind": "decode", "batch": 4, "longest": 131072, "heads": 32, "kv_heads": 4, "dim": 128,
         "dtype": "bf16", "page": 128, "window": 0},
        # A short question at the end of a history: few rows, the cache counts.
        {"name": "chunk_short", "kind": "chunk", "batch": 1, "chunk": 33, "singles": 0, "longest": 8000, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "window": 0},
        # A chunk of a long prompt, the largest contraction.
        {"name": "chunk_prompt", "kind": "chunk", "batch": 1, "chunk": 4096, "singles": 0, "longest": 16384, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "window": 0},
        # A mixed step: chunks of prompts beside sequences that decode one token.
        {"name": "chunk_mixed", "kind": "chunk", "batch": 24, "chunk": 500, "singles": 20, "longest": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "f16", "page": 32, "window": 0},
        # Prompts with a sliding window, small heads.
        {"name": "chunk_window_d64", "kind": "chunk", "batch": 3, "chunk": 2047, "singles": 0, "longest": 6000, "heads": 32,
         "kv_heads": 4, "dim": 64, "dtype": "bf16", "page": 16, "window": 1024},
    ]


def _size(rng, low, high):
    """A size between ``low`` and ``high``, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "decode", "decode", "chunk", "chunk"])
    heads, kv_heads = rng.choice([(32, 8), (32, 4), (16, 16), (28, 4), (8, 1), (40, 8), (64, 8)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128]),
            "dtype": rng.choice(["f16", "bf16"])}
    if kind in ("rope", "append"):
        case.update(tokens=_size(rng, 1, 8192), rotary=rng.choice([32, 64, case["dim"]]),
                    pairs=rng.choice(["halves", "neighbours"]), norm=rng.random() < 0.6, packed=rng.random() < 0.7)
        if kind == "append":
            case["page"] = rng.choice([16, 32, 64, 128])
        return case
    case.update(page=rng.choice([16, 32, 64, 128]), window=rng.choice([0, 0, 0, _size(rng, 16, 4096)]))
    if kind == "decode":
        batch = _size(rng, 1, 256)
        most = min(POSITIONS, (1 << 29) // (batch * kv_heads * case["dim"]))     # what the largest listed ones hold
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
    dtype, D, HQ, HK = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device, dtype=torch.float32).to(dtype)

    state = {"case": case, "dtype": dtype}
    if case["kind"] in ("rope", "append"):
        T, R = case["tokens"], case["rotary"]
        if case["packed"]:                   # slices of the projection's output
            qkv = normal(T, HQ + 2 * HK, D)
            q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
        else:
            q, k, v = normal(T, HQ, D), normal(T, HK, D), normal(T, HK, D)
        angle = torch.arange(POSITIONS, device=device, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, R, 2, device=device, dtype=torch.float64) / R)
        state.update(q=q, k=k, rotary=torch.cat([angle.cos(), angle.sin()], 1).float())
        if case["kind"] == "append":
            page = case["page"]
            pages = -(-2 * T // page) + 1    # twice the tokens: what is there already stays
            order = torch.randperm(pages, generator=g, device=device)[:-(-T // page)]
            at = torch.arange(T, device=device)
            state.update(v=v, slots=order[at // page] * page + at % page, k_cache=normal(pages, HK, page, D),
                         v_cache=normal(pages, HK, page, D))
        start = torch.randint(0, POSITIONS - T + 1, (1,), generator=g, device=device)
        state["positions"] = (start + torch.arange(T, device=device)).to(torch.int32)
        state["weights"] = ((1 + 0.1 * torch.randn((2, D), generator=g, device=device)).to(dtype).unbind(0)
                            if case["norm"] else ())
        return state

    lengths, counts = _lengths(case)
    page = case["page"]
    width = -(-max(lengths) // page)
    used = [-(-n // page) for n in lengths]
    pages = sum(used)
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    held = torch.arange(width, device=device)[None] < torch.tensor(used, device=device)[:, None]
    table = torch.zeros((len(used), width), dtype=torch.int32, device=device)
    table[held] = order
    offsets = torch.tensor([0] + counts, device=device).cumsum(0).to(torch.int32)
    state.update(q=normal(sum(counts), HQ, D), k_cache=normal(pages, HK, page, D), v_cache=normal(pages, HK, page, D),
                 page_table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device=device), offsets=offsets,
                 most=max(counts), width=width)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------
@lru_cache(maxsize=None)
def _artifact(name, dtype, constants):
    import intent_b200 as ib

    return ib.compile(getattr(ib.programs, name), constexprs={"ACT_DTYPE": dtype, **dict(constants)})


def _program(case):
    if case["kind"] in ("rope", "append"):
        constants = (("NORM", case["norm"]), ("EPS", EPS), ("PAIRS", case["pairs"]))
        return _artifact("qk_norm_rope" if case["kind"] == "rope" else "paged_kv_append", case["dtype"], constants)
    return _artifact("paged_attention" if case["kind"] == "chunk" else "paged_decode_attention", case["dtype"],
                     (("WINDOW", case["window"]),))


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        program, s = _program(case), state
        if kind == "rope":
            return program.run(s["q"], s["k"], s["positions"], s["rotary"], *s["weights"])
        if kind == "append":
            q = program.run(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rotary"], *s["weights"], s["k_cache"],
                            s["v_cache"])
            return q, s["k_cache"], s["v_cache"]
        if kind == "decode":
            return program.run(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"])
        return program.run(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["offsets"], s["lengths"])
    if kind in ("rope", "append"):
        weights = state["weights"] or (None, None)
        q = _rotate(state, state["q"], weights[0])
        k = _rotate(state, state["k"], weights[1])
        if kind == "rope":
            return q, k
        page = state["slots"] // case["page"]
        inside = state["slots"] % case["page"]
        state["k_cache"][page, :, inside] = k
        state["v_cache"][page, :, inside] = state["v"]
        return q, state["k_cache"], state["v_cache"]
    return _attend(state)


def _rotate(state, x, weight):
    case = state["case"]
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()
    R = case["rotary"]
    rows = state["rotary"][state["positions"].long()][:, None]
    cos, sin = rows[..., :R // 2], rows[..., R // 2:]
    turned = y[..., :R]
    if case["pairs"] == "halves":
        a, b = turned[..., :R // 2], turned[..., R // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., R:]], -1).to(x.dtype)


def _attend(state):
    """All sequences at once, padded to the longest: [batch, key heads, rows of the group, tokens]."""
    case, q = state["case"], state["q"]
    B, HQ, HK, D, page = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    n, length = state["most"], state["width"] * page
    lengths, offsets = state["lengths"].long(), state["offsets"].long()
    counts = offsets[1:] - offsets[:-1]
    at = torch.arange(n, device=q.device)
    real = at[None] < counts[:, None]                                   # [B, n]
    rows = torch.where(real, offsets[:-1, None] + at, 0)
    x = q[rows].float().view(B, n, HK, HQ // HK, D).permute(0, 2, 3, 1, 4).reshape(B, HK, -1, D)

    def gathered(cache):
        return cache[state["page_table"].long()].transpose(1, 2).reshape(B, HK, length, D).float()

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
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("rope", "append"):
        q = _exact_rotation(case, state, state["q"], 0)
        k = _exact_rotation(case, state, state["k"], 1)
        if case["kind"] == "rope":
            return q, k
        flat = [state[c].double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"]) for c in ("k_cache", "v_cache")]
        flat[0][state["slots"]] = k
        flat[1][state["slots"]] = state["v"].double()
        return (q, *(f.view(-1, case["page"], *f.shape[1:]).transpose(1, 2) for f in flat))
    lengths, counts = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    first = 0
    for b, (length, n) in enumerate(zip(lengths, counts)):
        pages = state["page_table"][b, :-(-length // case["page"])].long()
        for h in range(case["kv_heads"]):
            keys, values = (state[c][pages, h].reshape(-1, case["dim"])[:length].double() for c in ("k_cache", "v_cache"))
            for i in range(0, n, 1024):
                m = min(1024, n - i)
                position = torch.arange(length - n + i, length - n + i + m, device=keys.device)[:, None]
                token = torch.arange(length, device=keys.device)
                seen = (token <= position) & ((token > position - case["window"]) if case["window"] else True)
                x = state["q"][first + i:first + i + m, h * group:(h + 1) * group].double()
                logits = torch.einsum("mgd,ld->mgl", x, keys) / math.sqrt(case["dim"])
                logits = torch.where(seen[:, None], logits, -math.inf)
                weights = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
                out[first + i:first + i + m, h * group:(h + 1) * group] = torch.einsum("mgl,ld->mgd", weights, values)
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
    D, HQ, HK = case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] in ("rope", "append"):
        T = case["tokens"]
        heads = HQ + HK + (HK if case["kind"] == "append" else 0)
        size = T * (2 * heads * D * 2 + case["rotary"] * 4 + 4 + (8 if case["kind"] == "append" else 0))
        return {"bytes": float(size), "flops": float(T * (HQ + HK) * (3 * case["rotary"] + (4 * D if case["norm"] else 0)))}
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
    size = read * HK * D * 4 + rows * HQ * D * 4 + 4 * sum(-(-length // case["page"]) for length in lengths) + 8 * len(lengths)
    return {"bytes": float(size), "flops": float(4 * pairs * HQ * D)}
